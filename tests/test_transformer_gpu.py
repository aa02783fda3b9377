"""The transformer ops on the GPU, through `torch.ops.webgpu` and through the C ABI, against 64-bit
references: rotation by positions on several axes, the norm of queries and keys with it, dropout from
the counter-based generator, token log probabilities; their gradients, layouts, streams and graphs."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import transformer_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ABI_NAMES = {torch.float32: "float32", torch.float16: "float16", torch.bfloat16: "bf16"}


@pytest.fixture(scope="module", autouse=True)
def backend():
    import torch_webgpu
    assert torch.webgpu.is_available(), "no CUDA device behind the webgpu backend"
    return torch_webgpu


@pytest.fixture(scope="module")
def abi():
    from torch_webgpu import abi as _abi
    return _abi


ops = torch.ops.webgpu


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def freqs(r, dtype=torch.float32):
    return (10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)).to(dtype)


# ------------------------------------------------------------------------------------------
# rotation
# ------------------------------------------------------------------------------------------
# batch, seq, q heads, k heads, dim, turned, axes, adjacent
ROTARY = [
    (1, 1, 1, 1, 64, 64, 1, False),
    (2, 3, 4, 2, 128, 128, 3, False),
    (3, 17, 8, 1, 128, 64, 2, False),      # partial rotation, one shared k head
    (1, 5, 3, 3, 80, 32, 1, True),
    (2, 9, 5, 5, 96, 96, 2, True),         # lanes that do not fill their group
    (1, 130, 7, 1, 256, 256, 3, False),
    (1, 4, 2, 1, 72, 72, 1, False),        # no whole vectors in half a head: the element path
    (2, 3, 2, 2, 100, 50, 2, False),
    (1, 3, 1, 1, 7, 6, 1, False),          # an odd head, an element alone
    (1, 2, 1, 1, 2, 2, 1, False),
    (1, 2, 2, 1, 512, 512, 8, False),
    (1, 2, 1, 1, 511, 256, 1, True),
    (1, 3, 70, 6, 64, 64, 1, False),       # heads of one token over several CTAs
    (4, 150, 2, 2, 32, 16, 1, False),
]


def axis_list(r, axes):
    return [j % axes for j in range(r // 2)]


def make_positions(axes, b, s, far=4096, seed=0):
    g = torch.Generator().manual_seed(seed + 7)
    return torch.randint(-3, far, (axes, b, s), generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROTARY)
def test_rotary_forward_and_gradient(case, dtype):
    b, s, hq, hk, d, r, axes, adjacent = case
    q, k = rand(b, s, hq, d, dtype=dtype), rand(b, s, hk, d, dtype=dtype, seed=1)
    pos, f, axis = make_positions(axes, b, s), freqs(r), axis_list(r, axes)
    qd, kd = q.to("webgpu").requires_grad_(), k.to("webgpu").requires_grad_()
    qo, ko = ops.rotary_qk(qd, kd, pos.to("webgpu"), f.to("webgpu"), axis_of=axis, adjacent=adjacent)
    ang = R.angles(pos, f, axis, (b, s))
    for got, x in ((qo, q), (ko, k)):
        R.assert_within(got, R.turn(x.double(), ang, adjacent), R.TURN * R.pair_size(x.double(), r, adjacent), "rotated")
    gq, gk = rand(b, s, hq, d, dtype=dtype, seed=2), rand(b, s, hk, d, dtype=dtype, seed=3)
    dq, dk = torch.autograd.grad((qo, ko), (qd, kd), (gq.to("webgpu"), gk.to("webgpu")))
    for got, g in ((dq, gq), (dk, gk)):
        R.assert_within(got, R.turn(g.double(), -ang, adjacent), R.TURN * R.pair_size(g.double(), r, adjacent), "gradient")
    # the gradient is linear in the incoming one: differences of the op along it
    h = 0.25
    plus, minus = (R.turn(q.double() + e * h * dq.cpu().double(), ang, adjacent) for e in (1, -1))
    along = float((((plus - minus) / (2 * h)) * gq.double()).sum())
    exact = float(dq.cpu().double().square().sum())
    assert abs(along - exact) <= 4 * (R.half_step(dtype) + R.TURN) * (abs(exact) + float(gq.double().square().sum()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotary_layouts(dtype):
    """Slices of a projection, heads in front of tokens, a stride along the head, a misaligned start,
    broadcast heads, three-dimensional tensors and every form of positions."""
    b, s, h, d, r = 2, 6, 4, 64, 64
    f = freqs(r)
    base = rand(b, s, 3 * h, d, dtype=dtype)
    pos = make_positions(1, b, s)[0]
    ang = R.angles(pos[None], f, [0] * (r // 2), (b, s))
    on = base.to("webgpu")
    flat = rand(b * s * h * d + 1, dtype=dtype)
    wide = rand(b, s, h, 2 * d, dtype=dtype)
    one = rand(b, s, 1, d, dtype=dtype)
    views = {
        "slice": (base[:, :, h:2 * h], on[:, :, h:2 * h]),
        "heads first": (base[:, :, :h].transpose(1, 2).contiguous().transpose(1, 2), base[:, :, :h].transpose(1, 2).contiguous().to("webgpu").transpose(1, 2)),
        "strided head": (wide[..., ::2], wide.to("webgpu")[..., ::2]),
        "misaligned": (flat[1:].view(b, s, h, d), flat.to("webgpu")[1:].view(b, s, h, d)),
        "broadcast": (one.expand(b, s, h, d), one.to("webgpu").expand(b, s, h, d)),
    }
    for name, (x, xd) in views.items():
        got = ops.rotary(xd, pos.to("webgpu"), f.to("webgpu"))
        R.assert_within(got, R.turn(x.double(), ang, False), R.TURN * R.pair_size(x.double(), r, False), name)
    assert torch.equal(on.cpu(), base), "the inputs stay as they are"
    x3 = rand(s, h, d, dtype=dtype)
    for p, ref in ((pos[0], pos[0]), (pos[:1], pos[0]), (pos[0].int(), pos[0])):
        got = ops.rotary(x3.to("webgpu"), p.to("webgpu"), f.to("webgpu"), axis_of=[0] * (r // 2) if p.dim() == 2 else [])
        R.assert_within(got, R.turn(x3.double(), R.angles(ref[None], f, [0] * (r // 2), (s,)), False),
                        R.TURN * R.pair_size(x3.double(), r, False), "three dimensions")
    shared = R.angles(pos[None, :1], f, [0] * (r // 2), (b, s))
    for p in (pos[0], pos[:1], pos[None, :1], pos[0].expand(b, s)):
        got = ops.rotary(on[:, :, :h], p.to("webgpu"), f.to("webgpu"))
        R.assert_within(got, R.turn(base[:, :, :h].double(), shared, False), R.TURN * R.pair_size(base[:, :, :h].double(), r, False), "one position for all")


def test_rotary_of_far_positions_keeps_its_digits():
    s, d = 64, 128
    x = rand(1, s, 2, d)
    for f in (freqs(d), freqs(d, torch.float64)):
        for far in (10 ** 6, 2 ** 31 - 70, 2 ** 40, -2 ** 33):
            pos = far + torch.arange(s)[None, None]
            got = ops.rotary(x.to("webgpu"), pos.to("webgpu"), f.to("webgpu"), axis_of=[0] * (d // 2))
            # pos * inv_freq in float64: half a step of the angle, twice (the product and the turns),
            # here and in the reference's own reduction
            more = 4 * abs(far) * 2.0 ** -53 * 4
            R.assert_within(got, R.turn(x.double(), R.angles(pos, f, [0] * (d // 2), (1, s)), False),
                            (R.TURN + more) * R.pair_size(x.double(), d, False), f"position {far}")


def test_rotary_empty_and_refused_on_the_device():
    f, x = freqs(64).to("webgpu"), rand(2, 3, 4, 64).to("webgpu")
    pos = torch.zeros(2, 3, dtype=torch.long).to("webgpu")
    for shape in ((0, 3, 4, 64), (2, 0, 4, 64), (2, 3, 0, 64)):
        p = torch.zeros(shape[:2], dtype=torch.long).to("webgpu")
        assert ops.rotary(torch.empty(shape, device="webgpu"), p, f).shape == shape
    with pytest.raises(RuntimeError, match="one device"):
        ops.rotary(x, pos.cpu(), f)
    with pytest.raises(RuntimeError, match="do not belong"):
        ops.rotary(x, pos[:, :2], f)
    with pytest.raises(RuntimeError, match="float32, float16 and bfloat16"):
        ops.rotary(x.double(), pos, f)


# ------------------------------------------------------------------------------------------
# the norm of queries and keys with the rotation
# ------------------------------------------------------------------------------------------
def norm_reference(x, w, dy, ang, r, adjacent, eps):
    """Forward, dx, dw in float64 with their bounds."""
    x64, d = x.double(), x.shape[-1]
    w64 = torch.ones(d, dtype=torch.float64) if w is None else w.double()
    n = R.norm(x64, None, eps)
    y = R.turn(n * w64, ang, adjacent)
    y_bound = (R.NORM + R.TURN) * R.pair_size(n * w64, r, adjacent)
    g = R.turn(dy.double(), -ang, adjacent)
    g_size = R.pair_size(dy.double(), r, adjacent)
    inv = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + eps)
    h, h_size = g * w64, g_size * w64.abs()
    dx = inv * (h - n * (h * n).mean(-1, keepdim=True))
    # r^3 (three times r's error), the sum over the head (21), its products and quotient, g's own error
    size = inv * (h_size + n.abs() * (h_size * n.abs()).mean(-1, keepdim=True))
    dx_bound = (3 * R.RNORM + R.TURN + (21 + 8) * R.U) * size
    dims = tuple(range(x.dim() - 1))
    dw, rows = (g * n).sum(dims), x.numel() // d
    # a lane adds its rows one after the other, at most all of them; then lanes, warps, strands and CTAs
    depth = min(rows, 64) + 5 + 8 + 19 + 32
    dw_bound = (R.TURN + R.RNORM + (2 + depth) * R.U) * (g_size * n.abs()).sum(dims)
    return y, y_bound, dx, dx_bound, dw, dw_bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROTARY)
def test_qk_norm_rotary_forward_and_gradient(case, dtype):
    b, s, hq, hk, d, r, axes, adjacent = case
    q, k = rand(b, s, hq, d, dtype=dtype), rand(b, s, hk, d, dtype=dtype, seed=1, scale=3.0)
    wide = case[4] in (128, 100)                       # weights in float32 beside 16-bit heads
    wt = torch.float32 if wide else dtype
    qw, kw = (1 + rand(d, seed=5, scale=0.3)).to(wt), (1 + rand(d, seed=6, scale=0.3)).to(wt)
    pos, f, axis, eps = make_positions(axes, b, s), freqs(r), axis_list(r, axes), 1e-5
    gq, gk = rand(b, s, hq, d, dtype=dtype, seed=2), rand(b, s, hk, d, dtype=dtype, seed=3)
    leaves = [t.to("webgpu").requires_grad_() for t in (q, k, qw, kw)]
    out = ops.qk_norm_rotary(*leaves, pos.to("webgpu"), f.to("webgpu"), axis_of=axis, eps=eps, adjacent=adjacent)
    grads = torch.autograd.grad(out, leaves, (gq.to("webgpu"), gk.to("webgpu")))
    ang = R.angles(pos, f, axis, (b, s))
    for i, (x, w, g) in enumerate(((q, qw, gq), (k, kw, gk))):
        y, yb, dx, dxb, dw, dwb = norm_reference(x, w, g, ang, r, adjacent, float(np.float32(eps)))
        R.assert_within(out[i], y, yb, "forward")
        R.assert_within(grads[i], dx, dxb, "dx")
        R.assert_within(grads[2 + i], dw, dwb, "dw")
        assert grads[2 + i].dtype == wt


def test_qk_norm_gradient_against_differences():
    """Central differences of the 64-bit forward along random directions of x and of the weights."""
    b, s, h, d, r, eps = 2, 5, 3, 64, 32, 1e-5
    q, k = rand(b, s, h, d), rand(b, s, 1, d, seed=1)
    qw, kw, pos, f = 1 + rand(d, seed=5, scale=0.3), 1 + rand(d, seed=6, scale=0.3), make_positions(1, b, s), freqs(r)
    gq, gk = rand(b, s, h, d, seed=2), rand(b, s, 1, d, seed=3)
    leaves = [t.to("webgpu").requires_grad_() for t in (q, k, qw, kw)]
    out = ops.qk_norm_rotary(*leaves, pos.to("webgpu"), f.to("webgpu"), axis_of=[0] * (r // 2), eps=eps)
    grads = [g.cpu().double() for g in torch.autograd.grad(out, leaves, (gq.to("webgpu"), gk.to("webgpu")))]
    ang = R.angles(pos, f, [0] * (r // 2), (b, s))

    def loss(q, k, qw, kw):
        return float((R.turn(R.norm(q, qw, eps), ang, False) * gq.double()).sum() + (R.turn(R.norm(k, kw, eps), ang, False) * gk.double()).sum())

    point = [t.double() for t in (q, k, qw, kw)]
    for i in range(4):
        v = rand(*point[i].shape, seed=40 + i).double()
        step = 1e-5
        moved = [[p + e * step * v if j == i else p for j, p in enumerate(point)] for e in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        exact = float((grads[i] * v).sum())
        # float32 gradients, a second-order remainder of about step^2 and 2^-53 / step of cancellation
        allowed = 200 * R.U * float((grads[i].abs() * v.abs()).sum()) + 1e-6 * (1 + abs(slope))
        assert abs(slope - exact) <= allowed, (i, slope, exact, allowed)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_qk_norm_without_weights_and_on_slices(dtype):
    """No weights, q and k as slices of one projection, gradients that are broadcast."""
    b, s, hq, hk, d = 2, 33, 6, 2, 64
    qkv = rand(b, s, hq + 2 * hk, d, dtype=dtype)
    on = qkv.to("webgpu")
    q, k = on[:, :, :hq], on[:, :, hq:hq + hk]
    q.requires_grad_(), k.requires_grad_()
    pos, f = make_positions(1, b, s)[0], freqs(d)
    out = ops.qk_norm_rotary(q, k, None, None, pos.to("webgpu"), f.to("webgpu"))
    one = rand(1, 1, 1, d, dtype=dtype, seed=9)
    grads = torch.autograd.grad(out, (q, k), [one.to("webgpu").expand(o.shape) for o in out])
    ang = R.angles(pos[None], f, [0] * (d // 2), (b, s))
    for i, x in enumerate((qkv[:, :, :hq], qkv[:, :, hq:hq + hk])):
        y, yb, dx, dxb, _, _ = norm_reference(x, None, one.expand(x.shape), ang, d, False, float(np.float32(1e-6)))
        R.assert_within(out[i], y, yb, "forward")
        R.assert_within(grads[i], dx, dxb, "dx")
    # one weight and not the other
    w = (1 + rand(d, seed=5, scale=0.3)).to(dtype)
    wd = w.to("webgpu").requires_grad_()
    out = ops.qk_norm_rotary(q, k, None, wd, pos.to("webgpu"), f.to("webgpu"))
    (dw,) = torch.autograd.grad(out[1], wd, one.to("webgpu").expand(out[1].shape))
    _, _, _, _, ref, bound = norm_reference(qkv[:, :, hq:hq + hk], w, one.expand(out[1].shape), ang, d, False, float(np.float32(1e-6)))
    R.assert_within(dw, ref, bound, "dw of k alone")


def test_qk_norm_gradient_is_the_same_every_time_and_once_only():
    b, s, hq, hk, d = 1, 700, 8, 2, 128
    leaves = [t.to("webgpu").requires_grad_() for t in (rand(b, s, hq, d, dtype=torch.bfloat16), rand(b, s, hk, d, dtype=torch.bfloat16),
                                                         torch.ones(d), torch.ones(d))]
    pos, f = torch.arange(s)[None].to("webgpu"), freqs(d).to("webgpu")
    g = [rand(b, s, h, d, dtype=torch.bfloat16, seed=3).to("webgpu") for h in (hq, hk)]
    runs = [[t.cpu() for t in torch.autograd.grad(ops.qk_norm_rotary(*leaves, pos, f), leaves, g)] for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
    out = ops.qk_norm_rotary(*leaves, pos, f)
    gg = [t.clone().requires_grad_() for t in g]
    first = torch.autograd.grad(out, leaves[:2], gg, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(first, gg, g)


def test_qk_norm_of_no_tokens_has_zero_weight_gradients():
    f = freqs(64).to("webgpu")
    pos = torch.zeros(0, dtype=torch.long, device="webgpu")
    leaves = [torch.empty(0, 4, 64, device="webgpu").requires_grad_(), torch.empty(0, 2, 64, device="webgpu").requires_grad_(),
              torch.ones(64).to("webgpu").requires_grad_(), torch.ones(64).to("webgpu").requires_grad_()]
    out = ops.qk_norm_rotary(*leaves, pos, f)
    grads = torch.autograd.grad(out, leaves, [torch.empty_like(o) for o in out])
    assert grads[0].shape == (0, 4, 64) and torch.equal(grads[2].cpu(), torch.zeros(64)) and torch.equal(grads[3].cpu(), torch.zeros(64))


def test_rotation_in_place_and_beside_other_rows(abi):
    """C ABI: the output may be the input; what lies between and behind the rows stays as it was."""
    b, s, h, d = 1, 5, 3, 64
    for dtype, head in ((torch.float32, d), (torch.bfloat16, 40)):   # 40 of bfloat16: the element path for half heads
        x = rand(b, s, h + 1, d + 8, dtype=dtype).cuda()
        ref = x.cpu().clone()
        pos, f = torch.arange(s, device="cuda"), freqs(head).cuda()
        st = (x.stride(0), x.stride(1), x.stride(2), 1)
        w = (1 + rand(head, seed=4, scale=0.2)).to(dtype)
        desc = abi.rotary_desc(ABI_NAMES[dtype], (b, s), (h, 0), head, in_strides=(st, st), out_strides=(st, st), position_strides=(0, 0, 1),
                               weight_dtype=ABI_NAMES[dtype], eps=1e-5)
        wd = w.cuda()
        abi.check(abi.lib().twg_qk_norm_rotary(ctypes.byref(desc), x.data_ptr(), None, wd.data_ptr(), None, pos.data_ptr(), f.data_ptr(),
                                               x.data_ptr(), None, torch.cuda.current_stream().cuda_stream))
        got = x.cpu()
        rows = ref[:, :, :h, :head]
        ang = R.angles(torch.arange(s)[None, None], freqs(head), [0] * (head // 2), (b, s))
        y, yb, *_ = norm_reference(rows, w, rows, ang, head, False, float(np.float32(1e-5)))
        R.assert_within(got[:, :, :h, :head], y, yb, "in place")
        got[:, :, :h, :head] = ref[:, :, :h, :head]
        assert torch.equal(got, ref), "elements outside the rows changed"


# ------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------
def dropped(x, p, seed, offset, residual=None):
    keep = R.keep_mask(x.shape, p, seed, offset)
    y = torch.where(keep, x.double() / (1 - p) if p < 1 else 0.0, 0.0)
    return keep, y if residual is None else y + residual.double()


def check_dropout(got, x, p, seed, offset, residual, what):
    _, ref = dropped(x, p, seed, offset, residual)
    # the scale, the product and the sum round once each
    size = 0.0 if p == 1 else 2 * R.U * torch.nan_to_num(x.double()).abs() / (1 - p)
    if residual is not None:
        size = size + R.U * ref.abs()
    R.assert_within(got, ref, torch.as_tensor(size, dtype=torch.float64), what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (1001,), (7, 64), (5, 1030), (3, 4, 5, 6), (2049, 17), ()])
@pytest.mark.parametrize("with_residual", [False, True])
def test_dropout_forward_and_gradient(shape, dtype, with_residual):
    x = rand(*shape, dtype=dtype) if shape else torch.tensor(1.5, dtype=dtype)
    res = rand(*shape, dtype=dtype, seed=8) if with_residual and shape else None
    p, seed, offset = 0.3, 0x0123456789ABCDEF, 2 ** 33 + 5
    xd = x.to("webgpu").requires_grad_()
    rd = None if res is None else res.to("webgpu").requires_grad_()
    y = ops.dropout(xd, p, seed, offset, residual=rd)
    check_dropout(y, x, p, seed, offset, res, "forward")
    g = rand(*shape, dtype=dtype, seed=3) if shape else torch.tensor(-2.0, dtype=dtype)
    grads = torch.autograd.grad(y, [xd] + ([rd] if res is not None else []), g.to("webgpu"))
    check_dropout(grads[0], g, p, seed, offset, None, "gradient")
    if res is not None:
        assert torch.equal(grads[1].cpu(), g)


def test_generator_known_answers():
    """Published vectors of Philox4x32-10: through the reference, and through the kernel's decisions."""
    kat = [((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
           ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD))]
    for ctr, key, out in kat:
        assert [int(v) for v in R.philox([[c] for c in ctr], key)[:, 0]] == list(out)
    x = torch.ones(4, device="webgpu")
    for word in (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8):     # kept exactly where the word is not below p 2^32
        for step in (0, 1):
            kept = (ops.dropout(x, (word + step) / 2 ** 32, 0, 0).cpu() != 0).tolist()
            assert kept == [w >= word + step for w in (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_mask_follows_the_element_not_the_layout(dtype):
    p, seed, offset = 0.4, -17, 3
    base = rand(6, 40, 24, dtype=dtype)
    on = base.to("webgpu")
    flat = rand(6 * 40 * 24 + 1, dtype=dtype)
    views = {"dense": lambda t: t, "transposed": lambda t: t.transpose(0, 2), "sliced": lambda t: t[:, 3:, ::2], "rows": lambda t: t[:, :, :16],
             "broadcast": lambda t: t[:, :1].expand(6, 40, 24), "reversed order": lambda t: t.permute(2, 1, 0), "one row": lambda t: t[2, 5]}
    for name, view in views.items():
        x = view(base)
        check_dropout(ops.dropout(view(on), p, seed, offset), x, p, seed, offset, None, name)
        res = rand(*x.shape, dtype=dtype, seed=4)
        strided = torch.empty(*x.shape, 2, dtype=dtype)
        strided[..., 0] = res
        check_dropout(ops.dropout(view(on), p, seed, offset, residual=strided.to("webgpu")[..., 0]), x, p, seed, offset, res, name + ", strided residual")
    check_dropout(ops.dropout(flat.to("webgpu")[1:], p, seed, offset), flat[1:], p, seed, offset, None, "misaligned")


def test_dropout_extremes():
    x = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0] * 64)
    keep, _ = dropped(torch.zeros(256), 0.5, 1, 0)
    y = ops.dropout(x.to("webgpu"), 0.5, 1).cpu()
    assert torch.equal(y[~keep], torch.zeros(int((~keep).sum()))) and torch.equal(torch.isnan(y), torch.isnan(x) & keep)
    assert torch.equal(ops.dropout(x.to("webgpu"), 1.0, 1).cpu(), torch.zeros(256))
    assert torch.equal(ops.dropout(x.to("webgpu"), 0.0, 1).cpu()[3::4], x[3::4])
    assert ops.dropout(torch.empty(0, 5, device="webgpu"), 0.5, 1).shape == (0, 5)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(RuntimeError, match="between 0 and 1"):
            ops.dropout(x.to("webgpu"), p, 1)
    with pytest.raises(RuntimeError, match="residual"):
        ops.dropout(x.to("webgpu"), 0.5, 1, residual=x[:4].to("webgpu"))
    # rates over a million elements: within five standard deviations
    n = 1 << 20
    for p in (0.1, 0.5, 0.9):
        kept = int((ops.dropout(torch.ones(n, device="webgpu"), p, 77).cpu() != 0).sum())
        assert abs(kept - n * (1 - p)) <= 5 * (n * p * (1 - p)) ** 0.5


def test_dropout_state_and_second_gradient():
    x = rand(3, 50)
    xd = x.to("webgpu").requires_grad_()
    state = torch.tensor([-5, 40]).to("webgpu")
    y = ops.dropout_state(xd, 0.25, state, 2)
    check_dropout(y, x, 0.25, -5, 42, None, "state")
    for dtype in DTYPES:                                    # the dense kernel's own plan, and the strided one
        big, res = rand(9, 1000, dtype=dtype), rand(9, 1000, dtype=dtype, seed=5)
        check_dropout(ops.dropout_state(big.to("webgpu"), 0.25, state, -1, residual=res.to("webgpu")), big, 0.25, -5, 39, res, "dense state")
        check_dropout(ops.dropout_state(big.to("webgpu").t(), 0.25, state, -41), big.t(), 0.25, -5, -1, None, "strided state")
    g = rand(3, 50, seed=1).to("webgpu").requires_grad_()
    (dx,) = torch.autograd.grad(y, xd, g, create_graph=True)
    check_dropout(dx, g.cpu().detach(), 0.25, -5, 42, None, "gradient")
    v = rand(3, 50, seed=2)
    (dg,) = torch.autograd.grad(dx, g, v.to("webgpu"))
    check_dropout(dg, v, 0.25, -5, 42, None, "gradient of the gradient")
    y = ops.dropout_state(xd, 0.25, state)
    state.fill_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, xd, g)
    for bad in (torch.zeros(3, dtype=torch.long), torch.zeros(2)):
        with pytest.raises(RuntimeError, match="state must be"):
            ops.dropout_state(xd, 0.25, bad.to("webgpu"))


def test_torch_dropout_module():
    x = rand(64, 100)
    drop = torch.nn.Dropout(0.2)
    xd = x.to("webgpu").requires_grad_()
    torch.manual_seed(1234)
    y = drop(xd)
    check_dropout(y, x, 0.2, 1234, 0, None, "first call")
    before = torch.webgpu.get_rng_state()
    second = drop(xd)
    check_dropout(second, x, 0.2, 1234, 1, None, "second call")
    torch.webgpu.set_rng_state(before)
    assert torch.equal(drop(xd).cpu(), second.cpu())
    (dx,) = torch.autograd.grad(y, xd, torch.ones(64, 100).to("webgpu"))
    check_dropout(dx, torch.ones(64, 100), 0.2, 1234, 0, None, "gradient")
    drop.eval()
    assert torch.equal(drop(xd).cpu(), x)
    torch.webgpu.manual_seed(-1)
    assert torch.webgpu.initial_seed() == 2 ** 64 - 1
    check_dropout(torch.nn.functional.dropout(xd, 0.5), x, 0.5, -1, 0, None, "negative seed")


def test_checkpointed_dropout_draws_the_same_mask_again():
    from torch.utils.checkpoint import checkpoint
    drop = torch.nn.Dropout(0.5)
    x = rand(40, 50).to("webgpu").requires_grad_()
    torch.webgpu.manual_seed(5)
    drop(x)                                               # the generator does not stand at its start
    y = checkpoint(lambda t: drop(t) * 2.0, x, use_reentrant=False)
    after = torch.webgpu.get_rng_state()
    (dx,) = torch.autograd.grad(y, x, torch.ones(40, 50).to("webgpu"))
    assert torch.equal(dx.cpu() != 0, R.keep_mask((40, 50), 0.5, 5, 1)) and torch.equal(y.detach().cpu() != 0, dx.cpu() != 0)
    assert torch.equal(torch.webgpu.get_rng_state(), after)
    with torch.random.fork_rng(devices=[0], device_type="webgpu"):
        drop(x)
    assert torch.equal(torch.webgpu.get_rng_state(), after)


# ------------------------------------------------------------------------------------------
# token log probabilities
# ------------------------------------------------------------------------------------------
def check_logprobs(out, logits, tokens, scale, top, what=""):
    logp, entropy, lse, top_logp, top_ids = out
    ref = R.logprobs(logits, tokens, scale, top)
    R.assert_within(logp, ref[0], R.logp_bound(ref[0]), f"{what} logp")
    R.assert_within(lse, ref[2], R.logp_bound(ref[2]), f"{what} lse")
    # t sums |u| times the errors of e; its exponents add their own
    R.assert_within(entropy, ref[1], 3 * R.LN_S * (1 + ref[1]), f"{what} entropy")
    assert torch.equal(top_ids.cpu(), ref[4]), f"{what} alternatives"
    R.assert_within(top_logp, ref[3], R.logp_bound(ref[3]), f"{what} top_logp")


def check_logprobs_grad(dx, logits, tokens, scale, dlogp, dentropy, dlse, what=""):
    ref, bound = R.logprobs_grad(logits, tokens, scale, dlogp, dentropy, dlse)
    R.assert_within(dx, ref, bound, f"{what} gradient")


LOGPROBS = [(1, 1, 1), (1, 2, 2), (3, 7, 5), (5, 33, 32), (2, 1000, 20), (400, 257, 4), (1, 50257, 20), (7, 4099, 1), (2, 131072, 32),
            (3, 65536 + 3, 8), (300, 5000, 0), (40, 20011, 3), (1, 8 * 16384, 5)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", LOGPROBS)
def test_token_logprobs_forward_and_gradient(case, dtype):
    rows, vocab, top = case
    logits = rand(rows, vocab, dtype=dtype, scale=3.0)
    g = torch.Generator().manual_seed(5)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    xd = logits.to("webgpu").requires_grad_()
    out = ops.token_logprobs(xd, tokens.to("webgpu"), top=top, scale=0.75)
    check_logprobs([out[0].unsqueeze(-1)] + list(out[1:]), logits, tokens[:, None], 0.75, top)
    assert not out[3].requires_grad and out[4].dtype == torch.int64
    gs = [rand(rows, seed=11), rand(rows, seed=12), rand(rows, seed=13)]
    (dx,) = torch.autograd.grad(out[:3], xd, [t.to("webgpu") for t in gs])
    assert dx.dtype == dtype
    check_logprobs_grad(dx, logits, tokens[:, None], 0.75, gs[0][:, None], gs[1], gs[2])


def test_token_logprobs_gradient_against_differences():
    rows, vocab, scale = 4, 301, 1.5
    logits, tokens = rand(rows, vocab, scale=2.0), torch.tensor([[0, 300, 0], [5, 6, 7], [1, -1, 1], [9, 9, 9]])
    gs = [rand(rows, 3, seed=1), rand(rows, seed=2), rand(rows, seed=3)]
    xd = logits.to("webgpu").requires_grad_()
    out = ops.token_logprobs(xd, tokens.to("webgpu"), scale=scale)
    (dx,) = torch.autograd.grad(out[:3], xd, [t.to("webgpu") for t in gs])
    check_logprobs_grad(dx, logits, tokens, scale, *gs)

    def loss(x):
        logp, entropy, lse, _, _ = R.logprobs(x, tokens, scale)
        return float((logp * gs[0].double()).sum() + (entropy * gs[1].double()).sum() + (lse * gs[2].double()).sum())

    for i in range(3):
        v = rand(rows, vocab, seed=20 + i).double()
        slope = (loss(logits.double() + 1e-5 * v) - loss(logits.double() - 1e-5 * v)) / 2e-5
        exact = float((dx.cpu().double() * v).sum())
        assert abs(slope - exact) <= 1e-5 * float((dx.cpu().double() * v).abs().sum()) + 1e-6 * (1 + abs(slope))


@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_with_masked_and_extreme_logits(dtype):
    """-inf, the type's lowest value, rows of either alone, a row with one token left, equal logits."""
    low, ninf = torch.finfo(dtype).min, float("-inf")
    vocab, top = 3001, 6
    x = rand(9, vocab, dtype=dtype, scale=2.0)
    x[0, 1::2] = ninf
    x[1, 10:] = low
    x[2] = ninf
    x[3] = low
    x[4] = ninf
    x[4, 77] = 1.0
    x[5] = 2.0
    x[6, :] = torch.arange(vocab).to(dtype) / 64          # rising, with runs of equal values in 16 bits
    x[7] = ninf
    x[7, 2999], x[7, 5] = -3.0, -3.0
    x[8, ::3] = 0.0
    x[8, 1::3] = -0.0
    x[8, 2::3] = ninf
    tokens = torch.tensor([[0, 1], [3, 2000], [0, 1], [5, 3000], [77, 76], [9, 9], [3000, 0], [5, 2999], [1, 2]])
    xd = x.to("webgpu").requires_grad_()
    out = ops.token_logprobs(xd, tokens.to("webgpu"), top=top, scale=1.0)
    check_logprobs(out, x, tokens, 1.0, top)
    gs = [rand(9, 2, seed=1), rand(9, seed=2), rand(9, seed=3)]
    (dx,) = torch.autograd.grad(out[:3], xd, [t.to("webgpu") for t in gs])
    check_logprobs_grad(dx, x, tokens, 1.0, *gs)
    assert torch.equal(dx.cpu()[2], torch.zeros(vocab, dtype=dtype))
    masked = torch.isinf(x[0])
    masked[tokens[0]] = False
    assert torch.equal(dx.cpu()[0][masked], torch.zeros(int(masked.sum()), dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_of_far_logits(dtype):
    """Rows whose normaliser is so large that float32 holds no digits of it behind the point, or
    leaves float32 altogether: log probabilities and gradients come from the differences."""
    vocab, scale = 2050, 1.5
    x = torch.stack([rand(vocab, dtype=dtype, scale=2.0) + c for c in (3e4, -3e4, 900.0, 0.0)])
    x[3] = torch.finfo(dtype).min
    x = x.to(dtype)
    tokens = torch.tensor([[0, 9], [5, 2049], [7, 7], [1, 2]])
    xd = x.to("webgpu").requires_grad_()
    out = ops.token_logprobs(xd, tokens.to("webgpu"), top=3, scale=scale)
    ref = R.logprobs(x, tokens, scale, 3)
    for got, want in ((out[0], ref[0]), (out[2].detach()[:3], ref[2][:3]), (out[3], ref[3])):
        R.assert_within(got, want, R.logp_bound(want), "value")
    assert torch.isneginf(out[2].cpu()[3])
    R.assert_within(out[1], ref[1], 3 * R.LN_S * (1 + ref[1]), "entropy")
    gs = [rand(4, 2, seed=1), rand(4, seed=2), rand(4, seed=3)]
    (dx,) = torch.autograd.grad(out[:3], xd, [t.to("webgpu") for t in gs])
    check_logprobs_grad(dx, x, tokens, scale, *gs)


def test_token_logprobs_of_nan_and_infinity():
    x = rand(3, 700, scale=2.0)
    x[0, 5] = float("nan")
    x[1, 6] = float("inf")
    x[0, 699] = float("nan")
    tokens = torch.tensor([1, 2, 3])
    xd = x.to("webgpu").requires_grad_()
    logp, entropy, lse, top_logp, top_ids = ops.token_logprobs(xd, tokens.to("webgpu"), top=3)
    for t in (logp, entropy, lse, top_logp):
        bad = torch.isnan(t.cpu())
        assert bad[:2].all() and not bad[2:].any()
    assert top_ids.cpu()[0, :2].tolist() == [5, 699] and int(top_ids.cpu()[1, 0]) == 6
    (dx,) = torch.autograd.grad(logp, xd, torch.ones(3).to("webgpu"))
    assert torch.isnan(dx.cpu()[:2]).all() and torch.isfinite(dx.cpu()[2]).all()


def test_token_logprobs_padding_and_unknown_tokens():
    x = rand(2, 3, 500)
    tokens = torch.tensor([[-100, 4, 499], [-1, 500, 2 ** 40]])
    xd = x.to("webgpu").requires_grad_()
    logp, *_ = ops.token_logprobs(xd, tokens.to("webgpu"))
    ref = R.logprobs(x.view(6, 500), tokens.view(6, 1), 1.0)
    R.assert_within(logp.reshape(6, 1), ref[0], R.logp_bound(ref[0]), "logp")
    assert logp.cpu()[0, 0] == 0 and logp.cpu()[1, 0] == 0 and torch.isnan(logp.cpu()[1, 1:]).all()
    g = rand(2, 3, seed=1)
    (dx,) = torch.autograd.grad(logp, xd, g.to("webgpu"))
    zero = torch.zeros(6)
    check_logprobs_grad(dx.reshape(6, 500), x.view(6, 500), tokens.view(6, 1), 1.0, g.view(6, 1), zero, zero)
    assert not dx.cpu()[1].any() and not dx.cpu()[0, 0].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_layouts(dtype):
    """Padded vocabularies (rows at every alignment), strided and transposed logits, int32 and strided
    tokens, several tokens a row, outputs that only partly take part in the gradient."""
    base = rand(13, 1007, dtype=dtype, scale=2.0)
    on = base.to("webgpu")
    tok = torch.randint(0, 900, (13, 8), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    wide = base.t().contiguous()
    one = rand(1, 1007, dtype=dtype, scale=2.0, seed=3)
    views = {"padded": (base[:, :1001], on[:, :1001]), "shifted": (base[:, 5:], on[:, 5:]), "every other": (base[:, ::2], on[:, ::2]),
             "transposed": (base, wide.to("webgpu").t()), "broadcast": (one.expand(13, 1007), one.to("webgpu").expand(13, 1007))}
    for name, (x, xd) in views.items():
        t, td = tok[:, ::2] % x.shape[1], (tok % x.shape[1]).to("webgpu")[:, ::2]
        xd = xd.detach().requires_grad_()
        out = ops.token_logprobs(xd, td, top=4, scale=1.25)
        check_logprobs(out, x, t, 1.25, 4, name)
        g = rand(13, 4, seed=1)
        (dx,) = torch.autograd.grad(out[0], xd, g.to("webgpu"))
        zero = torch.zeros(13)
        check_logprobs_grad(dx, x, t, 1.25, g, zero, zero, name)
    out = ops.token_logprobs(on.view(13, 1, 1007).requires_grad_(), tok[:, :1].to("webgpu"), scale=1.25)
    assert out[0].shape == (13, 1) and out[1].shape == (13, 1)
    assert ops.token_logprobs(torch.empty(0, 50, device="webgpu"), torch.empty(0, dtype=torch.long, device="webgpu"))[0].shape == (0,)
    x = on.detach().requires_grad_()
    none = ops.token_logprobs(x, torch.empty(13, 0, dtype=torch.long, device="webgpu"), top=1)
    assert none[0].shape == (13, 0)
    (dx,) = torch.autograd.grad(none[2], x, torch.ones(13).to("webgpu"))
    check_logprobs_grad(dx, base, tok[:, :0], 1.0, torch.zeros(13, 0), torch.zeros(13), torch.ones(13), "no tokens")
    single = ops.token_logprobs(on[3], tok[3, 0].to("webgpu"), top=2)
    assert single[0].shape == () and single[3].shape == (2,)
    with pytest.raises(RuntimeError, match="once only"):
        x = on.detach().requires_grad_()
        lse = ops.token_logprobs(x, tok.to("webgpu"))[2]
        g = torch.ones(13).to("webgpu").requires_grad_()
        (dx,) = torch.autograd.grad(lse, x, g, create_graph=True)
        torch.autograd.grad(dx, g, torch.ones_like(dx))


def test_gradient_with_another_row_alignment(abi):
    """C ABI: dlogits rows at another alignment than the logits', and nothing written behind a row."""
    rows, vocab, stride = 5, 333, 341
    for dtype in (torch.float32, torch.bfloat16):
        x = rand(rows, vocab, dtype=dtype, scale=2.0).cuda()
        tokens = torch.tensor([0, 332, 8, 100, 330], device="cuda")
        dl = rand(rows, seed=1).cuda()
        buf = torch.full((rows * stride + 1,), 7.0, dtype=dtype, device="cuda")
        logp, ent, lse = (torch.empty(rows, device="cuda") for _ in range(3))
        d = abi.logprobs_desc(ABI_NAMES[dtype], rows, vocab, token_strides=(1, 1))
        s, size = torch.cuda.current_stream().cuda_stream, buf.element_size()
        abi.check(abi.lib().twg_token_logprobs(ctypes.byref(d), x.data_ptr(), tokens.data_ptr(), logp.data_ptr(), ent.data_ptr(), lse.data_ptr(),
                                               None, None, s))
        abi.check(abi.lib().twg_token_logprobs_backward(ctypes.byref(d), x.data_ptr(), tokens.data_ptr(), None, lse.data_ptr(), dl.data_ptr(), None,
                                                        None, buf.data_ptr() + size, stride, s))
        got = buf.cpu()[1:].view(rows, stride)
        zero = torch.zeros(rows)
        check_logprobs_grad(got[:, :vocab], x.cpu(), tokens.cpu()[:, None], 1.0, dl.cpu()[:, None], zero, zero)
        assert buf[0] == 7 and bool((got[:, vocab:] == 7).all())


# ------------------------------------------------------------------------------------------
# streams, graphs, compiled functions, all of them in a row
# ------------------------------------------------------------------------------------------
def test_ops_run_on_the_current_stream():
    x = rand(256, 2048)
    side = torch.Stream(device="webgpu")
    tokens = torch.arange(256)
    with side:
        xd = x.to("webgpu")
        y = ops.dropout(xd, 0.5, 9)
        out = ops.token_logprobs(y, tokens.to("webgpu"), top=2)
        qo = ops.rotary(xd.view(256, 16, 128), tokens.to("webgpu"), freqs(128).to("webgpu"))
        got = [t.cpu() for t in (y, *out, qo)]
    side.synchronize()
    check_dropout(got[0], x, 0.5, 9, 0, None, "side stream")
    check_logprobs([got[1][:, None]] + got[2:6], got[0], tokens[:, None], 1.0, 2)
    ang = R.angles(tokens[None], freqs(128), [0] * 64, (256,))
    R.assert_within(got[6], R.turn(x.view(256, 16, 128).double(), ang, False), R.TURN * R.pair_size(x.view(256, 16, 128).double(), 128, False), "rotated")


def test_backward_follows_the_forward_stream():
    """The gradient runs on the stream of the forward pass, wherever backward() is called from; two host
    threads may run the ops at once."""
    import threading
    b, s, h, d = 2, 64, 4, 64
    f, pos = freqs(d).to("webgpu"), torch.arange(s).expand(b, s).to("webgpu")
    torch.webgpu.synchronize()
    ang = R.angles(torch.arange(s).expand(b, s)[None], freqs(d), [0] * (d // 2), (b, s))
    failures = []

    def work(seed):
        try:
            q, k, gq, gk = (rand(b, s, h, d, seed=seed + i) for i in range(4))
            side = torch.Stream(device="webgpu")
            for _ in range(5):
                with side:
                    leaves = [t.to("webgpu").requires_grad_() for t in (q, k)]
                    out = ops.qk_norm_rotary(*leaves, None, None, pos, f)
                    g = [t.to("webgpu") for t in (gq, gk)]
                side.synchronize()
                torch.autograd.backward(out, g)
                torch.webgpu.synchronize()
                for leaf, x, gr in zip(leaves, (q, k), (gq, gk)):
                    _, _, dx, dxb, _, _ = norm_reference(x, None, gr, ang, d, False, float(np.float32(1e-6)))
                    R.assert_within(leaf.grad, dx, dxb, "dx")
        except BaseException as e:  # noqa: BLE001 - reported by the main thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=(100 * i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[0]


def test_no_gradient_for_frequencies():
    f = freqs(64).to("webgpu").requires_grad_()
    x, pos = rand(3, 2, 64).to("webgpu"), torch.arange(3).to("webgpu")
    with pytest.raises(RuntimeError, match="no gradient for inv_freq"):
        ops.rotary(x, pos, f)
    with torch.no_grad():
        assert ops.rotary(x, pos, f).shape == x.shape


def test_compiled_function_of_any_batch():
    from torch_webgpu import webgpu_backend

    def step(logits, tokens, state):
        return torch.ops.webgpu.token_logprobs(torch.ops.webgpu.dropout_state(logits, 0.1, state), tokens)[0]

    fn = torch.compile(step, backend=webgpu_backend, dynamic=True)
    for n in (3, 5, 8):
        args = [t.to("webgpu") for t in (rand(n, 70), torch.arange(n), torch.tensor([1, 2]))]
        assert torch.equal(fn(*args).cpu(), step(*args).cpu())


def test_graphs_replay_with_new_inputs_and_a_shared_workspace(abi):
    """Two captured graphs that share the gradient's workspace, replayed in turn on new contents; dropout
    draws another mask in every replay through its state."""
    L, b, s, hq, hk, d = abi.lib(), 1, 300, 4, 2, 64
    mk = lambda h, seed: rand(b, s, h, d, dtype=torch.bfloat16, seed=seed).cuda()  # noqa: E731
    q, k, gq, gk = mk(hq, 1), mk(hk, 2), mk(hq, 3), mk(hk, 4)
    w = torch.ones(d, device="cuda")
    pos, f = torch.arange(s, device="cuda"), freqs(d).cuda()
    desc = abi.rotary_desc("bf16", (b, s), (hq, hk), d, in_strides=(q.stride(), k.stride()), out_strides=(q.stride(), k.stride()),
                           grad_strides=(gq.stride(), gk.stride()), position_strides=(0, 0, 1), eps=1e-5)
    nbytes = L.twg_qk_norm_rotary_workspace_bytes(ctypes.byref(desc))
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    state = torch.tensor([11, 0], device="cuda")
    act, dropped_out = rand(77, 33).cuda(), torch.empty(77, 33, device="cuda")
    it = abi.IterDesc()
    abi.check(L.twg_iter_contiguous(ctypes.byref(it), 2, act.numel()))
    outs = []

    def work(scale):
        dq, dk, dqw, dkw = torch.empty_like(q), torch.empty_like(k), torch.empty_like(w), torch.empty_like(w)
        st = torch.cuda.current_stream().cuda_stream
        abi.check(L.twg_qk_norm_rotary_backward(ctypes.byref(desc), q.data_ptr(), k.data_ptr(), w.data_ptr(), w.data_ptr(), pos.data_ptr(),
                                                f.data_ptr(), gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), dqw.data_ptr(),
                                                dkw.data_ptr(), ws.data_ptr(), nbytes, st))
        abi.check(L.twg_dropout(ctypes.byref(it), abi.DTYPES["float32"], act.data_ptr(), None, dropped_out.data_ptr(), 0.5, 0, scale,
                                state.data_ptr(), st))
        return dq, dk, dqw, dkw

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work(0)
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(100 * i))
        graphs.append(g)
    ang = R.angles(pos.cpu()[None, None], f.cpu(), [0] * (d // 2), (b, s))
    for step in range(4):
        q.copy_(mk(hq, 10 + step))
        gk.copy_(mk(hk, 20 + step))
        state.copy_(torch.tensor([11, step], device="cuda"))
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        dq, dk, dqw, dkw = outs[step % 2]
        for x, g, dx, dw in ((q, gq, dq, dqw), (k, gk, dk, dkw)):
            _, _, rx, bx, rw, bw = norm_reference(x.cpu(), w.cpu(), g.cpu(), ang, d, False, float(np.float32(1e-5)))
            R.assert_within(dx, rx, bx, "dx")
            R.assert_within(dw, rw, bw, "dw")
        check_dropout(dropped_out, act.cpu(), 0.5, 11, step + 100 * (step % 2), None, "replayed mask")


def test_compiled_function_with_the_ops():
    from torch_webgpu import webgpu_backend

    def step(x, res, state, logits, tokens):
        y = torch.ops.webgpu.dropout_state(torch.relu(x + 1.0), 0.25, state, residual=res)
        return y * 2.0, torch.ops.webgpu.token_logprobs(logits, tokens, top=2)[3]

    x, res, logits, tokens = rand(20, 30), rand(20, 30, seed=1), rand(4, 90, seed=2), torch.tensor([1, 2, 3, 4])
    args = [t.to("webgpu") for t in (x, res, torch.tensor([3, 4]), logits, tokens)]
    y, top = torch.compile(step, backend=webgpu_backend)(*args)
    ye, tope = step(*args)
    assert torch.equal(y.cpu(), ye.cpu()) and torch.equal(top.cpu(), tope.cpu())


def test_a_training_step_of_all_of_them():
    """q, k -> norm and rotation -> dropout with a residual -> log probabilities, and back, against
    64-bit autograd of the same chain."""
    b, s, h, d = 2, 24, 4, 128
    q, k = rand(b, s, h, d), rand(b, s, h, d, seed=1)
    qw, kw = 1 + rand(d, seed=5, scale=0.2), 1 + rand(d, seed=6, scale=0.2)
    pos, f, axis = make_positions(3, b, s), freqs(d), axis_list(d, 3)
    tokens = torch.randint(0, h * d, (b, s), generator=torch.Generator().manual_seed(3))
    gs = [rand(b, s, seed=21), rand(b, s, seed=22) * 0.1, rand(b, s, seed=23) * 0.1]

    def chain(q, k, qw, kw, ref):
        if ref:
            ang = R.angles(pos, f, axis, (b, s))
            qo, ko = (R.turn(R.norm(x, w, float(np.float32(1e-6))), ang, False) for x, w in ((q, qw), (k, kw)))
            keep = R.keep_mask(qo.shape, 0.2, 5, 6)
            y = torch.where(keep, qo / 0.8, 0.0) + ko
            z = torch.log_softmax(y.reshape(b, s, h * d), -1)
            return (z.gather(-1, tokens[..., None])[..., 0], -(z.exp() * z).sum(-1), torch.logsumexp(y.reshape(b, s, h * d), -1))
        qo, ko = ops.qk_norm_rotary(q, k, qw, kw, pos.to("webgpu"), f.to("webgpu"), axis_of=axis)
        y = ops.dropout(qo, 0.2, 5, 6, residual=ko)
        return ops.token_logprobs(y.reshape(b, s, h * d), tokens.to("webgpu"))[:3]

    ref_leaves = [t.double().requires_grad_() for t in (q, k, qw, kw)]
    ref_out = chain(*ref_leaves, True)
    ref = torch.autograd.grad(ref_out, ref_leaves, [t.double() for t in gs])
    leaves = [t.to("webgpu").requires_grad_() for t in (q, k, qw, kw)]
    out = chain(*leaves, False)
    torch.autograd.backward(out, [t.to("webgpu") for t in gs])
    for a, r in zip(out, ref_out):
        # the row's logits are off by at most (NORM + TURN + 3 U) of their pairs' size, 16 at the most here
        R.assert_within(a, r, (R.NORM + R.TURN + 3 * R.U) * 16 * 4 + 3 * R.LN_S * 10, "output")
    for leaf, r in zip(leaves, ref):
        # relative errors of the probabilities (those of the logits) and of both gradients' sums, at the
        # scale of the whole gradient
        err = (leaf.grad.cpu().double() - r).norm() / r.norm()
        assert err <= 4 * (R.LN_S + 16 * (R.NORM + R.TURN) + 3 * R.RNORM + 100 * R.U), float(err)


def test_nothing_is_written_behind_the_outputs(abi):
    """Guard words behind every block of the allocator, odd sizes of everything."""
    L = abi.lib()
    abi.check(L.twg_set_guard_words(1))
    keep = []
    try:
        for dtype in DTYPES:
            for d, r in ((64, 64), (72, 72), (100, 50), (7, 4)):
                q, k = rand(1, 13, 5, d, dtype=dtype).to("webgpu").requires_grad_(), rand(1, 13, 1, d, dtype=dtype).to("webgpu").requires_grad_()
                w = torch.ones(d, dtype=dtype).to("webgpu").requires_grad_()
                pos, f = torch.arange(13).to("webgpu"), freqs(r).to("webgpu")
                out = ops.qk_norm_rotary(q, k, w, w.detach().clone().requires_grad_(), pos, f)
                keep += [q, k, w, pos, f, *out, *ops.rotary_qk(q, k, pos, f)]
                keep += torch.autograd.grad(out, (q, k, w), [torch.empty_like(o).fill_(1) for o in out])
            for n in (1, 7, 1001):
                x = rand(n, dtype=dtype).to("webgpu")
                keep += [x, ops.dropout(x, 0.3, 1), ops.dropout(x, 0.3, 1, residual=x)]
            for rows, vocab, top in ((1, 5, 5), (3, 1003, 7), (2, 40001, 20)):
                x = rand(rows, vocab, dtype=dtype).to("webgpu").requires_grad_()
                out = ops.token_logprobs(x, torch.zeros(rows, 3, dtype=torch.long).to("webgpu"), top=top)
                keep += [x, *out, torch.autograd.grad(out[0], x, torch.empty_like(out[0]).fill_(1))[0]]
        bad, first = ctypes.c_int64(-1), ctypes.c_void_p()
        abi.check(L.twg_check_guard_words(0, ctypes.byref(bad), ctypes.byref(first)))
        assert bad.value == 0, f"{bad.value} blocks were written behind their end, the first at {first.value:#x}"
    finally:
        abi.check(L.twg_set_guard_words(0))


def test_offsets_beyond_32_bits(abi):
    """C ABI: strides that put the second token, row or slice more than 2^31 elements behind the first."""
    L, far, d = abi.lib(), 2 ** 31 + 64, 128
    buf = torch.zeros(far + 4096, dtype=torch.bfloat16, device="cuda")
    x = rand(2, 2, d, dtype=torch.bfloat16)
    buf[:2 * d], buf[far:far + 2 * d] = x[0].reshape(-1).cuda(), x[1].reshape(-1).cuda()
    st = torch.cuda.current_stream().cuda_stream
    pos, f = torch.arange(2, device="cuda") + 5, freqs(d).cuda()
    wide, dense = (0, far, d, 1), (0, 2 * d, d, 1)
    out = torch.empty(1, 2, 2, d, dtype=torch.bfloat16, device="cuda")
    ang = R.angles(pos.cpu()[None, None], f.cpu(), [0] * (d // 2), (1, 2))
    desc = abi.rotary_desc("bf16", (1, 2), (2, 0), d, in_strides=(wide, wide), out_strides=(dense, dense), grad_strides=(wide, wide),
                           position_strides=(0, 0, 1), eps=1e-5)
    abi.check(L.twg_rotary(ctypes.byref(desc), buf.data_ptr(), None, pos.data_ptr(), f.data_ptr(), out.data_ptr(), None, st))
    R.assert_within(out, R.turn(x[None].double(), ang, False), R.TURN * R.pair_size(x[None].double(), d, False), "far token")
    ws = torch.empty(L.twg_qk_norm_rotary_workspace_bytes(ctypes.byref(desc)), dtype=torch.uint8, device="cuda")
    abi.check(L.twg_qk_norm_rotary_backward(ctypes.byref(desc), buf.data_ptr(), None, None, None, pos.data_ptr(), f.data_ptr(), buf.data_ptr(), None,
                                            out.data_ptr(), None, None, None, ws.data_ptr(), ws.numel(), st))
    _, _, dx, dxb, _, _ = norm_reference(x[None], None, x[None], ang, d, False, float(np.float32(1e-5)))
    R.assert_within(out, dx, dxb, "far gradient")

    rows = x.reshape(2, 2 * d)
    tokens, numbers = torch.tensor([3, 200], device="cuda"), torch.empty(3, 2, device="cuda")
    top_logp, ids = torch.empty(2, 4, device="cuda"), torch.empty(2, 4, dtype=torch.long, device="cuda")
    ld = abi.logprobs_desc("bf16", 2, 2 * d, row_stride=far, token_strides=(1, 1), top=4)
    abi.check(L.twg_token_logprobs(ctypes.byref(ld), buf.data_ptr(), tokens.data_ptr(), numbers[0].data_ptr(), numbers[1].data_ptr(),
                                   numbers[2].data_ptr(), top_logp.data_ptr(), ids.data_ptr(), st))
    check_logprobs([numbers[0][:, None], numbers[1], numbers[2], top_logp, ids], rows, tokens.cpu()[:, None], 1.0, 4)

    it = abi.make_desc((2, 2 * d), [((2, 2 * d), (2 * d, 1)), ((2, 2 * d), (far, 1))])
    abi.check(L.twg_dropout(ctypes.byref(it), abi.DTYPES["bf16"], buf.data_ptr(), None, out.data_ptr(), 0.5, 3, 4, None, st))
    assert abi.last_path() == "strided64"
    check_dropout(out.view(2, 2 * d), rows, 0.5, 3, 4, None, "far rows")
    grad = torch.zeros_like(buf)
    abi.check(L.twg_token_logprobs_backward(ctypes.byref(ld), buf.data_ptr(), tokens.data_ptr(), None, numbers[2].data_ptr(), numbers[1].data_ptr(),
                                            None, None, grad.data_ptr(), far, st))
    got = torch.stack([grad[:2 * d], grad[far:far + 2 * d]]).cpu()
    zero = torch.zeros(2)
    check_logprobs_grad(got, rows, tokens.cpu()[:, None], 1.0, numbers[1].cpu()[:, None], zero, zero)
    assert not bool(grad[2 * d:far].any())


def test_dropout_of_more_than_2_to_34_elements(abi):
    """Blocks whose number needs more than 32 bits, in place."""
    n = 2 ** 34 + 1027
    if torch.cuda.mem_get_info()[0] < 2 * n + (8 << 30):
        pytest.skip("needs 42 GB of free memory")
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    d = abi.IterDesc()
    abi.check(abi.lib().twg_iter_contiguous(ctypes.byref(d), 2, n))
    abi.check(abi.lib().twg_dropout(ctypes.byref(d), abi.DTYPES["bf16"], x.data_ptr(), None, x.data_ptr(), 0.5, 77, 5, None,
                                    torch.cuda.current_stream().cuda_stream))
    for lo in (0, 2 ** 33 - 512, 2 ** 34 - 1024, n - 1027):
        lo, hi = lo // 4 * 4, min(n, lo // 4 * 4 + 1028)
        block = np.arange(lo // 4, (hi + 3) // 4, dtype=np.uint64)
        same = np.ones_like(block)
        words = R.philox([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), same * np.uint64(5), same * np.uint64(0)], [77, 0]).T.reshape(-1)
        keep = torch.from_numpy(words >= np.uint64(2 ** 31))[:hi - lo]
        assert torch.equal(x[lo:hi].cpu().float(), torch.where(keep, 2.0, 0.0)), lo
    del x
    torch.cuda.empty_cache()


def test_second_device_is_honoured(abi):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x = rand(64, 256)
    xd = x.to("webgpu:1")
    y = ops.dropout(xd, 0.5, 9)
    assert y.device.index == 1 and torch.webgpu.current_device() == 0
    check_dropout(y, x, 0.5, 9, 0, None, "second device")
