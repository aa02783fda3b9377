"""Host-side checks of the transformer ops: what the C ABI and the torch ops refuse, result shapes, sizes
and the references' own ground, none of which needs a GPU."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import transformer_ref as R


@pytest.fixture(scope="module")
def abi():
    from torch_webgpu import abi as _abi
    return _abi


@pytest.fixture(scope="module", autouse=True)
def backend():
    import torch_webgpu
    return torch_webgpu


ops = torch.ops.webgpu
P = 4096  # stands for a device address; every call below returns before touching it


def rotary(abi, **over):
    st = (0, 512, 128, 1)
    args = dict(in_strides=(st, st), out_strides=(st, st), grad_strides=(st, st), position_strides=(0, 0, 1), weight_dtype="bf16")
    args.update({k: over.pop(k) for k in list(over) if k in ("axes", "axis_of", "rot_dim", "inverse", "eps")})
    d = abi.rotary_desc("bf16", (1, 3), (4, 2), 128, **args)
    for k, v in over.items():
        setattr(d, k, v)
    return d


def test_rotary_refusals(abi):
    L = abi.lib()

    def call(d, *ptrs):
        return L.twg_rotary(ctypes.byref(d) if d is not None else None, *(ptrs or (P,) * 6), None)

    for over, message in ((dict(dtype=8), b"float32, float16 or bfloat16"), (dict(weight_dtype=5), b"weights"), (dict(position_dtype=2), b"positions"),
                          (dict(freq_dtype=5), b"frequencies"), (dict(head_dim=1), b"head_dim"), (dict(head_dim=513), b"head_dim"),
                          (dict(rot_dim=127), b"rot_dim"), (dict(rot_dim=130), b"rot_dim"), (dict(rot_dim=0), b"rot_dim"), (dict(axes=0), b"axes"),
                          (dict(axes=9), b"axes"), (dict(batch=-1), b"negative"), (dict(seq=1 << 40), b"tokens"), (dict(batch=1 << 20, seq=1 << 20), b"tokens"),
                          (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps")):
        d = rotary(abi)
        for k, v in over.items():
            setattr(d, k, v)
        assert call(d) == abi.TWG_ERR_INVALID and message in L.twg_last_error(), (over, L.twg_last_error())
        assert L.twg_qk_norm_rotary_workspace_bytes(ctypes.byref(d)) == 0
    d = rotary(abi)
    d.axis_of[63] = 1
    assert call(d) == abi.TWG_ERR_INVALID and b"axis 1 of 1" in L.twg_last_error()
    d = rotary(abi)
    d.heads[0] = -1
    assert call(d) == abi.TWG_ERR_INVALID
    assert call(None) == abi.TWG_ERR_INVALID
    ok = rotary(abi)
    for i in range(6):
        ptrs = [P] * 6
        ptrs[i] = None
        assert call(ok, *ptrs) == abi.TWG_ERR_INVALID and b"null" in L.twg_last_error()
    assert call(ok, P + 1, P, P, P, P, P) == abi.TWG_ERR_INVALID and b"aligned" in L.twg_last_error()
    inverse = rotary(abi, inverse=True)
    assert L.twg_qk_norm_rotary(ctypes.byref(inverse), *(P,) * 8, None) == abi.TWG_ERR_INVALID
    with pytest.raises(abi.TwgError):
        rotary(abi, axis_of=[0] * 5)
    with pytest.raises(abi.TwgError):
        rotary(abi, axes=2, axis_of=[2] * 64)
    empty = rotary(abi)
    empty.seq = 0
    assert call(empty, *(None,) * 6) == abi.TWG_OK          # nothing to do: no pointer is looked at


def test_qk_norm_backward_refusals_and_workspace(abi):
    L, d = abi.lib(), rotary(abi)
    need = L.twg_qk_norm_rotary_workspace_bytes(ctypes.byref(d))
    assert need == 4 * 128 * (1 + 1) + 3 * 4 * 128         # one CTA's sums for q and for k, three tokens' tables
    big = rotary(abi)
    big.seq = 1 << 20
    assert L.twg_qk_norm_rotary_workspace_bytes(ctypes.byref(big)) == 4 * 128 * 148 * 2 + (1 << 20) * 4 * 128

    def call(ptrs, bytes_=need, desc=d):
        return L.twg_qk_norm_rotary_backward(ctypes.byref(desc), *ptrs, bytes_, None)

    full = [P] * 13
    assert call(full, need - 1) == abi.TWG_ERR_INVALID and b"smaller than" in L.twg_last_error()
    assert call(full[:12] + [None]) == abi.TWG_ERR_INVALID
    assert call(full[:12] + [P + 4]) == abi.TWG_ERR_INVALID and b"16-byte" in L.twg_last_error()
    for i in (0, 1, 4, 5, 6, 7, 8, 9):                     # not the weights, nor their gradients
        assert call([None if j == i else P for j in range(13)]) == abi.TWG_ERR_INVALID, i


def test_dropout_refusals(abi):
    L = abi.lib()
    d = abi.IterDesc()
    abi.check(L.twg_iter_contiguous(ctypes.byref(d), 2, 10))
    f32 = abi.DTYPES["float32"]

    def call(desc=d, dtype=f32, x=P, res=None, out=P, p=0.5, state=None):
        return L.twg_dropout(ctypes.byref(desc) if desc is not None else None, dtype, x, res, out, p, 1, 2, state, None)

    for bad in (dict(desc=None), dict(dtype=abi.DTYPES["float64"]), dict(x=None), dict(out=None), dict(p=-1e-9), dict(p=1.0000001),
                dict(p=float("nan")), dict(x=P + 2), dict(out=P + 1), dict(state=P + 4), dict(res=P)):  # the last: no third operand
        assert call(**bad) == abi.TWG_ERR_INVALID, bad
    broadcast = abi.make_desc((4, 5), [((4, 5), (5, 0)), ((4, 5), (5, 1))])
    assert call(desc=broadcast) == abi.TWG_ERR_INVALID and b"broadcast" in L.twg_last_error()
    abi.check(L.twg_iter_contiguous(ctypes.byref(d), 2, 0))
    assert call(x=None, out=None) == abi.TWG_OK


def test_logprobs_refusals(abi):
    L = abi.lib()

    def forward(d, *ptrs):
        return L.twg_token_logprobs(ctypes.byref(d), *(ptrs or (P,) * 7), None)

    def backward(d, *ptrs, stride=1000):
        return L.twg_token_logprobs_backward(ctypes.byref(d), *(ptrs or (P,) * 8), stride, None)

    for over in (dict(dtype=3), dict(token_dtype=2), dict(rows=-1), dict(rows=(1 << 27) + 1), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(row_stride=999),
                 dict(tokens_per_row=-1), dict(tokens_per_row=1025), dict(top=33), dict(top=-1), dict(scale=0.0), dict(scale=-1.0),
                 dict(scale=float("nan")), dict(scale=float("inf"))):
        d = abi.logprobs_desc("bf16", 4, 1000, top=2)
        for k, v in over.items():
            setattr(d, k, v)
        assert forward(d) == abi.TWG_ERR_INVALID and backward(d) == abi.TWG_ERR_INVALID, over
    d = abi.logprobs_desc("bf16", 4, 3, top=4)
    assert forward(d) == abi.TWG_ERR_INVALID and b"alternatives" in L.twg_last_error()
    d = abi.logprobs_desc("bf16", 4, 1000, top=2)
    for i in range(7):
        assert forward(d, *[None if j == i else P for j in range(7)]) == abi.TWG_ERR_INVALID, i
    assert forward(d, P + 1, *(P,) * 6) == abi.TWG_ERR_INVALID
    assert forward(d, P, P + 4, *(P,) * 5) == abi.TWG_ERR_INVALID
    for i in (0, 1, 2, 3, 7):                              # dlogp, dentropy, dlse may be absent
        assert backward(d, *[None if j == i else P for j in range(8)]) == abi.TWG_ERR_INVALID, i
    assert backward(d, stride=999) == abi.TWG_ERR_INVALID
    none = abi.logprobs_desc("bf16", 0, 1000)
    assert forward(none, *(None,) * 7) == abi.TWG_OK and backward(none, *(None,) * 8) == abi.TWG_OK


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_shapes_without_a_device():
    q, k, f = meta(2, 5, 8, 64, dtype=torch.bfloat16), meta(2, 5, 2, 64, dtype=torch.bfloat16), meta(32)
    pos = meta(2, 5, dtype=torch.long)
    assert [t.shape for t in ops.rotary_qk(q, k, pos, f)] == [q.shape, k.shape]
    out = ops.qk_norm_rotary(q, k, meta(64), None, meta(3, 2, 5, dtype=torch.int32), f, axis_of=[0, 1, 2, 2] * 8)
    assert out[0].dtype == torch.bfloat16
    grads = ops.qk_norm_rotary_backward(q, k, q, k, meta(64), None, pos, f)
    assert [tuple(t.shape) for t in grads] == [tuple(q.shape), tuple(k.shape), (64,), (0,)]
    assert ops.dropout(q, 0.5, 1, residual=q).shape == q.shape
    logp, entropy, lse, top_logp, top_ids = ops.token_logprobs(meta(4, 6, 100), meta(4, 6, 3, dtype=torch.long), top=7)
    assert (logp.shape, entropy.shape, lse.shape, top_logp.shape, top_ids.shape, top_ids.dtype) == ((4, 6, 3), (4, 6), (4, 6), (4, 6, 7), (4, 6, 7), torch.int64)


def test_op_refusals_without_a_device():
    q, k, f, pos = meta(2, 5, 8, 64), meta(2, 5, 2, 64), meta(32), meta(2, 5, dtype=torch.long)
    cases = [
        (lambda: ops.rotary(meta(5, 64), pos, f), "dimensions"),
        (lambda: ops.rotary(meta(2, 5, 8, 513), pos, f), "2 to 512"),
        (lambda: ops.rotary(meta(2, 5, 8, 62), pos, f), "frequencies"),
        (lambda: ops.rotary(q.double(), pos, f), "float32, float16 and bfloat16"),
        (lambda: ops.rotary(q, pos.float(), f), "int32 or int64"),
        (lambda: ops.rotary(q, pos, f.half()), "float32 or float64"),
        (lambda: ops.rotary(q, meta(3, 5, dtype=torch.long), f), "do not belong"),
        (lambda: ops.rotary(q, meta(2, 1, dtype=torch.long), f), "do not belong"),
        (lambda: ops.rotary(q, meta(9, 2, 5, dtype=torch.long), f, axis_of=[0] * 32), "axes"),
        (lambda: ops.rotary(q, meta(2, 2, 5, dtype=torch.long), f), "axis_of"),
        (lambda: ops.rotary(q, pos, f, axis_of=[0] * 31), "axis_of"),
        (lambda: ops.rotary(q, pos, f, axis_of=[1] * 32), "axis 1 of 1"),
        (lambda: ops.rotary(q, pos, f, axis_of=[-1] * 32), "axis -1"),
        (lambda: ops.rotary_qk(q, k.half(), pos, f), "one type"),
        (lambda: ops.rotary_qk(q, meta(2, 4, 2, 64), pos, f), "heads only"),
        (lambda: ops.rotary_qk(q, meta(2, 5, 64), pos, f), "as many dimensions"),
        (lambda: ops.qk_norm_rotary(q, k, meta(63), None, pos, f), "64 elements"),
        (lambda: ops.qk_norm_rotary(q, k, meta(64).half(), None, pos, f), "of q's type"),
        (lambda: ops.qk_norm_rotary(q.half(), k.half(), meta(64).half(), meta(64), pos, f), "of one type"),
        (lambda: ops.qk_norm_rotary(q, k, None, None, pos, f, eps=-1.0), "eps"),
        (lambda: ops.qk_norm_rotary_backward(q, q, q, k, None, None, pos, f), "does not belong"),
        (lambda: ops.dropout(q, 1.5, 0), "between 0 and 1"),
        (lambda: ops.dropout(q.long(), 0.5, 0), "float32, float16 and bfloat16"),
        (lambda: ops.dropout(q, 0.5, 0, residual=k), "residual"),
        (lambda: ops.dropout(q, 0.5, 0, residual=q.half()), "residual"),
        (lambda: ops.dropout_state(q, 0.5, meta(3, dtype=torch.long)), "state"),
        (lambda: ops.dropout(meta(1, 1, 1, 1, 1, 1, 1, 1, 1), 0.5, 0), "8 dimensions"),
        (lambda: ops.token_logprobs(meta(4, 100), meta(5, dtype=torch.long)), "do not belong"),
        (lambda: ops.token_logprobs(meta(4, 100), meta(4, 2, 2, dtype=torch.long)), "do not belong"),
        (lambda: ops.token_logprobs(meta(4, 100), meta(4)), "int32 or int64"),
        (lambda: ops.token_logprobs(meta(4, 0), meta(4, dtype=torch.long)), "vocabulary"),
        (lambda: ops.token_logprobs(meta(4, 10), meta(4, dtype=torch.long), top=11), "alternatives"),
        (lambda: ops.token_logprobs(meta(4, 100), meta(4, dtype=torch.long), top=33), "alternatives"),
        (lambda: ops.token_logprobs(meta(4, 100), meta(4, 1025, dtype=torch.long)), "tokens a row"),
        (lambda: ops.token_logprobs(meta(4, 100), meta(4, dtype=torch.long), scale=0.0), "scale"),
        (lambda: ops.token_logprobs_backward(meta(5), None, None, meta(4, 100), meta(4, dtype=torch.long), meta(4), meta(4)), "expected"),
    ]
    for i, (call, message) in enumerate(cases):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_shapes_of_symbols():
    """A graph traced for any batch: result shapes follow the symbols."""
    from torch.fx.experimental.proxy_tensor import make_fx
    seen = []

    def step(q, k, pos, f, logits, tokens):
        seen.append(type(q.shape[0]).__name__)
        out = ops.qk_norm_rotary(q, k, None, None, pos, f)
        back = ops.qk_norm_rotary_backward(*out, q, k, None, None, pos, f)
        turned = ops.rotary_qk(q, k, pos, f)
        o = ops.token_logprobs(logits, tokens, top=3)
        dx = ops.token_logprobs_backward(o[0], None, None, logits, tokens, o[1], o[2])
        return [*out, *back, *turned, ops.dropout(q, 0.5, 1), *o, dx]

    args = (meta(3, 5, 8, 64), meta(3, 5, 2, 64), meta(3, 5, dtype=torch.long), meta(32), meta(7, 100), meta(7, dtype=torch.long))
    gm = make_fx(step, tracing_mode="symbolic")(*args)
    assert seen == ["SymInt"]
    values = [tuple(int(s) for s in n.meta["val"].shape) for n in next(iter(reversed(gm.graph.nodes))).args[0]]
    q, k = (3, 5, 8, 64), (3, 5, 2, 64)
    assert values == [q, k, q, k, (0,), (0,), q, k, q, (7,), (7,), (7,), (7, 3), (7, 3), (7, 100)]


def test_generator_state_of_the_device_module():
    before = torch.webgpu.get_rng_state()
    torch.manual_seed(99)
    assert torch.webgpu.initial_seed() == 99
    state = torch.webgpu.get_rng_state()
    torch.webgpu.manual_seed(2 ** 64 - 3)
    assert torch.webgpu.initial_seed() == 2 ** 64 - 3
    assert torch.equal(torch.webgpu.get_rng_state().view(torch.int64), torch.tensor([-3, 0]))
    torch.webgpu.set_rng_state(state)
    assert torch.webgpu.initial_seed() == 99
    with pytest.raises(ValueError):
        torch.webgpu.set_rng_state(torch.zeros(3, dtype=torch.uint8))
    torch.webgpu.set_rng_state(before)


def test_torch_dropout_is_registered_and_refuses_to_be_traced():
    from torch._subclasses.fake_tensor import FakeTensorMode
    for key in ("PrivateUse1", "AutogradPrivateUse1"):
        assert any(l.startswith(key + ":") and "fallthrough" not in l.lower() for l in torch._C._dispatch_dump_table("aten::dropout").splitlines())
    with FakeTensorMode():
        x = torch.empty(4, 5, device="webgpu")
        with pytest.raises(RuntimeError, match="cannot be compiled"):
            torch.nn.functional.dropout(x, 0.5)
        assert torch.nn.functional.dropout(x, 0.5, training=False).shape == (4, 5)
        assert ops.dropout_state(x, 0.5, torch.empty(2, dtype=torch.long, device="webgpu")).shape == (4, 5)


def test_reference_generator_and_gradients():
    """The references against published vectors and against 64-bit autograd."""
    assert [int(v) for v in R.philox([[0]] * 4, [0, 0])[:, 0]] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert [int(v) for v in R.philox([[0xFFFFFFFF]] * 4, [0xFFFFFFFF] * 2)[:, 0]] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(3, 40, generator=g, dtype=torch.float64) * 2).requires_grad_()
    tokens = torch.tensor([[1, 1, 5], [2, 39, 0], [7, 8, 7]])
    gs = [torch.randn(3, 3, generator=g, dtype=torch.float64), torch.randn(3, generator=g, dtype=torch.float64), torch.randn(3, generator=g, dtype=torch.float64)]
    lp = torch.log_softmax(1.5 * x, -1)
    outs = (lp.gather(1, tokens), -(lp.exp() * lp).sum(-1), torch.logsumexp(1.5 * x, -1))
    (ref,) = torch.autograd.grad(outs, x, gs)
    dx, _ = R.logprobs_grad(x.detach(), tokens, 1.5, *gs)
    assert np.allclose(dx.numpy(), ref.numpy(), rtol=1e-12, atol=1e-13)
    for a, b in zip(R.logprobs(x.detach(), tokens, 1.5)[:3], outs):
        assert np.allclose(a.numpy(), b.detach().numpy(), rtol=1e-12)
