"""Cases that measure the framework's operators between a transformer's matrix products: the rotation of queries
and keys by positions on one or several axes, the norm of each head with that rotation in the same pass, dropout
from a counter-based generator, and the log probabilities of given tokens.

`run` computes them in plain torch operations, or with `own` through the library's C entry points on torch's own
CUDA tensors.
"""
import ctypes
import math
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ABI_NAMES = {"f32": "float32", "f16": "float16", "bf16": "bf16"}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one generated token for each of 16 sequences, far into long contexts: latency counts
        dict(name="rotary_step", op="rotary", dtype="bf16", b=16, s=1, hq=32, hk=8, d=128, r=128, axes=1,
             layout="blocks", adjacent=False, backward=False, far=1000000),
        # a long prompt of video patches: time, height and width rotate their own blocks of frequencies
        dict(name="rotary_video", op="rotary", dtype="bf16", b=1, s=16384, hq=32, hk=8, d=128, r=128, axes=3,
             layout="blocks", adjacent=False, backward=False, far=16384),
        # gradient of a partial rotation of adjacent pairs, an odd sequence length, full precision
        dict(name="rotary_partial_grad", op="rotary", dtype="f32", b=4, s=1023, hq=16, hk=16, d=80, r=32, axes=1,
             layout="blocks", adjacent=True, backward=True, far=4096),
        # one generated token for each of 64 sequences, q and k still in the projection's output
        dict(name="qk_norm_step", op="qk_norm", dtype="bf16", b=64, s=1, hq=32, hk=8, d=128, r=128, axes=1,
             layout="blocks", adjacent=False, train=False, far=32768),
        # a prompt of odd length with images: three axes whose frequencies alternate
        dict(name="qk_norm_prompt", op="qk_norm", dtype="f16", b=1, s=8191, hq=64, hk=8, d=128, r=128, axes=3,
             layout="interleaved", adjacent=False, train=False, far=8191),
        # a training step's forward and backward
        dict(name="qk_norm_train", op="qk_norm", dtype="bf16", b=8, s=2048, hq=32, hk=4, d=128, r=128, axes=1,
             layout="blocks", adjacent=False, train=True, far=2048),
        # a small activation of odd width
        dict(name="dropout_small", op="dropout", dtype="f32", rows=64, cols=1001, p=0.1, residual=False, train=False),
        # the end of a sublayer in training: dropout and the residual sum, and the gradient
        dict(name="dropout_add_train", op="dropout", dtype="bf16", rows=16384, cols=4096, p=0.1, residual=True, train=True),
        # the [4096, 4096] batch slabs of this repository's benchmark, four of them
        dict(name="dropout_slabs", op="dropout", dtype="f32", rows=16384, cols=4096, p=0.5, residual=False, train=False),
        # one generated token for each of four sequences: its log probability and 20 alternatives
        dict(name="logprobs_step", op="logprobs", dtype="bf16", rows=4, vocab=131072, m=1, top=20, scale=1.25,
             masked=0.0, train=False),
        # scoring a prompt: odd vocabulary, full precision, a tenth of the vocabulary masked out
        dict(name="logprobs_score", op="logprobs", dtype="f32", rows=2047, vocab=50257, m=1, top=5, scale=1.0,
             masked=0.1, train=False),
        # a policy's training step: log probability, entropy and normaliser with their gradient
        dict(name="logprobs_train", op="logprobs", dtype="bf16", rows=4096, vocab=131072, m=1, top=0, scale=1.0,
             masked=0.0, train=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "qk_norm", "dropout", "logprobs"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op in ("rotary", "qk_norm"):
        d = rng.choice([64, 72, 80, 96, 100, 128, 128, 128, 192, 256])
        hk = rng.choice([1, 2, 4, 5, 8])
        hq = hk * rng.choice([1, 2, 4, 7, 8])
        train = op == "qk_norm" and rng.random() < 0.5
        most = 16384 * 40 * 128 * 2 // BYTES[dtype] // (hq + hk) // d // (2 if train else 1)
        tokens = _spread(rng, 1, min(16384, most))
        b = _spread(rng, 1, min(64, tokens))
        r = rng.choice([d, d, d // 2 // 2 * 2])
        case = dict(op=op, dtype=dtype, b=b, s=tokens // b, hq=hq, hk=hk, d=d, r=r, axes=rng.choice([1, 1, 2, 3]),
                    layout=rng.choice(["blocks", "interleaved"]), adjacent=rng.random() < 0.3,
                    far=_spread(rng, 128, 2000000))
        case["train" if op == "qk_norm" else "backward"] = train if op == "qk_norm" else rng.random() < 0.4
        return case
    if op == "dropout":
        train = rng.random() < 0.5
        cols = _spread(rng, 64, 16384)
        most = 16384 * 4096 * (2 if dtype != "f32" and not train else 1)
        return dict(op=op, dtype=dtype, rows=_spread(rng, 1, max(1, most // 2 // cols)), cols=cols,
                    p=round(rng.uniform(0.02, 0.6), 3), residual=rng.random() < 0.5, train=train)
    train = rng.random() < 0.5
    vocab = _spread(rng, 1000, 262144)
    rows = _spread(rng, 1, max(1, min(8192, 4096 * 131072 // (2 if dtype == "f32" else 1) // 4 // vocab)))
    return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, m=rng.choice([1, 1, 1, 4]), top=0 if train else rng.choice([0, 1, 5, 20, 32]),
                scale=round(rng.uniform(0.6, 1.7), 3), masked=rng.choice([0.0, 0.0, 0.1, 0.6]), train=train)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _axis_of(case):
    """Axis of each frequency: consecutive blocks, or axes in turn."""
    n, a = case["r"] // 2, case["axes"]
    if case["layout"] == "interleaved":
        return [j % a for j in range(n)]
    return [min(j * a // n, a - 1) for j in range(n)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    op = case["op"]
    if op in ("rotary", "qk_norm"):
        b, s, hq, hk, d, r = (case[k] for k in ("b", "s", "hq", "hk", "d", "r"))
        axis = _axis_of(case)
        # the first axis counts on from where the context stands; the others are places within an image
        start = torch.randint(0, max(1, case["far"] - s + 1), (1, b, 1), device="cuda", generator=g)
        pos = start + torch.arange(s, device="cuda").expand(1, b, s)
        if case["axes"] > 1:
            pos = torch.cat([pos, torch.randint(0, min(case["far"], 1024), (case["axes"] - 1, b, s), device="cuda", generator=g)])
        freq = (10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)).float()
        st = dict(case=case, positions=pos.contiguous(), inv_freq=freq, axis=axis,
                  axis_index=torch.tensor(axis, device="cuda"))
        if op == "rotary":
            st.update(q=normal(b, s, hq, d), k=normal(b, s, hk, d))
            return st
        # q and k are views of the projection's output, v lies behind them
        qkv = normal(b, s, hq + 2 * hk, d)
        st.update(q=qkv[:, :, :hq], k=qkv[:, :, hq:hq + hk], eps=1e-6,
                  q_weight=(1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(dt),
                  k_weight=(1 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(dt))
        if case["train"]:
            st.update(dq_out=normal(b, s, hq, d), dk_out=normal(b, s, hk, d))
        return st
    if op == "dropout":
        n = (case["rows"], case["cols"])
        st = dict(case=case, x=normal(*n), seed=seed * 2654435761 + 12345, offset=seed % 1009 + (1 << 33))
        if case["residual"]:
            st["residual"] = normal(*n)
        if case["train"]:
            st["dout"] = normal(*n)
        return st
    n, v, m = case["rows"], case["vocab"], case["m"]
    logits = torch.empty(n, v, device="cuda", dtype=dt)
    step = max(1, (1 << 28) // v)
    for i in range(0, n, step):
        x = torch.randn(min(step, n - i), v, device="cuda", generator=g) * 2.5
        if case["masked"]:
            keep = torch.rand(v, device="cuda", generator=g) >= case["masked"]
            keep[0] = True
            x = x.masked_fill(~keep, float("-inf"))
        logits[i:i + step] = x.to(dt)
    tokens = torch.randint(0, v, (n, m), device="cuda", generator=g)
    if case["masked"]:
        tokens = torch.where(torch.isinf(logits.gather(1, tokens)), torch.zeros_like(tokens), tokens)
    st = dict(case=case, logits=logits, tokens=tokens)
    if case["train"]:
        st.update(dlogp=normal(n, m, dtype=torch.float32), dentropy=normal(n, dtype=torch.float32) * 0.01,
                  dlse=normal(n, dtype=torch.float32) * 0.001)
    return st


# ---------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------
def _cos_sin(st):
    # angles of far positions lose their digits in 32 bits
    ang = st["positions"][st["axis_index"]].double() * st["inv_freq"].double()[:, None, None]
    ang = ang.permute(1, 2, 0)[:, :, None, :]
    return ang.cos().float(), ang.sin().float()


def _rotate(x, cos, sin, r, adjacent):
    """x: 32-bit [b, s, h, d]; the first r elements of d are rotated in pairs."""
    rot, rest = x[..., :r], x[..., r:]
    if adjacent:
        u, v = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    else:
        u, v = rot[..., :r // 2], rot[..., r // 2:]
        y = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    return torch.cat([y, rest], -1)


def _plain_rotary(st):
    c = st["case"]
    cos, sin = _cos_sin(st)
    sin = -sin if c["backward"] else sin
    return [_rotate(st[n].float(), cos, sin, c["r"], c["adjacent"]).to(st[n].dtype) for n in ("q", "k")]


def _plain_norm(x, w, dy, cos, sin, st):
    c = st["case"]
    x32, w32 = x.float(), w.float()
    inv = torch.rsqrt(x32.square().mean(-1, keepdim=True) + st["eps"])
    n = x32 * inv
    y = _rotate(n * w32, cos, sin, c["r"], c["adjacent"]).to(x.dtype)
    if dy is None:
        return y, None, None
    g = _rotate(dy.float(), cos, -sin, c["r"], c["adjacent"])
    h = g * w32
    dx = inv * (h - n * (h * n).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), (g * n).sum((0, 1, 2)).to(w.dtype)


def _plain_qk_norm(st):
    cos, sin = _cos_sin(st)
    q, dq, dqw = _plain_norm(st["q"], st["q_weight"], st.get("dq_out"), cos, sin, st)
    k, dk, dkw = _plain_norm(st["k"], st["k_weight"], st.get("dk_out"), cos, sin, st)
    return [q, k] if dq is None else [q, k, dq, dk, dqw, dkw]


def _words(n, seed, offset):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): word i % 4 of the block with counter (i / 4, offset)."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64)
    c0, c1 = block & low, block >> 32
    c2 = torch.full_like(block, offset & low)
    c3 = torch.full_like(block, offset >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).flatten()[:n]


def _plain_dropout(st):
    c, x = st["case"], st["x"]
    keep = (_words(x.numel(), st["seed"], st["offset"]) >= round(c["p"] * 2 ** 32)).view_as(x)
    scale = 1.0 / (1.0 - c["p"])
    y = torch.where(keep, x.float() * scale, 0.0)
    if c["residual"]:
        y = y + st["residual"].float()
    if not c["train"]:
        return [y.to(x.dtype)]
    return [y.to(x.dtype), torch.where(keep, st["dout"].float() * scale, 0.0).to(x.dtype)]


def _plain_logprobs(st):
    c, x, tokens = st["case"], st["logits"], st["tokens"]
    z = x.float() * c["scale"]
    top = z.amax(-1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(-1, keepdim=True)
    lse = top + total.log()
    p = e / total
    logp = z.gather(1, tokens) - lse
    # where nothing of a probability is left its logarithm does not count
    surprise = torch.where(p > 0, z - lse, 0.0)
    entropy = -(p * surprise).sum(-1)
    out = [logp, entropy, lse[:, 0]]
    if c["top"]:
        # one whole number for each place, the larger logit first and the lower index where they tie
        bits = x.float().view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = (order << 32) - torch.arange(x.shape[1], device="cuda")
        ids = key.topk(c["top"], -1).indices
        out += [z.gather(1, ids) - lse, ids]
    if c["train"]:
        dz = -p * (st["dlogp"].sum(-1) - st["dlse"])[:, None] - st["dentropy"][:, None] * p * (surprise + entropy[:, None])
        dz.scatter_add_(1, tokens, st["dlogp"])
        out.append((dz * c["scale"]).to(x.dtype))
    return out


# ---------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------
_abi = None


def _library():
    global _abi
    if _abi is None:
        if "torch-webgpu_b200" not in sys.path:
            sys.path.insert(1, "torch-webgpu_b200")
        from torch_webgpu import abi
        _abi = abi
    return _abi


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _rotary_desc(abi, st, q_out, k_out, grads=None, **more):
    c, pos = st["case"], st["positions"]
    return abi.rotary_desc(ABI_NAMES[c["dtype"]], (c["b"], c["s"]), (c["hq"], c["hk"]), c["d"], rot_dim=c["r"],
                           in_strides=(st["q"].stride(), st["k"].stride()), out_strides=(q_out.stride(), k_out.stride()),
                           grad_strides=None if grads is None else [g.stride() for g in grads],
                           axes=c["axes"], axis_of=st["axis"], position_strides=pos.stride(), adjacent=c["adjacent"], **more)


def _own_rotary(st):
    abi, q, k = _library(), st["q"], st["k"]
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    d = _rotary_desc(abi, st, qo, ko, inverse=st["case"]["backward"])
    abi.check(abi.lib().twg_rotary(ctypes.byref(d), q.data_ptr(), k.data_ptr(), st["positions"].data_ptr(), st["inv_freq"].data_ptr(),
                                   qo.data_ptr(), ko.data_ptr(), _stream()))
    return [qo, ko]


def _own_qk_norm(st):
    abi, c, q, k, qw, kw = _library(), st["case"], st["q"], st["k"], st["q_weight"], st["k_weight"]
    qo = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    ko = torch.empty(k.shape, dtype=k.dtype, device="cuda")
    pos, freq, name = st["positions"], st["inv_freq"], ABI_NAMES[c["dtype"]]
    d = _rotary_desc(abi, st, qo, ko, weight_dtype=name, eps=st["eps"])
    abi.check(abi.lib().twg_qk_norm_rotary(ctypes.byref(d), q.data_ptr(), k.data_ptr(), qw.data_ptr(), kw.data_ptr(), pos.data_ptr(),
                                           freq.data_ptr(), qo.data_ptr(), ko.data_ptr(), _stream()))
    if not c["train"]:
        return [qo, ko]
    dqo, dko = st["dq_out"], st["dk_out"]
    dq, dk, dqw, dkw = torch.empty_like(qo), torch.empty_like(ko), torch.empty_like(qw), torch.empty_like(kw)
    d = _rotary_desc(abi, st, dq, dk, (dqo, dko), weight_dtype=name, eps=st["eps"])
    nbytes = abi.lib().twg_qk_norm_rotary_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    abi.check(abi.lib().twg_qk_norm_rotary_backward(
        ctypes.byref(d), q.data_ptr(), k.data_ptr(), qw.data_ptr(), kw.data_ptr(), pos.data_ptr(), freq.data_ptr(), dqo.data_ptr(),
        dko.data_ptr(), dq.data_ptr(), dk.data_ptr(), dqw.data_ptr(), dkw.data_ptr(), ws.data_ptr(), nbytes, _stream()))
    return [qo, ko, dq, dk, dqw, dkw]


def _own_dropout(st):
    abi, c, x = _library(), st["case"], st["x"]
    lib, dtype, s, n = abi.lib(), abi.DTYPES[ABI_NAMES[c["dtype"]]], _stream(), x.numel()
    d = abi.IterDesc()
    abi.check(lib.twg_iter_contiguous(ctypes.byref(d), 3 if c["residual"] else 2, n))
    y = torch.empty_like(x)
    res = st["residual"].data_ptr() if c["residual"] else None
    abi.check(lib.twg_dropout(ctypes.byref(d), dtype, x.data_ptr(), res, y.data_ptr(), c["p"], st["seed"], st["offset"], None, s))
    if not c["train"]:
        return [y]
    dx, dout = torch.empty_like(x), st["dout"]
    abi.check(lib.twg_dropout(ctypes.byref(d), dtype, dout.data_ptr(), None, dx.data_ptr(), c["p"], st["seed"], st["offset"], None, s))
    return [y, dx]


def _own_logprobs(st):
    abi, c, x, tokens = _library(), st["case"], st["logits"], st["tokens"]
    lib, s, (n, v), m, top = abi.lib(), _stream(), x.shape, c["m"], c["top"]
    d = abi.logprobs_desc(ABI_NAMES[c["dtype"]], n, v, row_stride=x.stride(0), tokens_per_row=m, token_strides=tokens.stride(),
                          top=top, scale=c["scale"])
    # one block for the row's numbers: logp [n, m], entropy [n], lse [n], the alternatives' [n, top]
    numbers = torch.empty(n * (m + 2 + top), dtype=torch.float32, device="cuda")
    logp, entropy, lse, top_logp = numbers.split([n * m, n, n, n * top])
    ids = torch.empty(n, top, dtype=torch.int64, device="cuda") if top else None
    abi.check(lib.twg_token_logprobs(ctypes.byref(d), x.data_ptr(), tokens.data_ptr(), logp.data_ptr(), entropy.data_ptr(), lse.data_ptr(),
                                     top_logp.data_ptr() if top else None, ids.data_ptr() if top else None, s))
    out = [logp.view(n, m), entropy, lse]
    if top:
        out += [top_logp.view(n, top), ids]
    if c["train"]:
        dx = torch.empty_like(x)
        abi.check(lib.twg_token_logprobs_backward(
            ctypes.byref(d), x.data_ptr(), tokens.data_ptr(), entropy.data_ptr(), lse.data_ptr(), st["dlogp"].data_ptr(),
            st["dentropy"].data_ptr(), st["dlse"].data_ptr(), dx.data_ptr(), dx.stride(0), s))
        out.append(dx)
    return out


_RUN = {"rotary": (_plain_rotary, _own_rotary), "qk_norm": (_plain_qk_norm, _own_qk_norm),
        "dropout": (_plain_dropout, _own_dropout), "logprobs": (_plain_logprobs, _own_logprobs)}


def run(state):
    return _RUN[state["case"]["op"]][1 if own else 0](state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    e, op = BYTES[case["dtype"]], case["op"]
    if op in ("rotary", "qk_norm"):
        tokens = case["b"] * case["s"]
        n = tokens * (case["hq"] + case["hk"]) * case["d"]
        small = 8 * case["axes"] * tokens + 4 * (case["r"] // 2)
        if op == "rotary":
            return {"bytes": 2 * n * e + small, "flops": 3 * n}
        weights = 2 * case["d"] * e
        if not case["train"]:
            return {"bytes": 2 * n * e + small + weights, "flops": 7 * n}
        # forward: x in, y out; backward: x is there already, dy in, dx and the weights' gradients out
        return {"bytes": 4 * n * e + small + 2 * weights, "flops": 20 * n}
    if op == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * e * (2 + (1 if case["residual"] else 0) + (2 if case["train"] else 0)), "flops": 3 * n * (2 if case["train"] else 1)}
    n, v, m, top = case["rows"], case["vocab"], case["m"], case["top"]
    small = n * (12 * m + 8 + 12 * top)
    if not case["train"]:
        return {"bytes": n * v * e + small, "flops": 6 * n * v}
    return {"bytes": 2 * n * v * e + small + n * (4 * m + 8), "flops": 14 * n * v}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_turn(st, sign=1.0):
    c = st["case"]
    pos = torch.stack([st["positions"][a] for a in st["axis"]], -1).to(torch.float64)
    return torch.polar(torch.ones_like(pos), sign * pos * st["inv_freq"].to(torch.float64))[:, :, None]


def _exact_rotate(x, turn, c):
    r, half = c["r"], c["r"] // 2
    rot = x[..., :r]
    pairs = rot.unflatten(-1, (half, 2)) if c["adjacent"] else rot.unflatten(-1, (2, half)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y = (y if c["adjacent"] else y.transpose(-1, -2)).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _exact_dropout(st):
    c = st["case"]
    n = c["rows"] * c["cols"]
    u = np.uint64
    low, w = u(0xFFFFFFFF), u(32)
    seed, offset = st["seed"], st["offset"]
    keep = np.empty((n + 3) // 4 * 4, np.bool_)
    limit = u(round(c["p"] * 2 ** 32))
    for lo in range(0, (n + 3) // 4, 1 << 18):
        hi = min(lo + (1 << 18), (n + 3) // 4)
        ctr = [np.arange(lo, hi, dtype=u) & low, np.arange(lo, hi, dtype=u) >> w, np.full(hi - lo, offset % 2 ** 32, u), np.full(hi - lo, offset // 2 ** 32, u)]
        key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
        for _ in range(10):
            p0, p1 = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
            ctr = [(p1 >> w) ^ ctr[1] ^ u(key[0]), p1 & low, (p0 >> w) ^ ctr[3] ^ u(key[1]), p0 & low]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        keep[4 * lo:4 * hi] = np.stack(ctr, 1).reshape(-1) >= limit
    mask = torch.from_numpy(keep[:n]).cuda().view(c["rows"], c["cols"]).to(torch.float64) / (1.0 - c["p"])
    y = st["x"].to(torch.float64) * mask
    if c["residual"]:
        y = y + st["residual"].to(torch.float64)
    return [y, st["dout"].to(torch.float64) * mask] if c["train"] else [y]


def _exact_logprobs(st):
    c = st["case"]
    parts = []
    step = max(1, (1 << 27) // c["vocab"])
    for i in range(0, c["rows"], step):
        x = st["logits"][i:i + step].to(torch.float64)
        tokens = st["tokens"][i:i + step]
        with torch.enable_grad():
            x.requires_grad_(c["train"])
            lsm = torch.log_softmax(x * c["scale"], -1)
            logp = lsm.gather(1, tokens)
            # a masked place has no probability, and its logarithm no weight
            entropy = -(lsm.exp() * lsm.masked_fill(torch.isinf(lsm), 0.0)).sum(-1)
            lse = torch.logsumexp(x * c["scale"], -1)
            part = [logp.detach(), entropy.detach(), lse.detach()]
            if c["top"]:
                part.append(lsm.detach().topk(c["top"], -1).values)
            if c["train"]:
                loss = (logp * st["dlogp"][i:i + step]).sum() + (lse * st["dlse"][i:i + step]).sum()
                loss = loss + (entropy * st["dentropy"][i:i + step]).sum()
                (grad,) = torch.autograd.grad(loss, x)
                part.append(grad)
        parts.append(part)
        del x, lsm
    out = [torch.cat(p) for p in zip(*parts)]
    return out[:4] + [None] + out[4:] if c["top"] else out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "dropout":
        return _exact_dropout(st)
    if case["op"] == "logprobs":
        return _exact_logprobs(st)
    if case["op"] == "rotary":
        turn = _exact_turn(st, -1.0 if case["backward"] else 1.0)
        return [_exact_rotate(st[n].to(torch.float64), turn, case) for n in ("q", "k")]
    turn, out, grads, dws = _exact_turn(st), [], [], []
    for n in ("q", "k"):
        with torch.enable_grad():
            x = st[n].to(torch.float64).requires_grad_(case["train"])
            w = st[n + "_weight"].to(torch.float64).requires_grad_(case["train"])
            y = _exact_rotate(x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["d"] + st["eps"]) * w, turn, case)
            if case["train"]:
                dx, dw = torch.autograd.grad(y, [x, w], st["d" + n + "_out"].to(torch.float64))
                grads.append(dx)
                dws.append(dw)
        out.append(y.detach())
    return out + grads + dws
