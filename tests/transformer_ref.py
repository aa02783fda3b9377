"""64-bit references of the transformer ops and the distances that their float32 arithmetic allows.

Every function computes on the CPU in float64 from the values the kernel read.  A bound is made of
the roundings on the way, each at most half a step relative (2^-24 in float32, `half_step` of the
result's type once at the end), multiplied by the magnitudes they apply to.
"""
from __future__ import annotations

import numpy as np
import torch

U = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def floor_of(dtype: torch.dtype) -> float:
    """Half the smallest subnormal of a result's type, and float32's smallest normal number, below
    which the exponentials are flushed."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 + 2.0 ** -126


def assert_within(got: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    """|got - ref| <= bound + one rounding to got's type; NaN and infinities in the same places."""
    dtype = got.dtype
    got, ref = got.detach().cpu().double(), ref.detach().double()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)} != {tuple(ref.shape)}"
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities differ"
    fin = torch.isfinite(ref)
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(ref)[fin]
    got, ref = got[fin], ref[fin]
    allowed = bound + half_step(dtype) * (ref.abs() + bound) + floor_of(dtype)
    off = (got - ref).abs() - allowed
    if off.numel():
        i = int(off.argmax())
        assert off[i] <= 0, f"{what}: {int((off > 0).sum())} of {off.numel()} too far; worst got {got[i]:.9g}, ref {ref[i]:.9g}, allowed {allowed[i]:.3g}"


# ---------------------------------------------------------------------------------------------
# rotation
# ---------------------------------------------------------------------------------------------
def angles(positions, inv_freq, axis_of, tokens):
    """positions [axes, *tokens] -> float64 [*tokens, 1, frequencies]."""
    pos = positions.double().cpu().expand(positions.shape[0], *tokens)
    return (pos[torch.tensor(axis_of)].movedim(0, -1) * inv_freq.double().cpu()).unsqueeze(-2)


def turn(x, ang, adjacent):
    r = 2 * ang.shape[-1]
    rot, rest = x[..., :r], x[..., r:]
    u, v = (rot[..., 0::2], rot[..., 1::2]) if adjacent else (rot[..., : r // 2], rot[..., r // 2:])
    a, b = u * ang.cos() - v * ang.sin(), v * ang.cos() + u * ang.sin()
    y = torch.stack([a, b], -1).flatten(-2) if adjacent else torch.cat([a, b], -1)
    return torch.cat([y, rest], -1)


def pair_size(x, r, adjacent):
    """|u| + |v| of every element's pair; the element alone behind the turned part."""
    x = x.abs()
    rot, rest = x[..., :r], x[..., r:]
    if adjacent:
        s = (rot[..., 0::2] + rot[..., 1::2]).repeat_interleave(2, -1)
    else:
        s = (rot[..., : r // 2] + rot[..., r // 2:]).repeat((1,) * (x.dim() - 1) + (2,))
    return torch.cat([s, rest], -1)


# The angle in half turns is rounded to float32 (an error of pi 2^-24 at most), its sine and cosine
# are off by at most two steps (4 U), two products and a sum round once each.
TURN = (3.2 + 4 + 3) * U
# r = rsqrt(mean + eps): a sum of at most 16 terms a lane and 5 rounds of lanes (21 U, halved by
# the root), a division and a sum (halved too), rsqrtf (2 steps, 4 U); x r w: two products more.
RNORM = (11.5 + 4) * U
NORM = RNORM + 2 * U


def norm(x, w, eps):
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return n if w is None else n * w


# ---------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 of Salmon, Moraes, Dror and Shaw (2011): uint64 arrays [4, n] of 32-bit words."""
    u, low, w = np.uint64, np.uint64(0xFFFFFFFF), np.uint64(32)
    c, k = [np.asarray(x, u) for x in counter], [int(key[0]), int(key[1])]
    for _ in range(10):
        p0, p1 = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(p1 >> w) ^ c[1] ^ u(k[0]), p1 & low, (p0 >> w) ^ c[3] ^ u(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c)


def keep_mask(shape, p, seed, offset):
    n = int(np.prod(shape, dtype=np.int64))
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    same = np.ones_like(block)
    words = philox([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), same * np.uint64(offset % 2 ** 32), same * np.uint64(offset >> 32)],
                   [seed % 2 ** 32, seed >> 32]).T.reshape(-1)[:n]
    return torch.from_numpy(words >= np.uint64(round(p * 2 ** 32))).reshape(shape)


# ---------------------------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------------------------
def logprobs(logits, tokens, scale, top=0):
    """float64 (logp, entropy, lse, top_logp, top_ids) of finite or -inf logits [rows, vocab]; a row of
    -inf alone as documented."""
    z = logits.double().cpu() * scale
    none = torch.isinf(z).all(-1) & (z[:, 0] < 0)
    m = torch.where(none, 0.0, z.amax(-1))
    e = (z - m[:, None]).exp()
    s = e.sum(-1)
    lse = torch.where(none, -torch.inf, m + s.log())
    lp = torch.where(none[:, None], -torch.inf, (z - m[:, None]) - s.clamp_min(1e-300).log()[:, None])
    p = e / s[:, None].clamp_min(1e-300)
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    tok = tokens.cpu().long()
    logp = lp.gather(1, tok.clamp(0, z.shape[1] - 1))
    logp = torch.where(tok < 0, 0.0, torch.where(tok >= z.shape[1], torch.nan, logp))
    key = logits.double().cpu() + 0.0
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :top]
    return logp, entropy, lse, lp.gather(1, ids), ids


# ln s: every e is off by 2^-22 (the exponential, 4 U) and by the rounding of its exponent u (two
# roundings of |u| bits; weighted with e their mean is at most log2 of the vocabulary, 18); each of at
# most 16 + 3 changes of the running maximum costs another exponential, two products and its exponent
# (10 U on average, most change nothing); a thread adds at most 512 terms and 11 rounds follow, whose
# roundings apply to partial sums: 64 U covers sums of positive terms that short.  logf: one step.
LN_S = (4 + 2 * 18 * 0.7 + 19 * 10 + 64 + 2) * U


def logp_bound(value):
    """Of a log probability or a normaliser: the difference from the largest logit, the scaling and the
    sum with ln s (20 at most) round at the value's magnitude."""
    return LN_S + 4 * U * (torch.nan_to_num(value, posinf=0.0, neginf=0.0).abs() + 20)


def logprobs_grad(logits, tokens, scale, dlogp, dentropy, dlse):
    """float64 gradient of logits and its bound, from the formula."""
    z = logits.double().cpu() * scale
    rows, vocab = z.shape
    logp, entropy, lse, _, _ = logprobs(logits, tokens, scale)
    none = torch.isinf(lse)[:, None]
    m = torch.where(none, 0.0, z.amax(-1, keepdim=True))
    lp = torch.where(none, -torch.inf, (z - m) - (z - m).exp().sum(-1, keepdim=True).log())
    p = lp.exp()
    lp = torch.where(p > 0, lp, 0.0)
    tok = tokens.cpu().long()
    real = (tok >= 0) & (tok < vocab)
    g = torch.where(real, dlogp.double().cpu(), 0.0)
    A = (dlse.double().cpu() - g.sum(-1))[:, None]
    dH, H = dentropy.double().cpu()[:, None], entropy[:, None]
    hot = torch.zeros_like(z).scatter_add_(1, tok.clamp(0, vocab - 1), g)
    hot_size = torch.zeros_like(z).scatter_add_(1, tok.clamp(0, vocab - 1), g.abs())
    hot, hot_size = torch.where(none, 0.0, hot), torch.where(none, 0.0, hot_size)
    dx = scale * (p * (A - dH * (lp + H)) + hot)
    # p: lse and the difference from it round at their magnitude, unless lse is so large that the row is
    # summed again; the exponential and its exponent as above; H carries ln s's error twice; the sum of
    # the tokens' gradients has as many roundings as tokens
    far = torch.nan_to_num(lse, neginf=0.0).abs()[:, None]
    size = torch.where(far > 1024, 20.0, 2 * far) + lp.abs()
    rel = LN_S + (4 * size + 2 * lp.abs() * 1.5 + 12) * U
    big_a = (dlse.double().cpu().abs() + g.abs().sum(-1) * (1 + tok.shape[1]))[:, None]
    bound = scale * (p * (rel * (big_a + dH.abs() * (lp.abs() + H)) + dH.abs() * 3 * LN_S * (1 + H)) + (4 + tok.shape[1]) * U * hot_size)
    return dx, bound
