"""The 4-bit key/value cache and its attention in 64 bits (test infrastructure): the definition in include/audio8_b200.h
written with plain torch operations."""
from __future__ import annotations

import torch

BF = torch.bfloat16
GROUP = 32


def rotate(x, cos, sin):
    """rotate_half of heads x [rows, heads, hd] (bf16 values) by table rows [rows, hd]: an fp32 sum of exact products,
    rounded to bf16. float64 in and out."""
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h].double(), x[..., h:].double(), cos[:, None, :h].double(), sin[:, None, :h].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1).float().to(BF).double()


def quantise(x):
    """(codes, scales) float64 of bf16-valued x [..., hd]; a group with an inf or NaN has scale NaN, codes 0."""
    g = x.double().unflatten(-1, (-1, GROUP))
    ok = torch.isfinite(g).all(-1)
    g = torch.where(ok[..., None], g, torch.zeros_like(g))
    s = (g.abs().amax(-1) / 7).float().to(BF).double()
    c = torch.where(s[..., None] > 0, torch.round(g / s.clamp(min=1e-300)[..., None]), torch.zeros_like(g)).clamp(-7, 7)
    return c, torch.where(ok, s, torch.full_like(s, float("nan")))


def values(x):
    """What the cache holds of bf16-valued x [..., hd], float64."""
    c, s = quantise(x)
    return (c * s[..., None]).flatten(-2)


def logit_error(q, k):
    """[m, n]: what q.k (before the softmax scale) may be off by, as `attention` derives it; batch dimensions allowed."""
    gq = q.abs().unflatten(-1, (-1, GROUP)).sum(-1)
    gk = k.abs().unflatten(-1, (-1, GROUP)).amax(-1) / 6.9
    return 2.0 ** -18 * (q.abs() @ k.abs().transpose(-1, -2)) + 2.0 ** -13 * (gq @ gk.transpose(-1, -2))


def attention(q, k, v, first, scale):
    """(out, err) [m, hd] float64: row i of q [m, hd] over keys [0, first + i] of k / v [n, hd], and a bound of what a
    kernel with fp32 sums and bf16 softmax weights may be off by. A rounding to bf16 is off by at most 2^-8 of its value:
    one on every weight (together at most 2^-8 sum p|v| / sum p), one on the output (2^-8 |out|). A logit sums, over the
    32-dim groups, s q.code: at most 128 exact products, 16 at a time, fewer than 32 roundings of 2^-23 of the sum so far:
    2^-18 scale sum_d |q_d k_d|. A kernel may hold the codes as code + 8 and take 8 sum q off afterwards; a group's sum of
    32 products of up to 15 |q_d| is then off by at most 40 roundings of 2^-23 of it, 2^-13 s sum_d |q_d|, with
    s <= max|k| / 6.9 over the group. A logit's error moves a weight by as much of itself, in the numerator and in the sum
    below; the fp32 sums over keys add at most n 2^-23, taken as 2^-10 (far above it at the lengths tested)."""
    m, n = q.shape[0], k.shape[0]
    z = q @ k.T * scale
    far = torch.arange(n)[None, :] > first + torch.arange(m)[:, None]
    z = z.masked_fill(far, float("-inf"))
    p = torch.softmax(z, -1)
    out = p @ v
    pv = p @ v.abs()
    logit = logit_error(q, k).mul(scale).masked_fill(far, 0).amax(-1, keepdim=True)
    return out, 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -10 + 2 * logit) * pv + 1e-30


def prompt_slack(q, k, v, first, scale):
    """What the prompt kernel's fp16 operands add to `attention`'s bound, [m, hd] float64. A tile of 64 keys is divided by
    a power of two 2^e <= its largest scale, a query vector by 2^f <= its largest element; V by the largest such power up to
    the tile. A scale's quotient and its product with a code (8 and 8 + 3 bits, below 2 and 14) are exact while they are
    normal fp16 numbers; below 2^-14 each is off by at most half a subnormal step, 2^-25, the quotient's error times a code
    of up to 7. So an element of V is off by at most (7 + 1) 2^-25 2^E, of K by 8 2^-25 2^e, and of q (one rounding) by
    2^-25 2^f. Where a tile's scales lie further apart and keys behind a row are in it, each key has its own exponents, below those
    of the largest that the row attends. With s <= (max|x| / 7)(1 + 2^-8), 2^e <= max|k| / 6.9 over the keys that the row
    attends (the weights add up to one, so V's term passes to the output as it is); a logit moves by at most
    scale (sum_d |q_d| 8 2^-25 max|k| / 6.9 + sum_d |k_d| 2^-25 max|q|), a weight by as much of itself, in the numerator and in
    the sum below. A weight below 2^-14 of its scale is off by 2^-25, against a sum of at least 2^6 (the largest is 2^6 or
    more), times up to 14 2^E of V: 14 2^-31 max|v| / 6.9 a key."""
    m = q.shape[0]
    out = torch.zeros(m, q.shape[1], dtype=torch.float64)
    for i in range(m):
        last = first + i + 1
        kmax, vmax = k[:last].abs().max(), v[:last].abs().max()
        move = scale * 2.0 ** -25 * (8 / 6.9 * q[i].abs().sum() * kmax + k[:last].abs().sum(1).max() * q[i].abs().max())
        out[i] = (8 / 6.9 * 2.0 ** -25 + last * 14 / 6.9 * 2.0 ** -31) * vmax + 2 * move * v[:last].abs().max(0).values
    return out
