"""The dense side of latent attention in 64 bits, from its formulas: rotation, packed rows, attention over all of a cache.

Everything is torch on the CPU and takes one sequence or one token at a time.  The attention returns, besides its results, bounds of what
a kernel may be off by that multiplies bf16 operands exactly, sums in fp32 and rounds softmax weights and results to bf16:

with e the error of a score (and of the exponential, as a relative one) a weight over its sum is off by a factor of
exp(+-2 e); rounding the weights to bf16 (half a step: 2^-8) makes that exp(2 e) (1 + 2^-8), the sum of the products over n keys adds
n 2^-24 of the sum of magnitudes, and the result's own rounding 2^-8 of it.  A score of d products in fp32 is off by at most
d 2^-24 times the sum of their magnitudes (plus its scaling and the exponential's approximation, 2^-20).
"""
import math

import torch

HALF_BF16 = 2.0 ** -8
E4M3_MAX = 448.0


def rotate(x, cos, sin, interleaved):
    """x [..., 64], cos / sin [..., 32] -> float64"""
    x, cos, sin = x.double(), cos.double(), sin.double()
    out = torch.empty_like(x)
    first, second = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    a, b = x[..., first], x[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out


def rotate_bound(x, cos, sin, interleaved):
    """|error| of the same in fp32, before its rounding to bf16"""
    return rotate(x.abs(), cos.abs(), -sin.abs(), interleaved).abs().maximum(rotate(x.abs(), cos.abs(), sin.abs(), interleaved).abs()) * 2.0 ** -22


def pack_latent(row):
    """A latent of 512 dims -> (512 e4m3 code bytes, 4 float64 scales)"""
    g = row.double().view(4, 128)
    amax = g.abs().amax(1)
    scales = []
    for a in amax.tolist():
        e = -126
        while a > E4M3_MAX * 2.0 ** e:
            e += 1
        scales.append(2.0 ** e)
    scale = torch.tensor(scales, dtype=torch.float64)
    codes = (g / scale[:, None]).float().to(torch.float8_e4m3fn)            # the quotients are exact in fp32
    return codes.reshape(512).view(torch.uint8), scale


def unpack_row(row):
    """A packed row of 656 bytes -> its 576 values as attention takes them: code x scale rounded to bf16"""
    codes = row[:512].view(torch.float8_e4m3fn).float().view(4, 128)
    scale = row[512:528].clone().view(torch.float32)
    return torch.cat(((codes * scale[:, None]).to(torch.bfloat16).view(512), row[528:].clone().view(torch.bfloat16)))


def attend(q, k, v, scale):
    """One query row over its keys: (out, lse, bound of out, bound of lse), float64.  q [d], k [n, d], v [n, dv]."""
    if len(k) == 0:
        z = torch.zeros(v.shape[1], dtype=torch.float64)
        return z, math.inf, z, 0.0
    q, k, v = q.double(), k.double(), v.double()
    s = k @ q * scale
    e = (k.shape[1] + 8) * 2.0 ** -24 * float((k.abs() @ q.abs()).max()) * abs(scale) + 2.0 ** -20
    p = torch.softmax(s, 0)
    out, lse = p @ v, float(torch.logsumexp(s, 0))
    mass = p @ v.abs()
    off = mass * (math.exp(2 * e) * (1 + HALF_BF16) - 1 + len(k) * 2.0 ** -24)
    return out, lse, off + (out.abs() + off) * HALF_BF16, e + len(k) * 2.0 ** -24 + abs(lse) * 2.0 ** -22


def decode(q, rows, pages, length, block, scale):
    """One sequence: q [q_len, heads, 576], rows [blocks * block, 576] values of the cache, pages: its row of the table."""
    sq, h, _ = q.shape
    length = min(max(int(length), 0), len(pages) * block)
    at = torch.arange(length)
    k = rows[pages.long()[at // block] * block + at % block]
    res = [[attend(q[j, i], k[:max(0, length - sq + 1 + j)], k[:max(0, length - sq + 1 + j), :512], scale) for i in range(h)] for j in range(sq)]
    return tuple(torch.stack([torch.stack([torch.as_tensor(c[x], dtype=torch.float64) for c in r]) for r in res]) for x in range(4))


def prefill(q, k_nope, k_rope, v, scale, causal=True):
    """One sequence: q [n, heads, 192], k_nope [m, heads, 128], k_rope [m, 64], v [m, heads, 128]"""
    n, h, _ = q.shape
    m = k_rope.shape[0]
    res = []
    for t in range(n):
        see = max(0, m - n + 1 + t) if causal else m
        res.append([attend(q[t, i], torch.cat((k_nope[:see, i], k_rope[:see]), 1), v[:see, i], scale) for i in range(h)])
    return tuple(torch.stack([torch.stack([torch.as_tensor(c[x], dtype=torch.float64) for c in r]) for r in res]) for x in range(4))
