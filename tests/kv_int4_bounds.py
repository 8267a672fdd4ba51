"""What the roundings of attention over 4-bit pages add up to, per row and head.

The kernels round four things: keys (half a step of fp16, 2^-11, in the prompt kernels; bf16 queries fit fp16 as they are),
probabilities or probabilities times a scale (2^-11), values (2^-11), and the output (bf16, 2^-8). Sums are fp32. A rounding of half
a step h is taken as spread evenly over +-h, a standard deviation of h / sqrt(3), and independent from one to the next, so that squares
add up. The output has one for each of its D >= 64 values: the norm of their errors is within 1.5 standard deviations (nine of the
norm's own, 1 / sqrt(5 D) each). The others are taken at four standard deviations, and for fewer than three keys, of which each may be a
half step off, that is more than the sum of all. Probabilities below fp16's normal range have a smallest step, 2^-24 of the largest
probability times magnitude (and 4 for tokens that share an exponent with larger ones). Over all rows of a call the norm of the errors
is within 1.5 standard deviations too, which a second rounding to bf16 anywhere is not.
"""
import math

import torch

from mythos_b200.ops import reference as ref

BF16, FP16 = 2.0 ** -8, 2.0 ** -11


def attention(q, kc, vc, table, first_row, n_new, n_keys, scale):
    """In 64 bits over the values that the pages stand for; keys without a page are seen by no query, and what a query does not
    see does not reach it, whatever it is. Returns the outputs [T, H, D], and of the error's norm the limit and the standard deviation [T, H]."""
    q, kc, vc, table = (t.cpu() for t in (q, kc, vc, table))
    T, H, D = q.shape
    Hk, page = kc.shape[1], kc.shape[2] // (D // 2 + D // 16)
    out = torch.zeros(T, H, D, dtype=torch.float64)
    limit, usual = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for b, (r0, nq, n) in enumerate(zip(first_row, n_new, n_keys)):
        if nq == 0 or n <= 0:
            continue
        pos = torch.arange(n)
        sid = torch.full_like(pos, b)
        k, v = (x.double() for x in ref.kv_read_int4(kc, vc, table, pos, sid, D, torch.float32))
        none = ~ref.kv4_places(table, page, kc.shape[0], pos, sid)[3]
        for h in range(H):
            for lo in range(0, nq, 512):
                rows = slice(r0 + lo, r0 + min(nq, lo + 512))
                at = torch.arange(lo, min(nq, lo + 512))
                hidden = (pos[None] > n - nq + at[:, None]) | none
                out[rows, h], limit[rows, h], usual[rows, h] = _head(q[rows, h].double(), k[:, h // (H // Hk)], v[:, h // (H // Hk)], hidden, scale)
    return out, limit, usual


def _head(q, k, v, hidden, scale):
    sc = (q @ k.T * scale).masked_fill(hidden, -math.inf)
    p = torch.softmax(sc, -1).nan_to_num(0.0)
    o = p @ v
    # roundings of p and of v, or of p times a scale, which multiplies a code or (every second token) what the code lacks to 15
    lo, hi = (f(v.unflatten(-1, (-1, 64)), -1).repeat_interleave(64, -1) for f in (torch.amin, torch.amax))
    size = torch.maximum(2 * v * v, ((v - lo) ** 2 + (hi - v) ** 2) / 2)
    delta = scale ** 2 * ((q * q) @ (k * k).T)                  # of a score, squared, in units of a key's rounding
    pp = p * p
    pd = pp * delta
    var = FP16 ** 2 / 3 * (pp @ size + pd @ (v * v) - 2 * o * (pd @ v) + o * o * pd.sum(-1, keepdim=True))
    m = v.abs().amax(-1)
    rel = torch.where(m[:, None] > 0, v / m[:, None].clamp_min(1e-300), 0.0)
    floor = (2.0 ** -22 * (p * m).amax(-1, keepdim=True)) ** 2 * ((~hidden).double() @ (rel * rel))
    last, rest = BF16 / math.sqrt(3) * o.norm(dim=-1), (var.clamp_min(0.0) + floor).sum(-1).sqrt()
    return o, 1.5 * last + 4 * rest, (last ** 2 + rest ** 2).sqrt()


def check(got, out, limit, usual):
    """Every row and head within its limit, and all of them together; outputs that are zero have to be zero."""
    assert bool(got.isfinite().all())
    off = (got.cpu().double() - out).norm(dim=-1)
    worst = torch.where(limit > 0, off / limit.clamp_min(1e-300), torch.where(off > 0, math.inf, 0.0))
    assert float(worst.max()) <= 1.0, (float(worst.max()), [int(i) for i in (worst == worst.max()).nonzero()[0]])
    if off.numel() >= 64 and bool(usual.any()):
        assert float(off.norm() / usual.norm()) <= 1.5, float(off.norm() / usual.norm())
