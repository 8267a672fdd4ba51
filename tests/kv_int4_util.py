"""Inputs and the 64-bit oracle of the 4-bit KV cache tests."""
import math

import torch

from mythos_b200.ops import functional as F, reference as ref


def make_cache(lens, Hk, D, page, device, seed=0, spare=2, stale=True):
    """Empty caches and a shuffled table for sequences of ``lens`` tokens; stale bytes everywhere."""
    g = torch.Generator().manual_seed(seed)
    used = [(n + page - 1) // page for n in lens]
    n_pages = sum(used) + spare
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(used))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (n_pages, Hk, page * F.kv4_token_bytes(D))
    fill = (lambda: torch.full(shape, 255, dtype=torch.uint8)) if stale else (lambda: torch.zeros(shape, dtype=torch.uint8))
    return fill().to(device), fill().to(device), table.to(device)     # 0xFFFF is a NaN as a scale and as a low


def token_lists(first, count, device):
    pos = torch.cat([torch.arange(f, f + c, dtype=torch.int32) for f, c in zip(first, count)])
    sid = torch.cat([torch.full((c,), b, dtype=torch.int32) for b, c in enumerate(count)])
    return pos.to(device), sid.to(device)


def random_rows(T, Hk, D, seed, device, size=1.0):
    """Keys with channels that stand out and an offset, values of unequal size."""
    g = torch.Generator().manual_seed(seed)
    stand = torch.exp(0.5 * torch.randn(Hk, D, generator=g))
    k = (torch.randn(T, Hk, D, generator=g) * stand + 0.5 * torch.randn(Hk, D, generator=g)) * size
    v = torch.randn(T, Hk, D, generator=g) * (0.3 + torch.rand(T, Hk, 1, generator=g)) * size
    return k.to(torch.bfloat16).to(device), v.to(torch.bfloat16).to(device)


def filled(lens, Hk, D, page, device, seed=0):
    kc, vc, table = make_cache(lens, Hk, D, page, device, seed)
    pos, sid = token_lists([0] * len(lens), lens, device)
    k, v = random_rows(sum(lens), Hk, D, seed + 1, device)
    if sum(lens):
        F.kv_append_int4(k, v, kc, vc, table, pos, sid)
    return kc, vc, table


def oracle(q, kc, vc, table, first_row, n_new, n_keys, scale):
    """Attention in 64 bits over the values that the pages stand for, one sequence after the other, and for every output
    the sum of p |v - middle of its group| (``centred``), of p |v| (``plain``), of p |v - o| (``spread``) and the largest
    scale sum |q| |k| over its visible keys (``logit``): what the kernels' roundings are bounded by."""
    q, kc, vc, table = (t.cpu() for t in (q, kc, vc, table))
    T, H, D = q.shape
    Hk = kc.shape[1]
    res = {n: torch.zeros(T, H, D, dtype=torch.float64) for n in ("out", "centred", "plain", "spread", "logit")}
    for b, (r0, nq, n) in enumerate(zip(first_row, n_new, n_keys)):
        if nq == 0 or n == 0:
            continue
        pos = torch.arange(n)
        k, v = ref.kv_read_int4(kc, vc, table, pos, torch.full_like(pos, b), D, torch.float32)
        k, v = k.double(), v.double()
        lo, hi = (f(v.unflatten(-1, (-1, 64)), -1, keepdim=True).expand(-1, -1, -1, 64).flatten(2) for f in (torch.amin, torch.amax))
        reach = hi - lo                                                    # at least scale |code - 8| for every value
        for h in range(H):
            kh, vh, wh = k[:, h // (H // Hk)], v[:, h // (H // Hk)], reach[:, h // (H // Hk)]
            qh = q[r0:r0 + nq, h].double()
            hidden = pos[None] > n - nq + torch.arange(nq)[:, None]
            p = torch.softmax((qh @ kh.T * scale).masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
            o = p @ vh
            res["out"][r0:r0 + nq, h] = o
            res["centred"][r0:r0 + nq, h] = p @ wh
            res["plain"][r0:r0 + nq, h] = p @ vh.abs()
            res["spread"][r0:r0 + nq, h] = torch.stack([(p[:, :, None] * (vh[None] - o[:, None]).abs()).sum(1)], 0)[0] if nq * n * D < 1 << 24 \
                else p @ vh.abs() + o.abs()
            res["logit"][r0:r0 + nq, h] = (qh.abs() @ kh.abs().T).masked_fill(hidden, 0).amax(-1, keepdim=True) * scale
    return res
