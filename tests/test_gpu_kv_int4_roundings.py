"""Attention over 4-bit pages held to the roundings that the kernels make (kv_int4_bounds.py): contexts of many parts, batches in
slices, queries that see nothing, values of any size."""
import math

import pytest
import torch

from kv_int4_bounds import attention, check
from kv_int4_util import filled, make_cache, random_rows, token_lists
from mythos_b200.ops import functional as F, native

pytestmark = pytest.mark.gpu


def _cu(new):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def _wide(table, tokens, page):
    wide = torch.full((table.shape[0], (tokens + page - 1) // page), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    return wide


def _queries(T, H, D, seed):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("H,Hk,D,lens,width", [
    (4, 1, 128, [40000], 300000),                                   # parts in more CTAs than the merge holds weights of
    (2, 1, 64, [34000, 20000, 1, 0, 700], 300000),
    (20, 5, 128, [2048, 2000, 1500, 2048, 33, 64, 1900, 2047], 0),
    (3, 3, 128, [6000, 1, 3000], 40000), (5, 1, 64, [5000, 31, 32, 33], 40000), (80, 1, 128, [500, 31], 40000),
    (8, 2, 128, [64 * i for i in range(40)], 40000), (8, 2, 128, [64 * i for i in range(40)], 0), (16, 2, 64, [900, 31000], 0),
    (8, 1, 128, [1100] * 32, 0)])
def test_decode(H, Hk, D, lens, width):
    kc, vc, table = filled(lens, Hk, D, 16, "cuda", seed=9)
    B, q = len(lens), _queries(len(lens), H, D, 9)
    want = attention(q, kc, vc, table, range(B), [1] * B, lens, 1 / math.sqrt(D))
    t = _wide(table, width, 16) if width else table
    check(F.paged_attn_decode_int4(q, kc, vc, t, torch.tensor(lens, dtype=torch.int32, device="cuda")), *want)
    native.check_status("cuda")


@pytest.mark.parametrize("H,Hk,D,new,old,width", [
    (8, 1, 128, [5, 0, 1, 4], [100, 40, 700, 0], 0), (6, 2, 128, [20, 3], [64, 2000], 40000), (4, 2, 64, [7] * 35, [i * 9 for i in range(35)], 40000),
    (4, 2, 128, [6, 3], [-4, 0], 0),                                # more new tokens than keys
    (8, 2, 128, [700, 0, 300], [300, 50, 0], 0), (6, 2, 128, [900, 33], [200, 1500], 0), (4, 4, 64, [1200, 1000, 5], [5, 0, 0], 0),
    (16, 8, 128, [513, 129, 700], [0, 1000, 255], 0), (5, 1, 64, [1000, 1, 1], [400, 2000, 0], 0), (2, 2, 128, [2500], [0], 0),
    (4, 2, 128, [900, 800], [-600, 0], 0),
    (32, 8, 128, [1] * 20 + [300], [1200 - 50 * i for i in range(20)] + [700], 2048),      # single tokens beside a portion
    (8, 8, 128, [130, 0, 70, 1, 200, 90, 33, 5, 260, 128], [700, 30, 0, 500, 90, 0, 5, 1000, 3, 400], 65536)])     # two slices
def test_new_tokens(H, Hk, D, new, old, width):
    lens = [a + b for a, b in zip(new, old)]
    kc, vc, table = filled(lens, Hk, D, 16, "cuda", seed=H + D)
    q, cu = _queries(sum(new), H, D, 8), _cu(new)
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    t = _wide(table, width, 16) if width else table
    got = F.paged_attn_prefill_int4(q, kc, vc, t, cu, torch.tensor(lens, dtype=torch.int32, device="cuda"), max(new), width or max(lens))
    check(got, *want)
    native.check_status("cuda")


@pytest.mark.parametrize("ks,vs", [(1e-30, 1e30), (20.0, 1e-20), (1e-3, 1e36), (1.0, 1e4), (1.0, 1e-30)])
@pytest.mark.parametrize("form", ["cluster", "line", "prompt"])
def test_values_of_any_size(ks, vs, form):
    H, Hk, D = 4, 2, 128
    lens = [1000, 700] if form == "prompt" else [300, 70]
    new = [900, 700] if form == "prompt" else [1, 1]
    kc, vc, table = make_cache(lens, Hk, D, 16, "cuda")
    pos, sid = token_lists([0, 0], lens, "cuda")
    k, v = random_rows(sum(lens), Hk, D, 11, "cuda")
    F.kv_append_int4((k.float() * ks).bfloat16(), (v.float() * vs).bfloat16(), kc, vc, table, pos, sid)
    q, cu, ctx = _queries(sum(new), H, D, 1), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    if form == "prompt":
        out = F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens))
    else:
        out = F.paged_attn_decode_int4(q, kc, vc, table if form == "cluster" else _wide(table, 40000, 16), ctx)
    check(out, *attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D)))
    native.check_status("cuda")
