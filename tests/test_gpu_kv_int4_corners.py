"""Corners of attention over 4-bit pages: first tiles that hold nothing, value sizes that change along a context, tokens of any size that
a query does not see, lengths that were not announced."""
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


def _written(k, v, lens, Hk, D, seed=0):
    kc, vc, table = make_cache(lens, Hk, D, 16, "cuda", seed=seed)
    pos, sid = token_lists([0] * len(lens), lens, "cuda")
    F.kv_append_int4(k.to(torch.bfloat16).contiguous(), v.to(torch.bfloat16).contiguous(), kc, vc, table, pos, sid)
    return kc, vc, table


def _queries(T, H, D, seed=8):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


# new tokens, keys, tiles of 128 keys without pages: whole items per CTA, and stretches that begin at any tile
HIDDEN = [([700, 300], [900, 700], [0]), ([700, 300], [900, 700], [0, 1]), ([2500], [2500], [0, 1]), ([1000], [3000], [0, 1, 3, 4, 5, 8, 10, 11, 12, 20])]


@pytest.mark.parametrize("size,offset", [(1.0, 0.0), (0.01, -8.0), (1e-4, -4.0), (1e-3, 12.0)])
@pytest.mark.parametrize("new,lens,tiles", HIDDEN)
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_without_pages_leave_the_rest_as_exact(D, new, lens, tiles, size, offset):
    H, Hk = 4, 2
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    q = _queries(sum(new), H, D)
    k[..., 0], q[..., 0] = 4.0, offset * math.sqrt(D) / 4       # moves every score by the offset
    kc, vc, table = _written(k, v.float() * size, lens, Hk, D)
    for t in tiles:
        table[0, 8 * t:8 * t + 8] = -1
    cu, ctx = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens))
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    check(got, *attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D)))


# sizes of the values, 128 tokens after 128
SIZES = [[1e-35, 4.0], [1e-35, 1e-3, 4.0, 1e-20, 1.0], [2.0 ** (20 * (-1) ** i) for i in range(30)], [1.0] + [1e-36] * 3 + [1e-12] * 9]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("new,lens", [([700, 300], [900, 700]), ([2500], [2500]), ([1000], [3000]), ([1, 1], [3000, 700])])
@pytest.mark.parametrize("D", [64, 128])
def test_value_sizes_that_change_along_a_context(D, new, lens, sizes):
    H, Hk = 4, 2
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    size = torch.cat([torch.tensor(sizes)[(torch.arange(n) // 128).clamp_max(len(sizes) - 1)] for n in lens]).cuda()
    kc, vc, table = _written(k, v.float() * size[:, None, None], lens, Hk, D)
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    for t in (table, _wide(table, 40000, 16)):
        check(F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, max(new), max(lens)), *want)
    native.check_status("cuda")


@pytest.mark.parametrize("width", [0, 40000])
def test_new_tokens_of_a_call_that_announces_none_are_reported(width):
    H, Hk, D = 4, 2, 128
    kc, vc, table = filled([64, 40], Hk, D, 16, "cuda", seed=4)
    t = _wide(table, width, 16) if width else table
    q, ctx = _queries(9, H, D), torch.tensor([64, 40], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 3.0)
    F.paged_attn_prefill_int4(q, kc, vc, t, _cu([5, 4]), ctx, 0, 64, out=out)
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    F.paged_attn_prefill_int4(q, kc, vc, t, _cu([0, 0]), ctx, 0, 64, out=out)       # none: nothing to report
    native.check_status("cuda")
    assert bool((out == 3.0).all())


@pytest.mark.parametrize("new,lens,most_new,most", [
    ([5, 4], [64, 40], 5, 63), ([5, 4], [64, 40], 4, 64), ([700], [700], 700, 699), ([700], [700], 699, 700), ([1000], [3000], 1000, 2999),
    ([1000], [3000], 999, 3000)])
@pytest.mark.parametrize("width", [0, 40000])
def test_one_token_more_than_announced_is_reported(new, lens, most_new, most, width):
    H, Hk, D = 4, 2, 128
    kc, vc, table = filled(lens, Hk, D, 16, "cuda", seed=4)
    t = _wide(table, width, 16) if width else table
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, max(new), max(lens))
    native.check_status("cuda")
    F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, most_new, most)
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")


def _one_large(D, Hk, lens, at, size, score):
    """Rows whose token ``at`` of every sequence has values ``size`` times larger and a score lower by ``score``."""
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    k[..., 0] = 0.0
    first = 0
    for n in lens:
        if at < n:
            v[first + at] = (v[first + at].float() * size).to(torch.bfloat16)
            k[first + at, :, 0] = -score * math.sqrt(D) / 8
        first += n
    return k, v


@pytest.mark.parametrize("size", [1e4, 1e9, 1e30])
@pytest.mark.parametrize("D,lens,at", [(128, [300, 70], 20), (64, [300, 70], 65), (128, [3000, 33], 32)])
def test_decode_beside_a_large_token_that_hardly_counts(D, lens, at, size):
    H, Hk = 4, 2
    k, v = _one_large(D, Hk, lens, at, size, 100.0)            # a weight of e^-100
    kc, vc, table = _written(k, v, lens, Hk, D)
    q = _queries(2, H, D)
    q[..., 0] = 8.0
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = attention(q, kc, vc, table, [0, 1], [1, 1], lens, 1 / math.sqrt(D))
    for t in (table, _wide(table, 40000, 16)):
        check(F.paged_attn_decode_int4(q, kc, vc, t, ctx), *want)
    native.check_status("cuda")


@pytest.mark.parametrize("ks,vs", [(1.0, 1e9), (1.0, 1e30), (1e30, 1.0), (1e30, 1e30)])
def test_a_few_queries_are_not_reached_by_a_large_token_behind_them(ks, vs):
    H, Hk, D, lens, new = 4, 2, 128, [300, 70], [6, 5]
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    last = [299, 369]
    small = _written(k, v, lens, Hk, D)
    k[last], v[last] = (k[last].float() * ks).to(torch.bfloat16), (v[last].float() * vs).to(torch.bfloat16)
    large = _written(k, v, lens, Hk, D)
    rows = [r for r in range(sum(new)) if r not in (5, 10)]     # the others see neither
    want = attention(q, *small, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    for width in (0, 40000):
        t = _wide(large[2], width, 16) if width else large[2]
        got = F.paged_attn_prefill_int4(q, large[0], large[1], t, cu, ctx, 6, 300)
        check(got[rows], *(w[rows] for w in want))
    native.check_status("cuda")


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-6])
@pytest.mark.parametrize("new,lens", [([700, 300], [900, 700]), ([2500], [2500]), ([1000], [3000]), ([1, 1], [3000, 700])])
def test_128_tokens_whose_values_are_zero(new, lens, size):
    H, Hk, D = 4, 2, 128
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    v = v.float() * size
    for first in [0, lens[0]] if len(lens) > 1 else [0]:
        v[first + 256:first + 384] = 0.0
    kc, vc, table = _written(k, v, lens, Hk, D)
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    for t in (table, _wide(table, 40000, 16)):
        check(F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, max(new), max(lens)), *want)
    native.check_status("cuda")


@pytest.mark.parametrize("ks,vs", [(1.0, 1e4), (1.0, 1e9), (1.0, 1e30), (1e4, 1.0), (1e30, 1.0), (1e30, 1e30)])
@pytest.mark.parametrize("D,new,lens", [(128, [700, 300], [900, 700]), (64, [2500], [2500]), (128, [1000], [3000])])
def test_a_prompt_is_not_reached_by_a_large_token_behind_it(D, new, lens, ks, vs):
    H, Hk = 4, 2
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    at = lens[0] - 200                                          # of the first sequence; its last 200 queries see the token
    k[at], v[at] = (k[at].float() * ks).to(torch.bfloat16), (v[at].float() * vs).to(torch.bfloat16)
    kc, vc, table = _written(k, v, lens, Hk, D)
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    got = F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens))
    # (a key of 1e30 gives scores whose difference from others no 32-bit number holds: what sees it is only finite)
    rows = [r for r in range(sum(new)) if not new[0] - 200 <= r < new[0]] if ks > 1e4 else list(range(sum(new)))
    assert bool(got.isfinite().all())
    check(got[rows], *(w[rows] for w in want))
    native.check_status("cuda")


@pytest.mark.parametrize("size", [1e4, 1e9, 1e30])
@pytest.mark.parametrize("D,new,lens", [(128, [700, 300], [900, 700]), (64, [2500], [2500]), (128, [1000], [3000])])
def test_a_prompt_beside_a_large_token_that_hardly_counts(D, new, lens, size):
    H, Hk = 4, 2
    k, v = _one_large(D, Hk, lens, 20, size, 100.0)
    kc, vc, table = _written(k, v, lens, Hk, D)
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q[..., 0] = 8.0
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    check(F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens)), *want)
    native.check_status("cuda")


@pytest.mark.parametrize("D", [64, 128])
def test_tokens_of_every_size_side_by_side(D):
    H, Hk, new, lens = 4, 2, [900, 800], [1500, 800]
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    size = torch.exp2(torch.randint(-40, 41, (sum(lens), 1, 1), generator=torch.Generator().manual_seed(2)).float()).cuda()
    kc, vc, table = _written(k * size.clamp(1e-6, 1.0), v.float() * size.flip(0), lens, Hk, D)
    for t in range(0, 12, 3):
        table[0, 8 * t + 3] = -1                                # and gaps among them
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens))
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    check(got, *attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D)))


def test_large_scores_beside_a_token_of_another_size():
    """Scores around 1e5 are off by 2^-7 in 32 bits; weights and their sum have to be off together."""
    H, Hk, D, lens = 4, 2, 128, [900]
    k, v = random_rows(900, Hk, D, 6, "cuda")
    k[..., 0] = 0.0
    k[::7, :, 0] = 10.0                                         # every seventh key far above the others
    v = v.float()
    v[5::128] *= 1e6
    kc, vc, table = _written(k, v, lens, Hk, D)
    q = torch.zeros(700, H, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1e5
    want = attention(q, kc, vc, table, [0], [700], lens, 1 / math.sqrt(D))
    check(F.paged_attn_prefill_int4(q, kc, vc, table, _cu([700]), torch.tensor(lens, dtype=torch.int32, device="cuda"), 700, 900), *want)
    native.check_status("cuda")


# further apart than 32-bit numbers go below one
FAR = [[1e-35, 1e10], [1e30, 1e-35], [1e-35, 1e30, 1e-30, 1e20, 1.0], [1e-30, 0.0, 1e25, 1e-30]]


@pytest.mark.parametrize("sizes", FAR)
@pytest.mark.parametrize("new,lens", [([700, 300], [900, 700]), ([2500], [2500]), ([1000], [3000]), ([1, 1], [3000, 700]), ([6, 2], [600, 300])])
@pytest.mark.parametrize("D", [64, 128])
def test_value_sizes_further_apart_than_32_bits_go(D, new, lens, sizes):
    H, Hk = 4, 2
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    size = torch.cat([torch.tensor(sizes)[(torch.arange(n) // 128).clamp_max(len(sizes) - 1)] for n in lens]).cuda()
    kc, vc, table = _written(k, v.float() * size[:, None, None], lens, Hk, D)
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    for t in (table, _wide(table, 40000, 16)):
        check(F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, max(new), max(lens)), *want)
    native.check_status("cuda")


@pytest.mark.parametrize("size", [1e33, 1e35, 1e37, 5e37])
@pytest.mark.parametrize("new,lens", [([1, 1], [3000, 700]), ([6, 2], [600, 300]), ([700, 300], [900, 700])])
@pytest.mark.parametrize("D", [64, 128])
def test_values_near_the_largest_there_are(D, new, lens, size):
    H, Hk = 4, 2
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    k[..., 0] = torch.arange(sum(lens), device="cuda")[:, None].remainder(97) / 8        # scores that rise again and again
    kc, vc, table = _written(k, v.float().clamp(-3, 3) * size, lens, Hk, D)
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q[..., 0] = 4.0
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    for t in (table, _wide(table, 40000, 16)):
        check(F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, max(new), max(lens)), *want)
    native.check_status("cuda")


@pytest.mark.parametrize("score", [10.0, 30.0, 60.0])
@pytest.mark.parametrize("new,lens", [([1, 1], [3000, 700]), ([700, 300], [900, 700]), ([2500], [2500])])
@pytest.mark.parametrize("D", [64, 128])
def test_a_token_of_zeros_that_takes_nearly_all_the_weight(D, new, lens, score):
    H, Hk = 4, 2
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    k[..., 0] = 0.0
    first = 0
    for n in lens:
        for at in (3, 400):
            v[first + at] = 0.0
            k[first + at, :, 0] = score * math.sqrt(D) / 8
        first += n
    kc, vc, table = _written(k, v, lens, Hk, D)
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q[..., 0] = 8.0
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    check(F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens)), *want)
    native.check_status("cuda")


@pytest.mark.parametrize("below", [2.0, 6.0, 10.0])
@pytest.mark.parametrize("new,lens", [([1, 1], [3000, 700]), ([6, 2], [600, 300]), ([700, 300], [900, 700]), ([1000], [3000])])
def test_small_weights_beside_the_largest_values_count_in_the_sum(new, lens, below):
    H, Hk, D = 4, 2, 128
    k, v = random_rows(sum(lens), Hk, D, 6, "cuda")
    v = v.float() * 1e-10
    k[..., 0] = 0.0
    first = 0
    for n in lens:                                              # a token of 1e37, scores of the others lower by `below`
        v[first + 20] *= 1e23
        v[first + 20] *= 1e24
        k[first + 20, :, 0] = below * math.sqrt(D) / 8
        first += n
    k[..., 1:] *= 0.1
    kc, vc, table = _written(k, v, lens, Hk, D)
    q, cu, ctx = _queries(sum(new), H, D), _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q[..., 0] = 8.0
    want = attention(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1 / math.sqrt(D))
    for t in (table, _wide(table, 40000, 16)):
        check(F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, max(new), max(lens)), *want)
    native.check_status("cuda")
