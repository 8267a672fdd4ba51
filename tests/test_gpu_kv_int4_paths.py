"""The forms that attention over 4-bit pages takes by its sizes: stretches of a line of chunks, clusters, prompts."""
import math

import pytest
import torch

from kv_int4_util import filled, make_cache, oracle, random_rows, token_lists
from mythos_b200.ops import functional as F, native, reference as ref
from test_gpu_kv_int4 import HALF, _decode_bound, _prefill_bound, _same_bits

pytestmark = pytest.mark.gpu


def _widen(table, tokens, page):
    """The same table with room for ``tokens`` tokens a sequence: the sizes that a call is planned by."""
    wide = torch.full((table.shape[0] + 1, (tokens + page - 1) // page), -1, dtype=torch.int32, device=table.device)
    wide[: table.shape[0], : table.shape[1]] = table
    return wide


def _cu(new, device="cuda"):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=device)


def _ragged(B, most, seed):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, most + 1, (B,), generator=g).tolist()
    lens[0], lens[B // 2], lens[-1] = 0, most, 0
    return lens


@pytest.mark.parametrize("H,Hk,D,page,lens", [
    (8, 2, 128, 16, _ragged(40, 300, 1)), (2, 1, 64, 32, _ragged(70, 200, 2)), (4, 1, 128, 16, [33, 0, 64]), (8, 8, 64, 16, [1]),
    (80, 1, 128, 16, [500, 31]), (5, 1, 64, 16, _ragged(33, 1000, 3)), (32, 8, 128, 16, _ragged(66, 130, 4)), (3, 3, 128, 16, [6000, 1, 3000]),
    (8, 2, 128, 16, [0] * 40)])
def test_decode_in_stretches_against_64_bits(H, Hk, D, page, lens):
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=H)
    B = len(lens)
    q = torch.randn(B, H, D, generator=torch.Generator().manual_seed(D)).to(torch.bfloat16).cuda()
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    wide = _widen(table, 40000, page)                       # no cluster takes 1250 chunks
    out = F.paged_attn_decode_int4(q, kc, vc, wide, ctx)
    res = oracle(q, kc, vc, table, range(B), [1] * B, lens, 1.0 / math.sqrt(D))
    for got in (out, F.paged_attn_decode_int4(q, kc, vc, table, ctx)):
        off = (got.cpu().double() - res["out"]).abs()
        assert (off <= _decode_bound(res)).all(), float((off / _decode_bound(res)).max())
        assert not got[ctx == 0].any()
    for _ in range(3):
        assert _same_bits(F.paged_attn_decode_int4(q, kc, vc, wide, ctx), out)
    native.check_status("cuda")


@pytest.mark.parametrize("H,Hk,D,page,new,old", [
    (8, 1, 128, 16, [5, 0, 1, 4], [100, 40, 700, 0]), (4, 2, 64, 16, [7] * 35, [i * 9 for i in range(35)]), (6, 2, 128, 48, [20, 3], [64, 2000])])
def test_short_prompts_in_stretches_against_64_bits(H, Hk, D, page, new, old):
    lens = [a + b for a, b in zip(new, old)]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=H + D)
    T = sum(new)
    q = torch.randn(T + 2, H, D, generator=torch.Generator().manual_seed(D)).to(torch.bfloat16).cuda()
    cu, kv = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    res = oracle(q[:T], kc, vc, table, cu[:-1].tolist(), new, lens, 1.0 / math.sqrt(D))
    for t in (_widen(table, 40000, page), table):
        out = torch.full((T + 2, H, D), 3.0, device="cuda", dtype=torch.bfloat16)
        F.paged_attn_prefill_int4(q, kc, vc, t, cu, kv, max(new), max(lens), out=out)
        off = (out[:T].cpu().double() - res["out"]).abs()
        assert (off <= _decode_bound(res)).all(), float((off / _decode_bound(res)).max())
        assert bool((out[T:] == 3.0).all())
        again = torch.full_like(out, 3.0)
        F.paged_attn_prefill_int4(q, kc, vc, t, cu, kv, max(new), max(lens), out=again)
        assert _same_bits(again, out)
    native.check_status("cuda")


# more than 64 query columns and more chunks than eight per resident warp: the prompt kernels. Groups that divide 128 and not,
# items whole per CTA (up to 148 items of up to 12 tiles) and in stretches
PROMPTS = [(8, 2, 128, 16, [700, 0, 300], [300, 50, 0]), (6, 2, 128, 48, [900, 33], [200, 1500]), (4, 4, 64, 16, [1200, 1000, 5], [5, 0, 0]),
           (16, 2, 64, 32, [600], [900]), (4, 1, 128, 16, [500], [3000]), (16, 8, 128, 16, [513, 129, 700], [0, 1000, 255]),
           (5, 1, 64, 16, [1000, 1, 1], [400, 2000, 0]), (2, 2, 128, 16, [2500], [0])]


@pytest.mark.parametrize("H,Hk,D,page,new,old", PROMPTS)
def test_prompts_against_64_bits(H, Hk, D, page, new, old):
    lens = [a + b for a, b in zip(new, old)]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=H + D)
    T = sum(new)
    q = torch.randn(T + 3, (H + 1) * D, generator=torch.Generator().manual_seed(H)).to(torch.bfloat16).cuda()[:, : H * D].unflatten(-1, (H, D))
    cu, kv = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((T + 3, H, D), 3.0, device="cuda", dtype=torch.bfloat16)
    F.paged_attn_prefill_int4(q, kc, vc, table, cu, kv, max(new), max(lens), out=out)
    res = oracle(q[:T], kc, vc, table, cu[:-1].tolist(), new, lens, 1.0 / math.sqrt(D))
    off = (out[:T].cpu().double() - res["out"]).abs()
    assert (off <= _prefill_bound(res)).all(), float((off / _prefill_bound(res)).max())
    assert float(off.norm() / res["out"].norm()) < 5e-3     # as a few independent roundings of 2^-9
    assert bool((out[T:] == 3.0).all())
    again = torch.full_like(out, 3.0)
    F.paged_attn_prefill_int4(q, kc, vc, table, cu, kv, max(new), max(lens), out=again)
    assert _same_bits(again, out)
    native.check_status("cuda")


def test_a_bad_token_in_a_prompt_reaches_only_the_queries_that_see_it():
    H, Hk, D, page, new = 4, 2, 128, 16, 800
    lens = [1000, 900]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=3)
    pos = torch.tensor([990, 400], dtype=torch.int32, device="cuda")
    k, v = random_rows(2, Hk, D, 9, "cuda")
    v[0, 0, 3] = math.inf
    k[1, 1, 70] = math.nan
    F.kv_append_int4(k, v, kc, vc, table, pos, torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    q = torch.randn(2 * new, H, D, device="cuda").to(torch.bfloat16)
    out = F.paged_attn_prefill_int4(q, kc, vc, table, _cu([new, new]), torch.tensor(lens, dtype=torch.int32, device="cuda"), new, 1000)
    want = torch.zeros(2 * new, H, dtype=torch.bool, device="cuda")
    want[790:800, :2] = True                                # queries at 990 .. 999 of the first sequence
    want[new + 300:, 2:] = True                             # at 400 .. 899 of the second
    assert torch.equal((~out.isfinite()).any(-1), want)
    native.check_status("cuda")


@pytest.mark.parametrize("ks,vs", [(1e-30, 1e30), (20.0, 1e-20), (1e-3, 1e36), (1.0, 1e4)])
@pytest.mark.parametrize("form", ["cluster", "line", "prompt"])
def test_values_of_any_size(ks, vs, form):
    H, Hk, D, page = 4, 2, 128, 16
    lens = [1000, 700] if form == "prompt" else [300, 70]
    new = [900, 700] if form == "prompt" else [1, 1]
    kc, vc, table = make_cache(lens, Hk, D, page, "cuda")
    pos, sid = token_lists([0, 0], lens, "cuda")
    k, v = random_rows(sum(lens), Hk, D, 11, "cuda")
    F.kv_append_int4((k.float() * ks).bfloat16(), (v.float() * vs).bfloat16(), kc, vc, table, pos, sid)
    T = sum(new)
    q = torch.randn(T, H, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if form == "prompt":
        out = F.paged_attn_prefill_int4(q, kc, vc, table, _cu(new), ctx, max(new), max(lens))
    else:
        out = F.paged_attn_decode_int4(q, kc, vc, table if form == "cluster" else _widen(table, 40000, page), ctx)
    res = oracle(q, kc, vc, table, _cu(new)[:-1].tolist(), new, lens, 1.0 / math.sqrt(D))
    res = {n: t if n == "logit" else t / vs for n, t in res.items()}        # (the bounds end with an absolute 1e-6, taken off here)
    bound = (_prefill_bound if form == "prompt" else _decode_bound)(res) - 1e-6
    off = (out.cpu().double() / vs - res["out"]).abs()
    assert out.isfinite().all() and (off <= bound).all(), float((off / bound).max())
    native.check_status("cuda")


@pytest.mark.parametrize("form", ["line", "prompt"])
def test_captured_calls_on_two_streams_share_no_scratch(form):
    H, Hk, D, page = 8, 2, 128, 16
    new, old = ([1] * 40, [5 * i for i in range(40)]) if form == "line" else ([700, 33], [300, 2000])
    lens = [a + b for a, b in zip(new, old)]
    sets = []
    for seed in (1, 2):
        kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=seed)
        q = torch.randn(sum(new), H, D, device="cuda").to(torch.bfloat16)
        ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cu, wide = _cu(new), _widen(table, 40000, page)
        if form == "line":
            sets.append(lambda q=q, kc=kc, vc=vc, wide=wide, ctx=ctx: F.paged_attn_decode_int4(q, kc, vc, wide, ctx))
        else:
            sets.append(lambda q=q, kc=kc, vc=vc, t=table, cu=cu, ctx=ctx: F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, 700, max(lens)))
    want = [f() for f in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    eager = []
    for i in range(10):
        for o in outs:
            o.fill_(5.0)
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager.append(sets[i & 1]())                         # a third call beside them
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for o, w in zip(outs, want):
            assert _same_bits(o, w)
        assert _same_bits(eager[-1], want[i & 1])
    native.check_status("cuda")


def test_lengths_that_the_call_did_not_announce_are_reported():
    H, Hk, D, page = 4, 2, 128, 16
    kc, vc, table = filled([64, 40], Hk, D, page, "cuda", seed=4)
    q = torch.randn(40, H, D, device="cuda").to(torch.bfloat16)
    ctx = torch.tensor([64, 40], dtype=torch.int32, device="cuda")
    cu = _cu([30, 10])
    for t in (table, _widen(table, 40000, page)):           # more new tokens than announced: those rows stay as they were
        out = torch.full_like(q, 3.0)
        F.paged_attn_prefill_int4(q, kc, vc, t, cu, ctx, 8, 64, out=out)
        with pytest.raises(RuntimeError, match="status 2"):
            native.check_status("cuda")
        assert bool((out[8:30] == 3.0).all()) and not bool((out[:8] == 3.0).all(-1).any())
    # lengths that no cache can hold end all the same, and reach no other sequence
    whole = F.paged_attn_decode_int4(q[:2], kc, vc, table, ctx)
    for t in (table, _widen(table, 40000, page)):
        for bad in (2 ** 31 - 1, 2 ** 30):
            out = F.paged_attn_decode_int4(q[:2], kc, vc, t, torch.tensor([64, bad], dtype=torch.int32, device="cuda"))
            with pytest.raises(RuntimeError, match="status 2"):
                native.check_status("cuda")
            assert float((out[0].float() - whole[0].float()).abs().max()) <= 2 * HALF * float(whole[0].abs().max())
        out = F.paged_attn_decode_int4(q[:2], kc, vc, t, torch.tensor([64, -5], dtype=torch.int32, device="cuda"))
        native.check_status("cuda")
        assert not out[1].any()


def test_a_prompt_longer_than_announced_is_reported():
    H, Hk, D, page = 8, 2, 128, 16
    kc, vc, table = filled([1300], Hk, D, page, "cuda", seed=4)
    q = torch.randn(1300, H, D, device="cuda").to(torch.bfloat16)
    ctx = torch.tensor([1300], dtype=torch.int32, device="cuda")
    F.paged_attn_prefill_int4(q, kc, vc, table, _cu([1300]), ctx, 1300, 700)
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    out = torch.full_like(q, 3.0)
    F.paged_attn_prefill_int4(q, kc, vc, table, _cu([1300]), ctx, 700, 1300, out=out)
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    assert bool((out[768:] == 3.0).all())


def test_pages_behind_two_gibibytes():
    H, Hk, D, page = 32, 8, 128, 64
    lens, new = [700, 130], [600, 100]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=6)
    n = (1 << 31) // kc[0].numel() + 200
    far = table + (n - kc.shape[0])
    far[table < 0] = -1
    kf, vf = (torch.empty(n, *kc.shape[1:], dtype=torch.uint8, device="cuda") for _ in range(2))
    pos, sid = token_lists([0] * 2, lens, "cuda")
    k, v = random_rows(sum(lens), Hk, D, 7, "cuda")         # (the rows that filled() wrote)
    F.kv_append_int4(k, v, kf, vf, far, pos, sid)
    assert torch.equal(kf[far[0, 0]], kc[table[0, 0]]) and torch.equal(vf[far[1, 1]], vc[table[1, 1]])
    for a, b in zip(F.kv_read_int4(kf, vf, far, pos, sid, D), F.kv_read_int4(kc, vc, table, pos, sid, D)):
        assert _same_bits(a, b)
    q = torch.randn(sum(new), H, D, device="cuda").to(torch.bfloat16)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = _cu(new)
    for t, f in ((table, far), (_widen(table, 40000, page), _widen(far, 40000, page))):
        assert _same_bits(F.paged_attn_decode_int4(q[:2], kc, vc, t, ctx), F.paged_attn_decode_int4(q[:2], kf, vf, f, ctx))
    assert _same_bits(F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, 600, 700), F.paged_attn_prefill_int4(q, kf, vf, far, cu, ctx, 600, 700))
    native.check_status("cuda")


def test_a_batch_whose_images_do_not_fit_at_once():
    """Ten sequences announced at up to 65536 keys: images of 2.7 GB, dealt with eight sequences at a time."""
    H, Hk, D, page, most = 8, 8, 128, 16, 65536
    new, old = [130, 0, 70, 1, 200, 90, 33, 5, 260, 128], [700, 30, 0, 500, 90, 0, 5, 1000, 3, 400]
    lens = [a + b for a, b in zip(new, old)]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=8)
    wide = _widen(table, most, page)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    cu, kv = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    res = oracle(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1.0 / math.sqrt(D))
    out = F.paged_attn_prefill_int4(q, kc, vc, wide, cu, kv, max(new), most)
    off = (out.cpu().double() - res["out"]).abs()
    assert (off <= _prefill_bound(res)).all(), float((off / _prefill_bound(res)).max())
    native.check_status("cuda")


@pytest.mark.parametrize("form", ["few", "prompt"])
def test_queries_that_see_nothing_get_zeros(form):
    H, Hk, D, page = 4, 2, 128, 16
    new, lens = ([6, 3], [2, 3]) if form == "few" else ([900, 800], [300, 800])      # more new tokens than keys
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=8)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    cu, kv = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    res = oracle(q, kc, vc, table, cu[:-1].tolist(), new, lens, 1.0 / math.sqrt(D))
    for t in (table, _widen(table, 40000, page)):
        out = torch.full_like(q, 3.0)
        F.paged_attn_prefill_int4(q, kc, vc, t, cu, kv, max(new), max(lens), out=out)
        off = (out.cpu().double() - res["out"]).abs()
        assert (off <= _prefill_bound(res)).all(), float((off / _prefill_bound(res)).max())
        assert not out[: new[0] - lens[0]].any()
    native.check_status("cuda")


@pytest.mark.parametrize("form", ["cluster", "line", "prompt"])
def test_a_query_that_is_not_finite_reaches_its_own_row_only_and_results_may_replace_the_queries(form):
    H, Hk, D, page = 4, 2, 128, 16
    new = [800, 700] if form == "prompt" else [1, 1]
    lens = [900, 700]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=5)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    cu, ctx = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")

    def call(q, out=None):
        if form == "prompt":
            return F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens), out=out)
        return F.paged_attn_decode_int4(q, kc, vc, table if form == "cluster" else _widen(table, 40000, page), ctx, out=out)

    want = call(q)
    bad = q.clone()
    bad[0, 1, 5] = math.nan
    bad[1, 3, 60] = math.inf
    got = call(bad)
    odd = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
    odd[0, 1] = odd[1, 3] = True
    assert torch.equal((~got.isfinite()).any(-1), odd) and _same_bits(got[~odd], want[~odd])
    assert _same_bits(call(q, out=q), want)
    native.check_status("cuda")


def test_a_context_without_any_page_gives_zeros_and_is_reported():
    H, Hk, D, page = 4, 2, 128, 16
    kc, vc, table = filled([64, 40], Hk, D, page, "cuda", seed=4)
    q = torch.randn(2, H, D, device="cuda").to(torch.bfloat16)
    ctx = torch.tensor([64, 40], dtype=torch.int32, device="cuda")
    table[0] = -1
    for t in (table, _widen(table, 40000, page)):
        out = F.paged_attn_decode_int4(q, kc, vc, t, ctx)
        with pytest.raises(RuntimeError, match="status 2"):
            native.check_status("cuda")
        assert not out[0].any() and out[1].any()
    nothing = F.paged_attn_decode_int4(q, kc[:0], vc[:0], table[:, :0], ctx)         # no pages, no columns
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    assert not nothing.any()


@pytest.mark.parametrize("D,form", [(128, "prompt"), (64, "prompt"), (128, "stretches"), (128, "few")])
def test_keys_without_a_page_are_seen_by_no_query(D, form):
    H, Hk, page = 4, 2, 16
    new, lens = {"prompt": ([700, 300], [900, 700]), "stretches": ([1000], [3000]), "few": ([6, 3], [200, 90])}[form]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=6)
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).cuda()
    cu, kv = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    # the first sixteen tokens, whole 128-token tiles, one in the middle of a tile, the last
    gaps, last = table.clone(), (lens[0] - 1) // page
    gone = sorted({0, 5, last} | ({*range(8, 16), 17, 19, 40} if form != "few" else set()))
    gaps[0, gone] = -1
    got = F.paged_attn_prefill_int4(q, kc, vc, gaps, cu, kv, max(new), max(lens))
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    whole = F.paged_attn_prefill_int4(q, kc, vc, table, cu, kv, max(new), max(lens))
    native.check_status("cuda")
    assert _same_bits(got[new[0]:], whole[new[0]:])         # the other sequence
    # attention over the tokens that are left: they move up, the queries keep what they see
    left = [t for t in range(lens[0]) if t // page not in gone]
    at = torch.tensor(left)
    k, v = (x.double() for x in ref.kv_read_int4(kc.cpu(), vc.cpu(), table.cpu(), at, torch.zeros_like(at), D, torch.float32))
    hidden = at > lens[0] - new[0] + torch.arange(new[0])[:, None]
    for h in range(H):
        qh = q[: new[0], h].cpu().double()
        kh, vh = k[:, h // 2], v[:, h // 2]
        p = torch.softmax((qh @ kh.T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
        o = p @ vh
        # the same roundings as everywhere, with |v| + |o| in place of |v - o|
        res = {"out": o, "plain": p @ vh.abs(), "centred": p @ vh.abs() + o.abs(), "spread": p @ vh.abs() + o.abs(),
               "logit": (qh.abs() @ kh.abs().T).masked_fill(hidden, 0).amax(-1, keepdim=True) / math.sqrt(D)}
        off = (got[: new[0], h].cpu().double() - o).abs()
        assert (off <= _prefill_bound(res)).all(), float((off / _prefill_bound(res)).max())
        assert float(off.norm() / o.norm()) < 5e-3


def test_fused_epilogue_refuses_what_its_stores_cannot_reach():
    C = native.require()
    H, Hk, D, page = 4, 2, 128, 16
    bytes_ = 3 * Hk * page * F.kv4_token_bytes(D)
    flat = torch.zeros(2, bytes_ + 16, device="cuda", dtype=torch.uint8)
    kc, vc = (x[:bytes_].view(3, Hk, -1) for x in flat)
    table = torch.arange(2, device="cuda", dtype=torch.int32)[:, None]
    acc = torch.randn(2, (H + 2 * Hk) * D, device="cuda")
    pos, sid = torch.zeros(2, device="cuda", dtype=torch.int32), torch.arange(2, device="cuda", dtype=torch.int32)
    q = torch.empty(2, H, D, device="cuda", dtype=torch.bfloat16)
    for off in (1, 2, 4, 8):
        odd = flat[0, off:bytes_ + off].view(3, Hk, -1)
        for caches in ((odd, vc), (kc, odd)):
            with pytest.raises(ValueError, match="aligned"):
                C.qkv_rope_append(acc, pos, sid, table, q, *caches, 10000.0)
    assert not flat.any()
    C.qkv_rope_append(acc, pos, sid, table, q, kc, vc, 10000.0)
    assert kc[:2].any() and not kc[2].any()


@pytest.mark.parametrize("H,Hk,D,lens,width", [
    (4, 1, 128, [40000], 300000),                                  # parts in more CTAs than the merge holds weights of
    (2, 1, 64, [34000, 20000, 1, 0, 700], 300000),
    (20, 5, 128, [2048, 2000, 1500, 2048, 33, 64, 1900, 2047], 0),  # 40 clusters: of fewer CTAs than would fit by number
    (8, 1, 128, [1100] * 32, 0), (16, 2, 128, [900, 31000], 0)])
def test_decode_over_many_parts_and_cluster_sizes(H, Hk, D, lens, width):
    kc, vc, table = filled(lens, Hk, D, 16, "cuda", seed=9)
    B = len(lens)
    q = torch.randn(B, H, D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if width:
        table = _widen(table, width, 16)
    out = F.paged_attn_decode_int4(q, kc, vc, table, ctx)
    res = oracle(q, kc, vc, table, range(B), [1] * B, lens, 1.0 / math.sqrt(D))
    off = (out.cpu().double() - res["out"]).abs()
    assert (off <= _decode_bound(res)).all(), float((off / _decode_bound(res)).max())
    assert not out[ctx == 0].any() and _same_bits(F.paged_attn_decode_int4(q, kc, vc, table, ctx), out)
    native.check_status("cuda")


@pytest.mark.parametrize("form", ["cluster", "line", "several"])
def test_a_heads_bits_do_not_depend_on_its_neighbours(form):
    H, Hk, D, page = 8, 2, 128, 16
    lens = [3000, 777]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=2)
    new = [3, 2] if form == "several" else [1, 1]
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    cu, ctx = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")

    def call(q):
        if form == "several":
            return F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens))
        return F.paged_attn_decode_int4(q, kc, vc, table if form == "cluster" else _widen(table, 400000, page), ctx)

    want = call(q)
    other = q.clone()
    other[:, ::2] *= 40                                     # every second head's maximum moves all the time
    got = call(other)
    assert _same_bits(got[:, 1::2], want[:, 1::2]) and not _same_bits(got[:, ::2], want[:, ::2])
    native.check_status("cuda")


@pytest.mark.parametrize("form", ["line", "prompt"])
def test_a_threads_first_call_may_be_captured(form):
    import threading

    H, Hk, D, page = 8, 2, 128, 16
    new, lens = ([800, 700], [900, 700]) if form == "prompt" else ([1, 1], [900, 700])
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=1)
    q = torch.randn(sum(new), H, D, device="cuda").to(torch.bfloat16)
    cu, ctx = _cu(new), torch.tensor(lens, dtype=torch.int32, device="cuda")
    wide = _widen(table, 40000, page)
    native.status_word(q.device)
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens)) if form == "prompt" else \
                    F.paged_attn_decode_int4(q, kc, vc, wide, ctx)
            g.replay()
            torch.cuda.synchronize()
            got.append(out.clone())
        except Exception as e:
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert isinstance(got[0], torch.Tensor), got[0]
    want = F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, max(new), max(lens)) if form == "prompt" else \
        F.paged_attn_decode_int4(q, kc, vc, wide, ctx)
    assert _same_bits(got[0], want)
    native.check_status("cuda")
