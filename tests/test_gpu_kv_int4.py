"""4-bit paged KV cache on the GPU: bytes against the format's definition, attention against 64 bits."""
import math

import pytest
import torch

from kv_int4_util import filled, make_cache, oracle, random_rows, token_lists
from mythos_b200.ops import functional as F, native, reference as ref

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8      # half a step of bf16, relative to the value


def _same_bits(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("Hk,lens", [(1, [1]), (3, [17, 1, 40]), (8, [130, 16])])
def test_append_writes_the_formats_bytes_and_read_returns_its_values(D, page, Hk, lens):
    kc, vc, table = make_cache(lens, Hk, D, page, "cuda", seed=D + page)
    kr, vr, tr = kc.cpu(), vc.cpu(), table.cpu()
    pos, sid = token_lists([0] * len(lens), lens, "cuda")
    T = sum(lens)
    k, v = random_rows(T, Hk, D, 5, "cuda")
    k[0, 0] = 1.25                                  # one value: scale 0
    v[T - 1, Hk - 1, : D // 2] = 0
    k[T // 2, 0, :4] = torch.tensor([3e38, -3e38, 1e-38, 0.0])     # a range beyond fp32
    order = torch.randperm(T, device="cuda")        # any order of tokens, rows that are views of a wider tensor
    wide = torch.empty(T, 2 * Hk * D + 8, device="cuda", dtype=torch.bfloat16)
    kw, vw = wide[:, : Hk * D].unflatten(-1, (Hk, D)), wide[:, Hk * D + 8:].unflatten(-1, (Hk, D))
    kw.copy_(k[order])
    vw.copy_(v[order])
    F.kv_append_int4(kw, vw, kc, vc, table, pos[order].contiguous(), sid[order].contiguous())
    ref.kv_append_int4(k.cpu(), v.cpu(), kr, vr, tr, pos.cpu(), sid.cpu())
    assert torch.equal(kc.cpu(), kr) and torch.equal(vc.cpu(), vr)          # stale bytes elsewhere untouched
    got = F.kv_read_int4(kc, vc, table, pos, sid, D)
    want = ref.kv_read_int4(kr, vr, tr, pos.cpu(), sid.cpu(), D)
    for g, w, x in zip(got, want, (k, v)):
        assert torch.equal(g.cpu().nan_to_num(7.0), w.nan_to_num(7.0)) and torch.equal(g.cpu().isnan(), w.isnan())
        # half a step of the code, the scale's rounding (15 codes of 2^-9), the result's rounding
        grp = x.double().unflatten(-1, (-1, 64))
        step = ((grp.amax(-1) - grp.amin(-1)) / 15).repeat_interleave(64, -1)
        off = (g.double() - x.double()).abs()
        bad = g.isnan() | (step > 1e37)
        assert (off <= 0.5 * step * (1 + HALF) + 7.5 * step * HALF + HALF * x.double().abs().amax(-1, keepdim=True))[~bad].all()
    assert got[0][T // 2, 0, :64].isnan().any()


def test_tokens_without_a_page_are_dropped_and_read_as_zeros():
    D, Hk, page = 128, 2, 16
    kc, vc, table = make_cache([40, 40], Hk, D, page, "cuda")
    table[1, 1] = -1
    table[0, 2] = kc.shape[0] + 5
    before = kc.clone(), vc.clone()
    pos = torch.tensor([20, 33, -1, 48, 0, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    sid = torch.tensor([1, 0, 0, 0, 2, 0], dtype=torch.int32, device="cuda")
    k, v = random_rows(6, Hk, D, 1, "cuda")
    F.kv_append_int4(k, v, kc, vc, table, pos, sid)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    for x in F.kv_read_int4(kc, vc, table, pos, sid, D):
        assert not x.any()
    sid[4] = -3
    F.kv_append_int4(k, v, kc, vc, table, pos, sid)
    assert torch.equal(kc, before[0])
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    F.kv_append_int4(k[:0], v[:0], kc, vc, table, none, none)
    assert F.kv_read_int4(kc, vc, table, none, none, D)[0].shape == (0, Hk, D)


def test_groups_that_are_not_finite_read_back_as_nan():
    D, Hk = 128, 2
    kc, vc, table = make_cache([8], Hk, D, 16, "cuda")
    pos, sid = token_lists([0], [8], "cuda")
    k, v = random_rows(8, Hk, D, 2, "cuda")
    k[1, 0, 3] = math.nan
    v[2, 1, 100] = math.inf
    v[3, 0, 0] = -math.inf
    F.kv_append_int4(k, v, kc, vc, table, pos, sid)
    kk, vv = F.kv_read_int4(kc, vc, table, pos, sid, D)
    assert kk[1, 0, :64].isnan().all() and kk[1, 0, 64:].isfinite().all()
    assert not vv[2, 1, 64:].isfinite().any() and vv[2, 1, :64].isfinite().all() and not vv[3, 0, :64].isfinite().any()
    assert int((~kk.isfinite()).sum()) == 64 and int((~vv.isfinite()).sum()) == 128


def _decode_bound(res):
    # p scale rounded to bf16 (half a step of each term), the output's rounding; scores in fp32: sums of 128 terms and the
    # offset 16 + code, at most 2^-16 of scale sum |q| (|k| + 2 range) -> twice that relative error of p, over the spread
    return HALF * (res["centred"] + res["out"].abs()) + 2.0 ** -14 * (res["logit"] + 1) * (res["spread"] + res["out"].abs()) + 1e-6


@pytest.mark.parametrize("H,Hk,D,page,lens", [
    (8, 2, 128, 16, [37, 200, 1]), (32, 8, 128, 16, [513]), (8, 1, 128, 16, [64, 0, 15, 16, 17]), (3, 3, 128, 32, [100, 7]),
    (4, 4, 64, 16, [129, 31]), (4, 1, 64, 64, [1, 2, 3, 500]), (20, 1, 128, 16, [300, 90]), (9, 1, 64, 16, [77]),
    (12, 4, 128, 16, [2049, 1025]), (2, 1, 64, 16, [5000])])
def test_decode_against_64_bits(H, Hk, D, page, lens):
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=H + D)
    B = len(lens)
    g = torch.Generator().manual_seed(H)
    qkv = torch.randn(B, (H + 2 * Hk) * D, generator=g).to(torch.bfloat16).cuda()
    q = qkv[:, : H * D].unflatten(-1, (H, D))
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scale = 1.0 / math.sqrt(D)
    out = F.paged_attn_decode_int4(q, kc, vc, table, ctx)
    res = oracle(q, kc, vc, table, range(B), [1] * B, lens, scale)
    off = (out.cpu().double() - res["out"]).abs()
    assert (off <= _decode_bound(res)).all(), float((off / _decode_bound(res)).max())
    for b, n in enumerate(lens):
        assert n > 0 or not out[b].any()
    # the same bits every time, and with a table wider than the sequences need
    wide = torch.full((B + 1, table.shape[1] + 300), -1, dtype=torch.int32, device="cuda")
    wide[:B, : table.shape[1]] = table
    for _ in range(3):
        assert _same_bits(F.paged_attn_decode_int4(q, kc, vc, table, ctx), out)
    again = F.paged_attn_decode_int4(q, kc, vc, wide, ctx, scale)
    off = (again.cpu().double() - res["out"]).abs()
    assert (off <= _decode_bound(res)).all()
    native.check_status("cuda")


def _prefill_bound(res):
    # K, V and p rounded to bf16 for the prompt kernel: half a step of every key moves a score by 2^-8 scale sum |q| |k| at
    # most, every p by twice that (and the exponential's 2^-10), every value and every p by half a step, and the output's rounding
    return (2 * HALF * res["logit"] + 2.0 ** -10) * (1 + HALF * res["logit"]) * res["spread"] + 2 * HALF * (1 + HALF) * res["plain"] \
        + HALF * (res["out"].abs() + res["centred"]) + 1e-6


@pytest.mark.parametrize("H,Hk,D,page,new,old", [
    (8, 2, 128, 16, [5, 5, 5], [100, 0, 33]), (4, 4, 64, 32, [3, 1, 0, 2], [10, 200, 50, 0]), (8, 1, 128, 16, [8], [1000]),
    (4, 2, 128, 16, [200, 1, 33], [0, 64, 300]), (4, 4, 64, 16, [300, 129], [5, 0]), (3, 1, 64, 64, [17, 90], [130, 1]),
    (16, 2, 128, 48, [70], [400]), (2, 2, 128, 16, [257, 0, 513], [0, 40, 255]), (20, 5, 128, 16, [16, 15], [3, 77])])
def test_prefill_against_64_bits(H, Hk, D, page, new, old):
    lens = [a + b for a, b in zip(new, old)]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=H + D)
    T, B = sum(new), len(new)
    g = torch.Generator().manual_seed(H)
    q = torch.randn(T + 3, (H + 1) * D, generator=g).to(torch.bfloat16).cuda()[:, : H * D].unflatten(-1, (H, D))
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((T + 3, H, D), 3.0, device="cuda", dtype=torch.bfloat16)
    F.paged_attn_prefill_int4(q, kc, vc, table, cu, kv, max(new), max(lens), out=out)
    res = oracle(q[:T], kc, vc, table, cu[:-1].tolist(), new, lens, 1.0 / math.sqrt(D))
    off = (out[:T].cpu().double() - res["out"]).abs()
    assert (off <= _prefill_bound(res)).all(), float((off / _prefill_bound(res)).max())
    # the typical error is that of a few independent roundings, far below the bound
    assert float(off.norm() / res["out"].norm()) < 5e-3
    assert bool((out[T:] == 3.0).all())                     # rows behind the last sequence
    again = torch.full_like(out, 3.0)
    F.paged_attn_prefill_int4(q, kc, vc, table, cu, kv, max(new), max(lens), out=again)
    assert _same_bits(again, out)
    native.check_status("cuda")


@pytest.mark.parametrize("new", [2, 40])
def test_one_bad_token_reaches_only_the_queries_that_see_it(new):
    H, Hk, D, page = 4, 2, 128, 16
    lens = [60 + new, 20 + new]
    kc, vc, table = filled(lens, Hk, D, page, "cuda", seed=3)
    pos = torch.tensor([lens[0] - 1, lens[1] - 1], dtype=torch.int32, device="cuda")
    sid = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    k, v = random_rows(2, Hk, D, 9, "cuda")
    v[0, 0, 3] = math.inf
    k[1, 1, 70] = math.nan
    F.kv_append_int4(k, v, kc, vc, table, pos, sid)
    cu = torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
    q = torch.randn(2 * new, H, D, device="cuda").to(torch.bfloat16)
    out = F.paged_attn_prefill_int4(q, kc, vc, table, cu, torch.tensor(lens, dtype=torch.int32, device="cuda"), new, max(lens))
    bad = (~out.isfinite()).any(-1)
    want = torch.zeros_like(bad)
    want[new - 1, :2] = True
    want[2 * new - 1, 2:] = True
    assert torch.equal(bad, want)
    one = F.paged_attn_decode_int4(q[[new - 1, 2 * new - 1]], kc, vc, table, torch.tensor(lens, dtype=torch.int32, device="cuda") - 1)
    assert one.isfinite().all()                             # the bad token lies behind the context


def test_a_context_token_without_a_page_is_reported_and_left_out():
    H, Hk, D, page = 4, 2, 128, 16
    kc, vc, table = filled([64, 40], Hk, D, page, "cuda", seed=4)
    q = torch.randn(2, H, D, device="cuda").to(torch.bfloat16)
    ctx = torch.tensor([64, 40], dtype=torch.int32, device="cuda")
    whole = F.paged_attn_decode_int4(q, kc, vc, table, ctx)
    native.check_status("cuda")
    table[0, 1] = -1
    out = F.paged_attn_decode_int4(q, kc, vc, table, ctx)
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    assert out.isfinite().all() and torch.equal(out[1], whole[1]) and not torch.equal(out[0], whole[0])
    longer = torch.tensor([64, 400], dtype=torch.int32, device="cuda")       # longer than the table
    out = F.paged_attn_decode_int4(q, kc, vc, table, longer)
    with pytest.raises(RuntimeError, match="status 2"):
        native.check_status("cuda")
    assert out[0].isfinite().all()        # (row 1 claims tokens of its last page that were never written)


def test_two_captured_graphs_and_another_stream_share_nothing():
    H, Hk, D, page = 8, 2, 128, 16
    sets = []
    for seed in (1, 2):
        kc, vc, table = filled([300, 70], Hk, D, page, "cuda", seed=seed)
        q = torch.randn(2, H, D, device="cuda").to(torch.bfloat16)
        ctx = torch.tensor([300, 70], dtype=torch.int32, device="cuda")
        want = F.paged_attn_decode_int4(q, kc, vc, table, ctx)
        sets.append((q, kc, vc, table, ctx, want))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q, kc, vc, table, ctx, _ in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(F.paged_attn_decode_int4(q, kc, vc, table, ctx))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, s in zip(outs, sets):
        assert _same_bits(o, s[-1])


def test_refusals_on_the_gpu():
    kc, vc, table = make_cache([16], 2, 128, 16, "cuda")
    pos, sid = token_lists([0], [4], "cuda")
    k, v = random_rows(4, 2, 128, 0, "cuda")
    q = torch.randn(1, 4, 128, device="cuda").to(torch.bfloat16)
    ctx = torch.ones(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    calls = [
        lambda: F.kv_append_int4(k.float(), v, kc, vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v[:, :1], kc, vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v, kc[:, :1], vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v, kc[..., :-16].contiguous(), vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v, kc, vc, table, pos[:3], sid),
        lambda: F.kv_append_int4(k, v, kc, vc, table, pos.long(), sid),
        lambda: F.kv_append_int4(k[..., :96], v[..., :96], kc, vc, table, pos, sid),
        lambda: F.kv_append_int4(k.transpose(0, 1), v.transpose(0, 1), kc, vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v, kc.cpu(), vc, table, pos, sid),
        lambda: F.kv_read_int4(kc, vc, table, pos, sid, 96),
        lambda: F.kv_read_int4(kc, vc, table[0], pos, sid, 128),
        lambda: F.paged_attn_decode_int4(q[:, :3], kc, vc, table, ctx),
        lambda: F.paged_attn_decode_int4(q, kc, vc, table, ctx.repeat(2)),
        lambda: F.paged_attn_decode_int4(q.half(), kc, vc, table, ctx),
        lambda: F.paged_attn_decode_int4(q, kc, vc, table, ctx, out=torch.empty(1, 4, 128, device="cuda")),
        lambda: F.paged_attn_prefill_int4(q, kc, vc, table, cu[:1], ctx, 1, 16),
        lambda: F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, 2, 16),
        lambda: F.paged_attn_prefill_int4(q, kc, vc, table, cu, ctx, 1, 17),
    ]
    for i, call in enumerate(calls):
        with pytest.raises((RuntimeError, ValueError, IndexError)):
            call()
            pytest.fail(f"call {i} was not refused")
    empty = F.paged_attn_decode_int4(q[:0], kc, vc, table, ctx[:0])
    assert empty.shape == (0, 4, 128)


# ------------------------------------------------------------------------------------------------ together, in the engine
@pytest.mark.parametrize("D", [128, 64])
def test_fused_epilogue_writes_what_rope_and_append_write(D):
    C = native.require()
    torch.manual_seed(D)
    H, Hk, page, T = 4, 2, 32, 5
    kc, vc, table = make_cache([40] * T, Hk, D, page, "cuda")
    kr, vr = kc.clone(), vc.clone()
    acc = torch.randn(T, (H + 2 * Hk) * D, device="cuda") * 2
    qkv = acc.to(torch.bfloat16)
    pos = torch.tensor([5, 17, 0, 33, 2], device="cuda", dtype=torch.int32)
    sid = torch.arange(T, device="cuda", dtype=torch.int32)
    sid[4] = T + 3                                  # outside the table: dropped
    q = torch.empty(T, H, D, device="cuda", dtype=torch.bfloat16)
    C.qkv_rope_append(acc, pos, sid, table, q, kc, vc, 10000.0)
    qk = qkv[:, : (H + Hk) * D].clone().unflatten(-1, (H + Hk, D))
    C.rope(qk, pos, 10000.0, False)
    F.kv_append_int4(qk[:, H:].contiguous(), qkv[:, (H + Hk) * D:].unflatten(-1, (Hk, D)), kr, vr, table, pos, sid)
    assert torch.equal(vc, vr) and float(acc.abs().max()) == 0.0
    # the two rotations round differently in places: a key may be a bf16 step off, its code then one step of the grid
    got, want = (F.kv_read_int4(c, vc, table, pos, sid, D)[0].float() for c in (kc, kr))
    step = (want.unflatten(-1, (-1, 64)).amax(-1) - want.unflatten(-1, (-1, 64)).amin(-1)) / 15
    assert ((got - want).abs().unflatten(-1, (-1, 64)) <= 1.1 * step[..., None] + 2 * HALF * want.abs().amax()).all()
    assert float((q.float() - qk[:, :H].float()).abs().max()) <= 2 * HALF * float(qk.float().abs().max())


def _engine(kv_dtype, D=128, **kw):
    from mythos_b200.infer.engine import InferenceEngine
    from mythos_b200.models import TransformerConfig

    cfg = TransformerConfig(vocab_size=512, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=D,
                            ffn_hidden_size=512, max_seq_len=512, oil_block_size=256, codebook_group=2)
    return InferenceEngine.random(cfg, seed=7, device="cuda", max_batch=8, max_seq_len=512, kv_dtype=kv_dtype, **kw)


def _off(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


@pytest.mark.parametrize("D", [128, 64])
def test_engine_over_4_bit_pages(D):
    """Prompts, portions, prefix hits, decoding, offload: logits of the 4-bit engine against the bf16 engine's and against
    each other. A 4-bit value is a step / sqrt(12) off, a tenth of its spread: logits stay within a quarter; two ways to the
    same pages differ by bf16 roundings that move a few codes by a step: half of that."""
    g = torch.Generator().manual_seed(1)
    head = torch.randint(0, 512, (150,), generator=g).tolist()
    a, b = head + [5, 6, 7], head + [9, 10, 11, 12, 13]
    wide, eng = _engine("bf16", D), _engine("int4", D)
    assert eng.cache.int4 and eng.cache.size_bytes() * 32 == wide.cache.size_bytes() * 9
    ref_logits = wide.start_sequence(b, reuse_prefix=False)[1]
    sa, la = eng.start_sequence(a)
    sb, lb = eng.start_sequence(b)                       # over the shared pages of the first prompt
    assert eng.last_prefix_hit == 144
    sc, lc = eng.start_sequence(b, reuse_prefix=False)
    assert _off(lb, ref_logits) < 0.25 and _off(lc, ref_logits) < 0.25 and _off(lb, lc) < 0.25
    seq = eng.cache.new_sequence()                       # the same prompt in portions through step()
    for lo in range(0, len(b), 61):
        ls = eng.step([seq], [b[lo:lo + 61]])
    assert _off(ls, lb) < 0.125
    tokens = [int(lb.float().argmax())] * 4
    out = eng.decode([sa, sb, sc, seq], tokens)
    assert _off(out[1], out[3]) < 0.125 and out.isfinite().all()
    eng.fused_decode = False                             # one more token through the separate kernels and through step()
    handle = eng.cache.offload_sequence(sb)
    sb = eng.cache.restore_sequence(handle)
    eng.cache.sync_tables()
    one = eng.decode([sb], [3])
    many = eng.step([seq], [[3]])
    assert _off(one, many) < 0.125
    for s in (sa, sb, sc, seq):
        eng.release(s)
    assert eng.cache.alloc.used == 0
    native.check_status("cuda")


def test_engine_generates_over_4_bit_pages():
    from mythos_b200.infer.serving import ContinuousBatcher

    eng = _engine("int4")
    g = torch.Generator().manual_seed(3)
    prompts = torch.randint(0, 512, (2, 128), generator=g, dtype=torch.int32)
    eager = eng.generate(prompts, max_new_tokens=12, use_graph=False).tokens
    assert eng.generate(prompts, max_new_tokens=12, use_graph=True).tokens == eager
    ragged = [prompts[0].tolist(), prompts[1, :77].tolist(), [4]]
    res = eng.generate(ragged, max_new_tokens=5)
    assert [len(t) for t in res.tokens] == [5, 5, 5]
    batcher = ContinuousBatcher(eng, chunk_tokens=40)
    reqs = [batcher.submit(p, max_new_tokens=6) for p in ragged]
    batcher.run_until_idle()
    assert all(len(r.output) == 6 for r in reqs) and eng.cache.alloc.used == 0
    native.check_status("cuda")
