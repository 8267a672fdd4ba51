"""4-bit paged KV cache on the CPU: the format bit by bit, the reference operators, refusals."""
import math

import pytest
import torch

from kv_int4_util import filled, make_cache, oracle, random_rows, token_lists
from mythos_b200.ops import functional as F, reference as ref


def _value(cache, D, page, page_id, head, n, d, is_key):
    """One value of a page, from its bytes: written from the format's description."""
    rec = cache[page_id, head].tolist()
    tile = rec[n // 16 * 16 * (D // 2 + D // 16):]
    m = n % 16
    order = 8 * (m // 8) + 2 * (m % 4) + m // 4 % 2
    g, e = d // 64, d % 64
    if is_key:
        word = (e // 16 * (D // 64) + g) * 2 + e % 16 // 8
        row = order
    else:
        word = ((e // 8) ^ (4 * (m // 2 % 2))) * (D // 64) + g
        row = m
    at = row * D // 2 + 4 * word
    w = int.from_bytes(bytes(tile[at:at + 4]), "little")
    if is_key:
        w = (w >> 3 | w << 29) & 0xFFFFFFFF
    code = w >> 4 * (e % 8 // 2 + 4 * (e % 2)) & 15
    pair = 16 * D // 2 + order * D // 16 + 4 * g
    scale, low = torch.tensor(tile[pair:pair + 4], dtype=torch.uint8).view(torch.bfloat16).double().tolist()
    return code, scale, low


@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (128, 48)])
def test_format_bit_by_bit(D, page):
    lens = [37, 3]
    kc, vc, table = make_cache(lens, 2, D, page, "cpu", seed=D)
    pos, sid = token_lists([0, 0], lens, "cpu")
    k, v = random_rows(40, 2, D, 1, "cpu")
    F.kv_append_int4(k, v, kc, vc, table, pos, sid)
    kk, vv = F.kv_read_int4(kc, vc, table, pos, sid, D)
    for t in (0, 5, 15, 16, 22, 36, 37, 39):
        p = int(table[sid[t], pos[t] // page])
        for h in range(2):
            for is_key, x, got in ((True, k, kk), (False, v, vv)):
                row = x[t, h].double()
                for d in (0, 1, 7, 8, 17, 31, 42, 63, D - 1, D - 30):
                    code, scale, low = _value(kc if is_key else vc, D, page, p, h, int(pos[t]) % page, d, is_key)
                    grp = row[d // 64 * 64: d // 64 * 64 + 64]
                    want = float(((grp.max() - grp.min()) / 15).to(torch.bfloat16))
                    assert scale == want and low == float(grp.min())
                    assert abs(code - (float(row[d]) - low) / scale) <= 0.5 or code == 15
                    assert float(got[t, h, d]) == float(torch.tensor(code * scale + low).to(torch.bfloat16))


def test_quantiser_edges():
    x = torch.zeros(6, 1, 64, dtype=torch.bfloat16)
    x[1] = -2.5                                            # one value: scale 0, read back exactly
    x[2, 0, 5] = math.nan
    x[3, 0, 5] = math.inf
    x[4, 0, 0], x[4, 0, 1] = 3e38, -3e38                   # range beyond fp32
    x[5, 0] = torch.arange(64) % 16                        # 0 .. 15: exact
    kc, vc, table = make_cache([6], 1, 64, 16, "cpu")
    pos, sid = token_lists([0], [6], "cpu")
    F.kv_append_int4(x, x, kc, vc, table, pos, sid)
    for y in F.kv_read_int4(kc, vc, table, pos, sid, 64):
        assert torch.equal(y[0], x[0]) and torch.equal(y[1], x[1]) and torch.equal(y[5], x[5])
        assert not y[2].isfinite().any() and not y[3].isfinite().any() and not y[4].isfinite().any()


def test_half_a_step_ties_to_even():
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2], x[0, 0, 3] = 15.0, 0.5, 1.5, 2.5
    code, scale, low = ref.kv4_quantise(x)
    assert float(scale) == 1.0 and float(low) == 0.0 and code[0, 0, :4].tolist() == [15, 0, 2, 2]


def test_reference_attention_over_pages_and_lengths_of_zero():
    H, Hk, D, page = 4, 2, 64, 16
    new, old = [3, 0, 1, 2], [20, 5, 0, 0]
    lens = [a + b for a, b in zip(new, old)]
    kc, vc, table = filled(lens, Hk, D, page, "cpu")
    q = torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    cu = torch.tensor([0, 3, 3, 4, 6], dtype=torch.int32)
    out = F.paged_attn_prefill_int4(q, kc, vc, table, cu, torch.tensor(lens, dtype=torch.int32), 3, 23)
    res = oracle(q, kc, vc, table, [0, 3, 3, 4], new, lens, 1 / math.sqrt(D))
    assert ((out.double() - res["out"]).abs() <= 2.0 ** -8 * res["out"].abs() + 1e-5).all()
    ctx = torch.tensor([23, 0, 1, 2], dtype=torch.int32)
    dec = F.paged_attn_decode_int4(q[:4], kc, vc, table, ctx)
    assert not dec[1].any() and dec.isfinite().all()


def test_tokens_without_a_page():
    kc, vc, table = make_cache([40, 40], 2, 128, 16, "cpu")
    table[1, 1] = -1
    table[0, 2] = kc.shape[0]
    before = kc.clone()
    pos = torch.tensor([20, 33, -1, 48, 0], dtype=torch.int32)
    sid = torch.tensor([1, 0, 0, 0, 2], dtype=torch.int32)
    k, v = random_rows(5, 2, 128, 1, "cpu")
    F.kv_append_int4(k, v, kc, vc, table, pos, sid)
    assert torch.equal(kc, before)
    for x in F.kv_read_int4(kc, vc, table, pos, sid, 128):
        assert not x.any()


def test_a_key_without_a_page_is_seen_by_no_query():
    H, Hk, D, page = 4, 2, 64, 16
    kc, vc, table = filled([50], Hk, D, page, "cpu")
    gaps = table.clone()
    gaps[0, 1], gaps[0, 3] = -1, kc.shape[0]
    q = torch.randn(20, H, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    lens = torch.tensor([50], dtype=torch.int32)
    out = F.paged_attn_prefill_int4(q, kc, vc, gaps, torch.tensor([0, 20], dtype=torch.int32), lens, 20, 50)
    here = torch.tensor([*range(16), *range(32, 48)])
    k, v = (x.double() for x in ref.kv_read_int4(kc, vc, table, here, torch.zeros_like(here), D, torch.float32))
    for h in range(H):
        sc = q[:, h].double() @ k[:, h // 2].T / math.sqrt(D)
        want = torch.softmax(sc.masked_fill(here > 30 + torch.arange(20)[:, None], -math.inf), -1) @ v[:, h // 2]
        # (the output's rounding; sums of 64 terms in 32 bits)
        assert ((out[:, h].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()


def test_refusals():
    kc, vc, table = make_cache([16], 2, 128, 16, "cpu")
    pos, sid = token_lists([0], [4], "cpu")
    k, v = random_rows(4, 2, 128, 0, "cpu")
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    ctx = torch.ones(1, dtype=torch.int32)
    calls = [
        lambda: F.kv4_token_bytes(96),
        lambda: F.kv_append_int4(k, v[:, :1], kc, vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v, kc[:, :1], vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v, kc[..., :-16].contiguous(), vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v, kc.to(torch.int8), vc, table, pos, sid),
        lambda: F.kv_append_int4(k, v, kc, vc, table, pos[:3], sid),
        lambda: F.kv_append_int4(k, v, kc, vc, table[0], pos, sid),
        lambda: F.kv_read_int4(kc, vc, table, pos, sid, 96),
        lambda: F.paged_attn_decode_int4(q[:, :3], kc, vc, table, ctx),
        lambda: F.paged_attn_decode_int4(q, kc, vc, table, ctx.repeat(2)),
        lambda: F.paged_attn_prefill_int4(q, kc, vc, table, ctx, ctx, 1, 16),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_paged_cache_of_4_bit_pages():
    from mythos_b200.infer.kv_paged import PagedKVCache

    c = PagedKVCache(2, 3, 128, num_pages=8, page_size=32, max_seqs=2, max_pages_per_seq=4, device="cpu", dtype=torch.uint8)
    wide = PagedKVCache(2, 3, 128, num_pages=8, page_size=32, max_seqs=2, max_pages_per_seq=4, device="cpu")
    assert c.int4 and not wide.int4 and c.size_bytes() * 32 == wide.size_bytes() * 9
    s = c.new_sequence()
    c.reserve(s, 40)
    c.sync_tables()
    k, v = random_rows(40, 3, 128, 0, "cpu")
    pos, sid = token_lists([0], [40], "cpu")
    for li in range(2):
        F.kv_append_int4(k, v, c.k[li], c.v[li], c.block_table, pos, sid)
    c.advance(s, 40)
    want = F.kv_read_int4(c.k[1], c.v[1], c.block_table, pos, sid, 128)
    other = c.new_sequence()
    c.reserve(other, 20)                          # so that the pages move
    s = c.restore_sequence(c.offload_sequence(s))
    c.sync_tables()
    got = F.kv_read_int4(c.k[1], c.v[1], c.block_table, pos, torch.full_like(sid, s), 128)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 128, 4, page_size=24, device="cpu", dtype=torch.uint8)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 96, 4, device="cpu", dtype=torch.uint8)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 64, 4, device="cpu", dtype=torch.uint8, layer_shapes=[(1, 64, 64)])


def test_engine_refuses_what_4_bit_pages_cannot_hold():
    from mythos_b200.infer.engine import InferenceEngine
    from mythos_b200.models import TransformerConfig

    cfg = TransformerConfig(vocab_size=64, hidden_size=96, num_layers=1, num_heads=1, head_dim=96, ffn_hidden_size=64, max_seq_len=64)
    with pytest.raises(ValueError):
        InferenceEngine(cfg, device="cpu", kv_dtype="int4")
    cfg.head_dim = 64
    with pytest.raises(ValueError):
        InferenceEngine(cfg, device="cpu", kv_dtype="int4", page_size=8)
    with pytest.raises(ValueError):
        InferenceEngine(cfg, device="cpu", kv_dtype="fp4")
