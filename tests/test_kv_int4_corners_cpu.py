"""Corners of the CPU form of attention over 4-bit pages."""
import math
from fractions import Fraction

import pytest
import torch

from kv_int4_util import filled, make_cache, token_lists
from mythos_b200.ops import functional as F, reference as ref


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_a_value_that_is_not_finite_reaches_only_the_queries_that_see_it(what):
    H, Hk, D, page = 4, 2, 64, 16
    kc, vc, table = filled([50], Hk, D, page, "cpu")
    q = torch.randn(20, H, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    cu, lens = torch.tensor([0, 20], dtype=torch.int32), torch.tensor([50], dtype=torch.int32)
    whole = F.paged_attn_prefill_int4(q, kc, vc, table, cu, lens, 20, 50)
    pos, sid = torch.tensor([45], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    k, v = F.kv_read_int4(kc, vc, table, pos, sid, D)
    v[0, 0, 3] = what
    F.kv_append_int4(k, v, kc, vc, table, pos, sid)
    out = F.paged_attn_prefill_int4(q, kc, vc, table, cu, lens, 20, 50)
    assert not out[15:, :2].isfinite().any() and out[:, 2:].isfinite().all()       # queries at 45 .. 49, heads of the first kv head
    # (the other head's row was quantised again: its codes are the same)
    assert torch.equal(out[:15], whole[:15])


def _nearest_bf16(x):
    """The bf16 number nearest to a fraction, ties to even."""
    if x == 0:
        return 0.0
    a, e = abs(x), 0
    while a >= 256:
        a, e = a / 2, e + 1
    while a < 128:
        a, e = a * 2, e - 1
    return math.copysign(round(a) * 2.0 ** e, x)          # (round: ties to even)


def test_values_are_rounded_once():
    """scale * code + low where the product lies halfway between two bf16 numbers and low is far smaller, and where the product passes
    the largest 32-bit number although the sum does not."""
    D, page = 64, 16
    top = float(torch.tensor(3.3895e38).to(torch.bfloat16))
    groups = [(-1e-18, 1e17), (1e-18, 1e17), (-1e-30, 3.7), (2e-30, 0.51), (-top, 1e-20), (-top, -1e-20), (-3.0, 1e-9)]
    g = torch.Generator().manual_seed(0)
    x = torch.stack([lo + (hi - lo) * torch.rand(D, generator=g, dtype=torch.float64) for lo, hi in groups]).clamp(-top, top)
    x[:, 0], x[:, 1] = torch.tensor([lo for lo, _ in groups]), torch.tensor([hi for _, hi in groups])
    x = x.to(torch.bfloat16)[:, None]
    kc, vc, table = make_cache([len(groups)], 1, D, page, "cpu")
    pos, sid = token_lists([0], [len(groups)], "cpu")
    F.kv_append_int4(x, x, kc, vc, table, pos, sid)
    got = F.kv_read_int4(kc, vc, table, pos, sid, D)
    code, scale, low = ref.kv4_quantise(x)
    for t in range(len(groups)):
        want = [_nearest_bf16(Fraction(int(c)) * Fraction(float(scale[t, 0, 0])) + Fraction(float(low[t, 0, 0]))) for c in code[t, 0]]
        assert got[0][t, 0].tolist() == want and got[1][t, 0].tolist() == want, t
