"""Corners of the CPU form of attention over 4-bit pages."""
import math

import pytest
import torch

from kv_int4_util import filled
from mythos_b200.ops import functional as F


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
