"""The limits that the GPU tests of attention over 4-bit pages go by, against faults that they have to find."""
import math

import pytest
import torch

from kv_int4_bounds import attention, check
from kv_int4_util import filled
from mythos_b200.ops import functional as F


@pytest.mark.parametrize("H,Hk,D,n", [(4, 2, 128, 6000), (2, 1, 64, 5000), (2, 1, 128, 40000)])
def test_a_chunk_that_is_left_out_is_found(H, Hk, D, n):
    kc, vc, table = filled([n], Hk, D, 16, "cpu", seed=9)
    q = torch.randn(1, H, D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    want = attention(q, kc, vc, table, [0], [1], [n], 1 / math.sqrt(D))
    check(want[0].to(torch.bfloat16), *want)
    gaps = table.clone()
    gaps[0, 100:102] = -1                                   # 32 tokens
    less = attention(q, kc, vc, gaps, [0], [1], [n], 1 / math.sqrt(D))[0].to(torch.bfloat16)
    with pytest.raises(AssertionError):
        check(less, *want)


def test_operands_rounded_to_bf16_are_found():
    H, Hk, D, new, n = 4, 2, 128, 60, 700
    kc, vc, table = filled([n], Hk, D, 16, "cpu", seed=3)
    q = torch.randn(new, H, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    want = attention(q, kc, vc, table, [0], [new], [n], 1 / math.sqrt(D))
    ctx = torch.tensor([n], dtype=torch.int32)
    check(F.paged_attn_prefill_int4(q, kc, vc, table, torch.tensor([0, new], dtype=torch.int32), ctx, new, n), *want)
    pos = torch.arange(n, dtype=torch.int32)
    k, v = (x.double() for x in F.kv_read_int4(kc, vc, table, pos, torch.zeros_like(pos), D))       # bf16 values
    got = torch.empty_like(want[0])
    for h in range(H):
        hidden = pos > n - new + torch.arange(new)[:, None]
        p = torch.softmax((q[:, h].double() @ k[:, h // 2].T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
        got[:, h] = p.to(torch.bfloat16).double() @ v[:, h // 2]
    with pytest.raises(AssertionError):
        check(got.to(torch.bfloat16), *want)
