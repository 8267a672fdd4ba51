"""Pure-PyTorch restatements of every kernel, written from the reference's formulas.

They run on CPU (and on CUDA tensors through torch operators) and serve two purposes: the
numerical oracle that each sm_100a kernel is tested against, and the execution path of
CPU-only runs (the tiny byte-level configuration). All math is fp32 regardless of the input
dtype; results are cast back to the input dtype.

Formula sources in the reference tree: RMSNorm ``src/math.cpp:182-205``; RoPE
``src/transformer.cpp:108-135``; SiLU / SwiGLU ``src/transformer.cpp:373-387``; attention
``src/autograd.cpp:361-461``; cross-entropy ``src/autograd.cpp:1166-1215``; AdamW
``src/optimizer.cpp:91-119``; nearest-centroid quantisation ``src/codebook.cpp:172-186``;
router ``src/moe_variants.cpp:25-91``; sampler ``src/sampler.cpp:12-120``.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rmsnorm(x, gamma, eps: float = 1e-5, residual=None):
    """Returns ``(y, h)`` with ``h = x + residual`` (or ``x``) and ``y = rmsnorm(h) * gamma``."""
    h = x.float() if residual is None else (x.float() + residual.float())
    if residual is not None:
        h = h.to(x.dtype).float()  # the kernel normalises the rounded sum
    rstd = torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    y = h * rstd * gamma.float()
    return y.to(x.dtype), h.to(x.dtype)


def layernorm(x, gamma, beta=None, eps: float = 1e-5):
    xf = x.float()
    mu = xf.mean(-1, keepdim=True)
    var = (xf - mu).pow(2).mean(-1, keepdim=True)
    y = (xf - mu) * torch.rsqrt(var + eps) * gamma.float()
    if beta is not None:
        y = y + beta.float()
    return y.to(x.dtype)


def rope_tables(pos, head_dim: int, theta: float):
    j = torch.arange(head_dim // 2, device=pos.device, dtype=torch.float32)
    inv_freq = theta ** (-2.0 * j / head_dim)
    ang = pos.float()[:, None] * inv_freq[None, :]
    return torch.cos(ang), torch.sin(ang)


def rope(x, pos, theta: float = 10000.0, inverse: bool = False):
    """Half-split rotary embedding. x: [tokens, heads, head_dim]; pos: [tokens]."""
    d = x.shape[-1]
    cos, sin = rope_tables(pos, d, theta)
    if inverse:
        sin = -sin
    xf = x.float()
    a, b = xf[..., : d // 2], xf[..., d // 2:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    out = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return out.to(x.dtype)


def silu(x):
    return x / (1.0 + torch.exp(-x))


def swiglu(gate_up):
    """gate_up: [..., 2*ffn] with gate in the first half. Returns silu(gate) * up."""
    f = gate_up.shape[-1] // 2
    g, u = gate_up[..., :f].float(), gate_up[..., f:].float()
    return (silu(g) * u).to(gate_up.dtype)


def relu2(x):
    return torch.relu(x.float()).pow(2).to(x.dtype)


def gelu_erf(x):
    xf = x.float()
    return (0.5 * xf * (1.0 + torch.erf(xf / math.sqrt(2.0)))).to(x.dtype)


def gelu_tanh(x):
    xf = x.float()
    return (0.5 * xf * (1.0 + torch.tanh(0.7978845608028654 * (xf + 0.044715 * xf ** 3)))).to(x.dtype)


def attention(q, k, v, causal: bool = True, scale: float | None = None):
    """Naive softmax(Q K^T * scale) V. q: [B,S,H,D]; k, v: [B,Skv,Hkv,D] (standard GQA grouping:
    query head h uses kv head h // (H/Hkv)). Returns (o [B,S,H,D], lse [B,H,S])."""
    B, S, H, D = q.shape
    Skv, Hkv = k.shape[1], k.shape[2]
    scale = (1.0 / math.sqrt(D)) if scale is None else scale
    qf = q.float().permute(0, 2, 1, 3)
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(H // Hkv, dim=1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(H // Hkv, dim=1)
    s = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    if causal:
        mask = torch.ones(S, Skv, dtype=torch.bool, device=q.device).tril(diagonal=Skv - S)
        s = s.masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(s, dim=-1)
    p = torch.exp(s - lse[..., None])
    o = torch.matmul(p, vf).permute(0, 2, 1, 3)
    return o.to(q.dtype), lse


def cross_entropy(logits, targets):
    """Per-row loss ``logsumexp - logit[target]`` with targets clamped to [0, V-1]."""
    lf = logits.float()
    t = targets.long().clamp(0, lf.shape[-1] - 1)
    return torch.logsumexp(lf, dim=-1) - lf.gather(-1, t[:, None]).squeeze(-1)


def cross_entropy_grad(logits, targets, grad_scale: float):
    lf = logits.float()
    t = targets.long().clamp(0, lf.shape[-1] - 1)
    p = torch.softmax(lf, dim=-1)
    p.scatter_add_(-1, t[:, None], -torch.ones_like(p[:, :1]))
    return (p * grad_scale).to(logits.dtype)


def adamw_step(p, m, v, g, lr, beta1, beta2, eps, weight_decay, step, grad_scale: float = 1.0):
    """In-place AdamW in the reference's form (decoupled decay, bias-corrected moments)."""
    g = g.float() * grad_scale
    p.mul_(1.0 - lr * weight_decay)
    m.mul_(beta1).add_(g, alpha=1.0 - beta1)
    v.mul_(beta2).addcmul_(g, g, value=1.0 - beta2)
    bc1 = 1.0 - beta1 ** step
    bc2 = 1.0 - beta2 ** step
    p.addcdiv_(m / bc1, (v / bc2).sqrt() + eps, value=-lr)
    return p, m, v


def nearest_centroid(w, codebooks, cb_map, bs: int):
    """Brute-force nearest centroid, first minimum wins. w: flat fp32 [n]; codebooks [n_cb, C];
    cb_map: int [n_blocks] or None (block b uses codebook b). Returns (indices u8, dequantised fp32)."""
    n = w.numel()
    nb = (n + bs - 1) // bs
    pad = nb * bs - n
    wf = F.pad(w.float().reshape(-1), (0, pad)).reshape(nb, bs)
    cbi = torch.arange(nb, device=w.device) if cb_map is None else cb_map.long()
    idx = torch.empty(nb, bs, dtype=torch.uint8, device=w.device)
    deq = torch.empty(nb, bs, dtype=torch.float32, device=w.device)
    step = max(1, (1 << 22) // (bs * codebooks.shape[-1]))
    for s in range(0, nb, step):
        cb = codebooks[cbi[s:s + step]].float()  # [b, C]
        d = (wf[s:s + step, :, None] - cb[:, None, :]).pow(2)
        j = d.argmin(dim=-1)  # torch.argmin returns the first minimum on ties
        idx[s:s + step] = j.to(torch.uint8)
        deq[s:s + step] = torch.gather(cb, 1, j)
    return idx.reshape(-1)[:n], deq.reshape(-1)[:n]


def i2s_quant(w, bs: int):
    """I2_S ternary: per-block absmean scale, trit = clamp(round(w/scale), -1, 1).
    Returns (codes u8 in {0,1,2} = trit+1, scales fp32 [n_blocks], dequantised fp32)."""
    n = w.numel()
    nb = (n + bs - 1) // bs
    pad = nb * bs - n
    wf = F.pad(w.float().reshape(-1), (0, pad)).reshape(nb, bs)
    cnt = torch.full((nb,), bs, dtype=torch.float32, device=w.device)
    if pad:
        cnt[-1] = bs - pad
    a = wf.abs()
    amax = a.amax(-1)
    # a block that already is {-s, 0, +s} keeps s, so quantising twice equals quantising once
    exact = ((a == 0) | (a == amax[:, None])).all(-1)
    scale = torch.where(exact, amax, a.sum(-1) / cnt)
    inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    t = torch.round(wf * inv[:, None]).clamp(-1, 1)
    deq = t * scale[:, None]
    return (t + 1).to(torch.uint8).reshape(-1)[:n], scale, deq.reshape(-1)[:n]


def router_topk(logits, k: int):
    """softmax over all experts, top-k by probability, weights are those probabilities
    (not renormalised over the chosen k). Returns (weights [T,k], experts [T,k], probs [T,E])."""
    probs = torch.softmax(logits.float(), dim=-1)
    w, e = torch.topk(probs, k, dim=-1)
    return w, e, probs


def load_balance_loss(probs, experts, num_experts: int):
    """E * sum_e f_e * P_e with f_e = fraction of tokens routed to e (any of the k slots) and
    P_e = mean over tokens of the probability of e when chosen."""
    T = probs.shape[0]
    onehot = torch.zeros(T, num_experts, device=probs.device, dtype=torch.float32)
    onehot.scatter_(1, experts, 1.0)
    f = onehot.sum(0) / T
    P = (probs * onehot).sum(0) / T
    return num_experts * (f * P).sum()


def z_loss(logits, coef: float):
    return coef * torch.logsumexp(logits.float(), dim=-1).pow(2).mean()


# --------------------------------------------------------------------------------------- 4-bit KV cache
# Format (csrc/kernels/kv_int4.cuh): groups of 64 values with scale = bf16((max - min) / 15), low = min and codes
# clamp(round((x - low) / scale), 0, 15), standing for scale * code + low; caches [pages, kv_heads, page_size / 16 tiles
# of 16 code rows and 16 (scale, low) rows] bytes.
KV4_TILE, KV4_GROUP = 16, 64


def kv4_token_bytes(head_dim: int) -> int:
    """Bytes of one token's row (one kv head, K or V) in a 4-bit page: codes and one 4-byte pair per 64 values."""
    if head_dim not in (64, 128):
        raise ValueError(f"4-bit pages: head_dim must be 64 or 128, got {head_dim}")
    return head_dim // 2 + head_dim // 16


def kv4_check(k_cache, v_cache, block_table, kv_heads: int, head_dim: int) -> int:
    """Checks a pair of caches and their table; returns the page size."""
    per = kv4_token_bytes(head_dim)
    for c in (k_cache, v_cache):
        if c.dtype != torch.uint8 or c.dim() != 3 or not c.is_contiguous():
            raise ValueError("4-bit caches are contiguous uint8 tensors [pages, kv_heads, page bytes]")
    if k_cache.shape != v_cache.shape or k_cache.shape[1] != kv_heads:
        raise ValueError("4-bit caches: k and v caches of one shape, with the kv heads of the rows")
    if k_cache.shape[2] == 0 or k_cache.shape[2] % (per * KV4_TILE):
        raise ValueError(f"4-bit caches: a page holds a multiple of {KV4_TILE} tokens of {per} bytes each")
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise ValueError("4-bit caches: block_table is int32 [sequences, pages]")
    return k_cache.shape[2] // per


def kv4_quantise(x):
    """x [..., D] (bf16) -> (codes uint8 [..., D], scale, low: bf16 [..., D / 64])."""
    g = x.float().unflatten(-1, (-1, KV4_GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    # (a tensor divisor: torch turns a division by a scalar into a product with its reciprocal)
    scale = ((hi - lo) / torch.full_like(lo, 15.0)).to(torch.bfloat16).float()
    code = torch.round((g - lo) / scale).clamp(0, 15)
    code = torch.where((scale > 0) & ~code.isnan(), code, torch.zeros_like(code))
    return code.to(torch.uint8).flatten(-2), scale.squeeze(-1).to(torch.bfloat16), lo.squeeze(-1).to(torch.bfloat16)


def kv4_values(code, scale, low, dtype=torch.bfloat16):
    """scale * code + low (fp32 tensors that broadcast) rounded once to ``dtype``, as the kernels' fused multiply-add does: a sum in 32
    bits would lose a low far below the product, and with it which way a bf16 tie goes."""
    p, low = code.double() * scale.double(), low.double()
    s = p + low
    y = s.float()
    if dtype == torch.bfloat16:
        b = s - p
        rest = (s - y.double()) + ((p - (s - b)) + (low - b))          # what y lacks (two-sum)
        tie = (y.view(torch.int32) & 0xFFFF) == 0x8000
        y = torch.where(tie & (rest != 0), torch.nextafter(y, torch.where(rest > 0, torch.inf, -torch.inf).to(y)), y)
    return y.to(dtype)


def _kv4_row(n):
    return (n & 8) + ((n & 3) << 1) + ((n >> 2) & 1)


def kv4_places(block_table, page_size: int, n_pages: int, positions, seq_ids):
    """(page, tile in the page, place in the tile, has a page) of every token."""
    pos, seq = positions.long(), seq_ids.long()
    ok = (seq >= 0) & (seq < block_table.shape[0]) & (pos >= 0) & (pos < block_table.shape[1] * page_size)
    pos, seq = torch.where(ok, pos, 0), torch.where(ok, seq, 0)
    if block_table.numel() == 0:
        return pos, pos, pos, ok & False
    page = block_table[seq, pos // page_size].long()
    ok = ok & (page >= 0) & (page < n_pages)
    return torch.where(ok, page, 0), pos % page_size // KV4_TILE, pos % KV4_TILE, ok


def _kv4_views(cache, page_size: int, D: int):
    tiles = cache.view(cache.shape[0], cache.shape[1], page_size // KV4_TILE, -1)
    split = KV4_TILE * D // 2
    return tiles[..., :split].unflatten(-1, (KV4_TILE, D // 2)), tiles[..., split:].unflatten(-1, (KV4_TILE, D // 16))


def _kv4_word_order(D: int, n, is_key: bool):
    """Word of the row that holds values 8 w .. 8 w + 7, for every token: [tokens, D / 8]."""
    w = torch.arange(D // 8, device=n.device)
    g, u = w // 8, w % 8
    if is_key:
        return ((u // 2 * (D // 64) + g) * 2 + u % 2).expand(n.numel(), -1)
    return (u ^ (4 * (n // 2 % 2))[:, None]) * (D // 64) + g


def kv_append_int4(k, v, k_cache, v_cache, block_table, positions, seq_ids):
    """Quantises k, v [tokens, kv_heads, D] into the 4-bit pages (in place); tokens without a page are dropped."""
    T, H, D = k.shape
    page_size = kv4_check(k_cache, v_cache, block_table, H, D)
    if v.shape != k.shape or positions.numel() != T or seq_ids.numel() != T:
        raise ValueError("kv_append_int4: k and v of one shape, one position and one sequence per token")
    page, tile, n, ok = kv4_places(block_table, page_size, k_cache.shape[0], positions, seq_ids)
    page, tile, n = page[ok], tile[ok], n[ok]
    at = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=k.device)      # bit position of value e of a word
    for x, cache, is_key in ((k, k_cache, True), (v, v_cache, False)):
        code, scale, low = kv4_quantise(x[ok])
        w = (code.long().unflatten(-1, (-1, 8)) << at).sum(-1)              # [tokens, H, D / 8]
        if is_key:
            w = (w << 3 | w >> 29) & 0xFFFFFFFF
        order = _kv4_word_order(D, n, is_key)[:, None].expand_as(w)
        w = torch.empty_like(w).scatter_(2, order, w)
        w = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32).contiguous().view(torch.uint8)
        rows, pairs = _kv4_views(cache, page_size, D)
        rows[page, :, tile, _kv4_row(n) if is_key else n] = w
        pairs[page, :, tile, _kv4_row(n)] = torch.stack([scale, low], -1).flatten(2).contiguous().view(torch.uint8)


def kv_read_int4(k_cache, v_cache, block_table, positions, seq_ids, head_dim: int, dtype=torch.bfloat16):
    """The rows at (seq_ids, positions): k, v [tokens, kv_heads, D]; zeros for tokens without a page."""
    D, H = head_dim, k_cache.shape[1]
    page_size = kv4_check(k_cache, v_cache, block_table, H, D)
    if positions.numel() != seq_ids.numel():
        raise ValueError("kv_read_int4: one position and one sequence per token")
    page, tile, n, ok = kv4_places(block_table, page_size, k_cache.shape[0], positions, seq_ids)
    at = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=k_cache.device)
    out = []
    for cache, is_key in ((k_cache, True), (v_cache, False)):
        rows, pairs = _kv4_views(cache, page_size, D)
        if cache.shape[0] == 0:
            out.append(torch.zeros(n.numel(), H, D, dtype=dtype, device=cache.device))
            continue
        w = rows[page, :, tile, _kv4_row(n) if is_key else n].contiguous().view(torch.int32).long() & 0xFFFFFFFF
        if is_key:
            w = (w >> 3 | w << 29) & 0xFFFFFFFF
        w = w.gather(2, _kv4_word_order(D, n, is_key)[:, None].expand_as(w))
        code = (w[..., None] >> at & 15).flatten(2).float().unflatten(-1, (-1, KV4_GROUP))
        pair = pairs[page, :, tile, _kv4_row(n)].contiguous().view(torch.bfloat16).float().unflatten(-1, (-1, 2))
        x = kv4_values(code, pair[..., :1], pair[..., 1:], dtype).flatten(2)
        out.append(torch.where(ok[:, None, None], x, torch.zeros_like(x)))
    return out[0], out[1]


def paged_attn_int4(q, k_cache, v_cache, block_table, cu_q, kv_lens, scale: float):
    """Causal attention of packed new tokens q [T, heads, D] (sequence b: rows cu_q[b] .. cu_q[b + 1], the last of its
    kv_lens[b] keys) over 4-bit pages. A sequence without keys, and a query that sees none, give zeros; a key without a page
    is seen by none."""
    T, H, D = q.shape
    Hk = k_cache.shape[1]
    page_size = kv4_check(k_cache, v_cache, block_table, Hk, D)
    if Hk == 0 or H % Hk or cu_q.numel() != kv_lens.numel() + 1 or block_table.shape[0] < kv_lens.numel():
        raise ValueError("paged_attn_int4: heads in groups of the kv heads, cu_q with one entry more than kv_lens")
    out = torch.zeros_like(q)
    cu, lens = cu_q.tolist(), kv_lens.tolist()
    for b, n in enumerate(lens):
        a, e = cu[b], cu[b + 1]
        if e <= a or n <= 0:
            continue
        pos = torch.arange(n, device=q.device)
        k, v = kv_read_int4(k_cache, v_cache, block_table, pos, torch.full_like(pos, b), D, torch.float32)
        k, v = (x.repeat_interleave(H // Hk, 1) for x in (k, v))
        s = torch.einsum("qhd,khd->hqk", q[a:e].float(), k) * scale
        hidden = pos[None] > n - (e - a) + torch.arange(e - a, device=q.device)[:, None]
        hidden = hidden | ~kv4_places(block_table, page_size, k_cache.shape[0], pos, torch.full_like(pos, b))[3]
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        p = torch.where(hidden.all(-1)[:, None], torch.zeros_like(p), p)
        bad = ~v.isfinite()                    # left out where they are not seen: a weight of zero would not do
        o = torch.einsum("hqk,khd->qhd", p, v.masked_fill(bad, 0.0))
        if bad.any():
            o = o.masked_fill(torch.einsum("qk,khd->qhd", (~hidden).float(), bad.float()) > 0, math.nan)
        out[a:e] = o.to(q.dtype)
    return out
