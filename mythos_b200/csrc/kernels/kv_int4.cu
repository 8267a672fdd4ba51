// 4-bit paged KV cache: writing, reading back, and attention over it (format: kv_int4.cuh).
//
//   kv_append_int4            new K / V rows -> codes, scales and lows in their pages
//   kv_read_int4              tokens of the cache -> bf16 rows
//   paged_attn_decode_int4    one query token per sequence
//   paged_attn_prefill_int4   several new query tokens per sequence, causal, over everything in the pages
#include <climits>

#include "api.h"
#include "common.cuh"
#include "host_util.h"
#include "kv_int4.cuh"
#include "tc.cuh"

namespace mb {
namespace {

// ------------------------------------------------------------------------------------------------ write
// Four lanes share a group of 64 values, sixteen each; extremes travel as bf16 pairs (min and max that keep a NaN), codes
// leave as two words per lane. Moves 2 + 0.5625 bytes per value. 1536 threads a SM hide the loads (2048: spills, 21.4 -> 22.6 us
// for 4 x 2048 tokens of 8 heads); blocks of 128 rather than 256 spread short calls better (999 tokens of 3 heads: 4.8 -> 4.5 us).
constexpr int KV4_APPEND = 128;
template <int D>
__global__ void __launch_bounds__(KV4_APPEND, 12)
kv_append_int4_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, uint8_t* __restrict__ k_cache,
                      uint8_t* __restrict__ v_cache, const Kv4Pages pages, const int* __restrict__ positions,
                      const int* __restrict__ seq_ids, int units, Kv4Div by_token, long long k_stride, long long v_stride) {
  using L = KvInt4<D>;
  constexpr int PER_ROW = D / 16, GR = L::GROUPS;
  // units is a multiple of the lanes of a row: groups and rows are here as a whole
  const unsigned mask = 0xFu << (threadIdx.x & 28), row_mask = ((1u << PER_ROW) - 1u) << (threadIdx.x & (32 - PER_ROW));
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= units) return;
  const int t = by_token(i), c = i - t * pages.kv_heads * PER_ROW;
  const int head = c / PER_ROW, g = (c % PER_ROW) >> 2, u = c & 3;
  const int seq = seq_ids[t], pos = positions[t];
  bf16x8 x[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    x[0][h] = ldg8(k, t * k_stride + c * 16 + 8 * h);
    x[1][h] = ldg8(v, t * v_stride + c * 16 + 8 * h);
  }
  const int tile = pages.tile(seq, pos, head);
  const int n = pos & 15;                                        // (page sizes are multiples of 16)
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    __nv_bfloat162 lo = x[s][0].v[0], hi = lo;
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      lo = __hmin2_nan(lo, x[s][e >> 2].v[e & 3]);
      hi = __hmax2_nan(hi, x[s][e >> 2].v[e & 3]);
    }
#pragma unroll
    for (int o = 2; o > 0; o >>= 1) {
      lo = __hmin2_nan(lo, __shfl_xor_sync(mask, lo, o));
      hi = __hmax2_nan(hi, __shfl_xor_sync(mask, hi, o));
    }
    if (tile < 0) continue;
    float scale, low;
    const uint32_t pair = kv4_make_pair(__hmin_nan(lo.x, lo.y), __hmax_nan(hi.x, hi.y), scale, low);
    const float inv = __frcp_rn(scale);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = kv4_word(x[s][h], scale, low, inv);
    uint8_t* dst = (s ? v_cache : k_cache) + (long long)tile * L::TILE_BYTES;
    if (s == 0) {
      *reinterpret_cast<uint2*>(dst + kv4_key_word<D>(n, g, 2 * u)) = make_uint2(kv4_rotate(w[0]), kv4_rotate(w[1]));
    } else if (GR == 1) {
      *reinterpret_cast<uint2*>(dst + kv4_value_word<D>(n, g, 2 * u)) = make_uint2(w[0], w[1]);
    } else {
      // the two groups' words of a place lie side by side: this lane stores those of place 2 u + g
      const uint32_t other = __shfl_xor_sync(row_mask, g ? w[0] : w[1], 4);
      *reinterpret_cast<uint2*>(dst + kv4_value_word<D>(n, 0, 2 * u + g)) = g ? make_uint2(other, w[1]) : make_uint2(w[0], other);
    }
    if (u == 0) *reinterpret_cast<uint32_t*>(dst + kv4_pair<D>(n, g)) = pair;
  }
}

// ------------------------------------------------------------------------------------------------ read
// Eight values of a row. 0x4300 | code is the bf16 number 128 + code; taking 128 off is exact, and the fused bf16
// multiply-add rounds scale * code + low once.
__device__ __forceinline__ bf16x8 kv4_expand(uint32_t w, uint32_t pair) {
  const __nv_bfloat16 s = __ushort_as_bfloat16((unsigned short)pair), low = __ushort_as_bfloat16((unsigned short)(pair >> 16));
  const __nv_bfloat162 s2(s, s), low2(low, low), k128(__ushort_as_bfloat16(0x4300), __ushort_as_bfloat16(0x4300));
  bf16x8 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = (w >> (4 * i) & 0x000F000Fu) | 0x43004300u;
    y.v[i] = __hfma2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), k128), s2, low2);
  }
  return y;
}

// Tokens named by (sequence, position): the counterpart of the append. One word per thread, tensor and step, so that a warp's
// stores are 512 bytes side by side (two words per thread left half-written 32-byte sectors between its stores: 174 us
// instead of 62 for 8 ragged sequences of up to 8192 tokens); four steps at once (50 us), because a word is behind three
// loads that wait for one another (position, page, code). Calls that one step per thread spreads over the GPU at once take one
// (1000 tokens of 5 heads: 2.8 us against 3.5).
constexpr int KV4_READ = 4;
template <int D, int STEPS>
__global__ void __launch_bounds__(256)
kv_read_int4_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const Kv4Pages pages,
                    const int* __restrict__ positions, const int* __restrict__ seq_ids, __nv_bfloat16* __restrict__ k,
                    __nv_bfloat16* __restrict__ v, int units, Kv4Div by_token) {
  using L = KvInt4<D>;
  constexpr int PER_ROW = D / 8;
  const int first = blockIdx.x * (256 * STEPS) + threadIdx.x;
  uint32_t kw[STEPS], vw[STEPS], kp[STEPS], vp[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int i = first + 256 * s;
    kw[s] = vw[s] = kp[s] = vp[s] = 0u;                          // a token without a page reads as zeros
    if (i < units) {
      const int t = by_token(i), c = i - t * pages.kv_heads * PER_ROW;
      const int head = c / PER_ROW, g = (c % PER_ROW) >> 3, u = c & 7;
      const int pos = positions[t], tile = pages.tile(seq_ids[t], pos, head), n = pos & 15;
      if (tile >= 0) {
        const uint8_t* ks = k_cache + (long long)tile * L::TILE_BYTES;
        const uint8_t* vs = v_cache + (long long)tile * L::TILE_BYTES;
        kw[s] = *reinterpret_cast<const uint32_t*>(ks + kv4_key_word<D>(n, g, u));
        vw[s] = *reinterpret_cast<const uint32_t*>(vs + kv4_value_word<D>(n, g, u));
        kp[s] = *reinterpret_cast<const uint32_t*>(ks + kv4_pair<D>(n, g));
        vp[s] = *reinterpret_cast<const uint32_t*>(vs + kv4_pair<D>(n, g));
      }
    }
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int i = first + 256 * s;
    if (i < units) {
      stg8(k, i * 8LL, kv4_expand(kv4_unrotate(kw[s]), kp[s]));
      stg8(v, i * 8LL, kv4_expand(vw[s], vp[s]));
    }
  }
}

Kv4Pages kv4_pages(const KvInt4Cache& c) {
  return {c.block_table, c.n_seqs, c.max_pages, c.n_pages, c.kv_heads, c.page_size, kv4_div(c.page_size)};
}

void kv4_check(const KvInt4Cache& c, const char* who) {
  MB_REQUIRE(c.head_dim == 64 || c.head_dim == 128, std::string(who) + ": head_dim must be 64 or 128");
  MB_REQUIRE(c.page_size > 0 && c.page_size % 16 == 0, std::string(who) + ": page size must be a multiple of 16 tokens");
  MB_REQUIRE(c.kv_heads > 0, std::string(who) + ": at least one kv head");
  MB_REQUIRE((long long)c.n_pages * c.kv_heads * (c.page_size / 16) < (1LL << 31), std::string(who) + ": too many tiles in the cache");
  MB_REQUIRE(((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15) == 0,
             std::string(who) + ": caches must be 16-byte aligned");
}

// Threads of an append or a read, one per `values` of each tensor.
int kv4_units(const KvInt4Cache& c, int tokens, int values, const char* who) {
  const long long n = (long long)tokens * c.kv_heads * (c.head_dim / values);
  MB_REQUIRE(n < (1LL << 31) - 256 * KV4_READ, std::string(who) + ": too many tokens in one call");
  return (int)n;
}

}  // namespace

void kv_append_int4(const KvInt4Cache& c, const void* k, const void* v, const int* positions, const int* seq_ids, int tokens,
                    long long k_stride, long long v_stride, cudaStream_t stream) {
  kv4_check(c, "kv_append_int4");
  MB_REQUIRE(k_stride % 8 == 0 && v_stride % 8 == 0, "kv_append_int4: token strides must be multiples of 8 elements");
  MB_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0, "kv_append_int4: k and v must be 16-byte aligned");
  if (tokens == 0) return;
  const int units = kv4_units(c, tokens, 16, "kv_append_int4"), per_token = c.kv_heads * (c.head_dim / 16);
  const auto go = [&](auto kern) {
    kern<<<(units + KV4_APPEND - 1) / KV4_APPEND, KV4_APPEND, 0, stream>>>(
        (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (uint8_t*)c.k, (uint8_t*)c.v, kv4_pages(c), positions, seq_ids, units, kv4_div(per_token), k_stride, v_stride);
  };
  if (c.head_dim == 128) go(kv_append_int4_kernel<128>);
  else go(kv_append_int4_kernel<64>);
  count_launch();
  check_launch();
}

void kv_read_int4(const KvInt4Cache& c, const int* positions, const int* seq_ids, int tokens, void* k, void* v, cudaStream_t stream) {
  kv4_check(c, "kv_read_int4");
  MB_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0, "kv_read_int4: k and v must be 16-byte aligned");
  if (tokens == 0) return;
  const int units = kv4_units(c, tokens, 8, "kv_read_int4"), per_token = c.kv_heads * (c.head_dim / 8);
  const bool small = units <= 8 * 256 * sm_count();
  const int per = 256 * (small ? 1 : KV4_READ);
  const auto go = [&](auto kern) {
    kern<<<(units + per - 1) / per, 256, 0, stream>>>((const uint8_t*)c.k, (const uint8_t*)c.v, kv4_pages(c), positions, seq_ids,
                                                      (__nv_bfloat16*)k, (__nv_bfloat16*)v, units, kv4_div(per_token));
  };
  if (c.head_dim == 128) {
    if (small) go(kv_read_int4_kernel<128, 1>);
    else go(kv_read_int4_kernel<128, KV4_READ>);
  } else {
    if (small) go(kv_read_int4_kernel<64, 1>);
    else go(kv_read_int4_kernel<64, KV4_READ>);
  }
  count_launch();
  check_launch();
}

namespace {
void kv4_workspace(const void* workspace, long long bytes) {
  MB_REQUIRE(bytes == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
             "attention over 4-bit pages: workspace missing or not 16-byte aligned");
}
}  // namespace

long long paged_attn_decode_int4_workspace(const KvInt4Cache& c, int batch, int heads) {
  return batch == 0 || c.kv_heads <= 0 ? 0 : few_query_int4_workspace(c, batch, 1, heads);
}

long long paged_attn_prefill_int4_workspace(const KvInt4Cache& c, int batch, int total_q, int max_q, int max_kv, int heads) {
  if (batch == 0 || c.kv_heads <= 0) return 0;
  if (!few_query_int4_takes(batch, max_q, max_kv, heads, c.kv_heads, c.head_dim))
    return prompt_int4_workspace(batch, total_q, max_q, max_kv, heads, c.kv_heads, c.head_dim);
  return few_query_int4_workspace(c, batch, max_q, heads);
}

void paged_attn_decode_int4(const KvInt4Cache& c, const void* q, long long q_stride, const int* context_lens, void* out, int batch,
                            int heads, float scale, void* workspace, int* status, cudaStream_t stream) {
  kv4_check(c, "paged_attn_decode_int4");
  MB_REQUIRE(heads > 0 && heads % c.kv_heads == 0, "paged_attn_decode_int4: heads must be a multiple of kv_heads");
  MB_REQUIRE(q_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0,
             "paged_attn_decode_int4: q must be 16-byte aligned with a token stride of a multiple of 8 elements");
  MB_REQUIRE(scale > 0.f, "paged_attn_decode_int4: scale must be positive");
  if (batch == 0) return;
  kv4_workspace(workspace, paged_attn_decode_int4_workspace(c, batch, heads));
  few_query_int4(c, q, q_stride, nullptr, context_lens, out, (long long)heads * c.head_dim, batch, batch, 1, INT_MAX, heads, scale,
                 workspace, status, stream);
}

void paged_attn_prefill_int4(const KvInt4Cache& c, const void* q, long long q_stride, const int* cu_q, const int* kv_lens, void* out,
                             long long o_stride, int batch, int total_q, int max_q, int max_kv, int heads, float scale,
                             void* workspace, int* status, cudaStream_t stream) {
  kv4_check(c, "paged_attn_prefill_int4");
  MB_REQUIRE(heads > 0 && heads % c.kv_heads == 0, "paged_attn_prefill_int4: heads must be a multiple of kv_heads");
  MB_REQUIRE(q_stride % 8 == 0 && o_stride % 8 == 0 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
             "paged_attn_prefill_int4: q and out must be 16-byte aligned with token strides of multiples of 8 elements");
  MB_REQUIRE(scale > 0.f, "paged_attn_prefill_int4: scale must be positive");
  if (batch == 0) return;         // (without queries: the lengths are still looked at)
  kv4_workspace(workspace, paged_attn_prefill_int4_workspace(c, batch, total_q, max_q, max_kv, heads));
  if (few_query_int4_takes(batch, max_q, max_kv, heads, c.kv_heads, c.head_dim)) {
    few_query_int4(c, q, q_stride, cu_q, kv_lens, out, o_stride, batch, total_q, max_q, max_kv, heads, scale, workspace, status, stream);
    return;
  }
  prompt_int4(c, q, q_stride, cu_q, kv_lens, out, o_stride, batch, total_q, max_q, max_kv, heads, scale, workspace, status, stream);
}

}  // namespace mb
