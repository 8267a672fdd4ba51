// 4-bit paged KV cache: writing, reading back, and attention over it (format: kv_int4.cuh).
//
//   kv_append_int4            new K / V rows -> codes, scales and lows in their pages
//   kv_read_int4              tokens of the cache -> bf16 rows
//   paged_attn_decode_int4    one query token per sequence
//   paged_attn_prefill_int4   several new query tokens per sequence, causal, over everything in the pages
#include "api.h"
#include "common.cuh"
#include "host_util.h"
#include "kv_int4.cuh"
#include "tc.cuh"

namespace mb {
namespace {

// ------------------------------------------------------------------------------------------------ write
// Eight lanes share a group of 64 values, one 16-byte load each; extremes travel as bf16 pairs (min and max
// that keep a NaN), codes leave as one word per lane. Moves 2 + 0.5625 bytes per value.
template <int D>
__global__ void __launch_bounds__(256)
kv_append_int4_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, uint8_t* __restrict__ k_cache,
                      uint8_t* __restrict__ v_cache, const int* __restrict__ block_table, const int* __restrict__ positions,
                      const int* __restrict__ seq_ids, long long units, int kv_heads, int page_size, int max_pages, int n_seqs,
                      int n_pages, long long k_stride, long long v_stride) {
  using L = KvInt4<D>;
  constexpr int PER_ROW = D / 8;
  const int per_tok = kv_heads * PER_ROW;
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < units; i += step) {
    const unsigned mask = 0xFFu << (threadIdx.x & 24);           // units is a multiple of 8: a group is here as a whole
    const int t = (int)(i / per_tok), c = (int)(i % per_tok);
    const int head = c / PER_ROW, g = (c % PER_ROW) >> 3, u = c & 7;
    const bf16x8 kx = ldg8(k, t * k_stride + (long long)c * 8), vx = ldg8(v, t * v_stride + (long long)c * 8);
    __nv_bfloat162 lo[2], hi[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bf16x8& x = s ? vx : kx;
      lo[s] = __hmin2_nan(__hmin2_nan(x.v[0], x.v[1]), __hmin2_nan(x.v[2], x.v[3]));
      hi[s] = __hmax2_nan(__hmax2_nan(x.v[0], x.v[1]), __hmax2_nan(x.v[2], x.v[3]));
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        lo[s] = __hmin2_nan(lo[s], __shfl_xor_sync(mask, lo[s], o));
        hi[s] = __hmax2_nan(hi[s], __shfl_xor_sync(mask, hi[s], o));
      }
    }
    const int seq = seq_ids[t], pos = positions[t];
    const int tile = seq >= 0 && seq < n_seqs
        ? kv4_tile(block_table + (long long)seq * max_pages, pos, max_pages, n_pages, page_size, kv_heads, head) : -1;
    if (tile < 0) continue;
    const int n = (pos % page_size) & 15;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float f[8], scale, low;
      unpack8(s ? vx : kx, f);
      const uint32_t pair = kv4_make_pair(__hmin_nan(lo[s].x, lo[s].y), __hmax_nan(hi[s].x, hi[s].y), scale, low);
      const uint32_t w = kv4_word(f, scale, low);
      uint8_t* dst = (s ? v_cache : k_cache) + (long long)tile * L::TILE_BYTES;
      if (s == 0) *reinterpret_cast<uint32_t*>(dst + kv4_key_word<D>(n, g, u)) = kv4_rotate(w);
      else *reinterpret_cast<uint32_t*>(dst + kv4_value_word<D>(n, g, u)) = w;
      if (u == 0) *reinterpret_cast<uint32_t*>(dst + kv4_pair<D>(n, g)) = pair;
    }
  }
}

// ------------------------------------------------------------------------------------------------ read
// Eight values of a row: scale * code + low, rounded once (the product of a bf16 and a 4-bit integer is exact
// in fp32).
__device__ __forceinline__ bf16x8 kv4_expand(uint32_t w, uint32_t pair) {
  const float s = kv4_scale(pair), low = kv4_low(pair);
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = fmaf((float)((w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u), s, low);
  return pack8(f);
}

// Tokens named by (sequence, position): the counterpart of the append. One word per thread and tensor.
template <int D>
__global__ void __launch_bounds__(256)
kv_read_int4_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const int* __restrict__ block_table,
                    const int* __restrict__ positions, const int* __restrict__ seq_ids, __nv_bfloat16* __restrict__ k,
                    __nv_bfloat16* __restrict__ v, long long units, int kv_heads, int page_size, int max_pages, int n_seqs,
                    int n_pages) {
  using L = KvInt4<D>;
  constexpr int PER_ROW = D / 8;
  const int per_tok = kv_heads * PER_ROW;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < units; i += (long long)gridDim.x * blockDim.x) {
    const int t = (int)(i / per_tok), c = (int)(i % per_tok);
    const int head = c / PER_ROW, g = (c % PER_ROW) >> 3, u = c & 7;
    const int seq = seq_ids[t], pos = positions[t];
    const int tile = seq >= 0 && seq < n_seqs
        ? kv4_tile(block_table + (long long)seq * max_pages, pos, max_pages, n_pages, page_size, kv_heads, head) : -1;
    uint32_t kw = 0u, vw = 0u, kp = 0u, vp = 0u;                 // a token without a page reads as zeros
    if (tile >= 0) {
      const int n = (pos % page_size) & 15;
      const uint8_t* ks = k_cache + (long long)tile * L::TILE_BYTES;
      const uint8_t* vs = v_cache + (long long)tile * L::TILE_BYTES;
      kw = kv4_unrotate(*reinterpret_cast<const uint32_t*>(ks + kv4_key_word<D>(n, g, u)));
      vw = *reinterpret_cast<const uint32_t*>(vs + kv4_value_word<D>(n, g, u));
      kp = *reinterpret_cast<const uint32_t*>(ks + kv4_pair<D>(n, g));
      vp = *reinterpret_cast<const uint32_t*>(vs + kv4_pair<D>(n, g));
    }
    stg8(k, i * 8, kv4_expand(kw, kp));
    stg8(v, i * 8, kv4_expand(vw, vp));
  }
}

void kv4_check(const KvInt4Cache& c, const char* who) {
  MB_REQUIRE(c.head_dim == 64 || c.head_dim == 128, std::string(who) + ": head_dim must be 64 or 128");
  MB_REQUIRE(c.page_size > 0 && c.page_size % 16 == 0, std::string(who) + ": page size must be a multiple of 16 tokens");
  MB_REQUIRE(c.kv_heads > 0, std::string(who) + ": at least one kv head");
  MB_REQUIRE((long long)c.n_pages * c.kv_heads * (c.page_size / 16) < (1LL << 31), std::string(who) + ": too many tiles in the cache");
  MB_REQUIRE(((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15) == 0,
             std::string(who) + ": caches must be 16-byte aligned");
}

int kv4_grid(long long units, int per_sm) {
  const long long g = (units + 255) / 256, cap = (long long)sm_count() * per_sm;
  return (int)(g < cap ? g : cap);
}

}  // namespace

void kv_append_int4(const KvInt4Cache& c, const void* k, const void* v, const int* positions, const int* seq_ids, int tokens,
                    long long k_stride, long long v_stride, cudaStream_t stream) {
  kv4_check(c, "kv_append_int4");
  MB_REQUIRE(k_stride % 8 == 0 && v_stride % 8 == 0, "kv_append_int4: token strides must be multiples of 8 elements");
  MB_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0, "kv_append_int4: k and v must be 16-byte aligned");
  if (tokens == 0) return;
  const long long units = (long long)tokens * c.kv_heads * (c.head_dim / 8);
  const auto go = [&](auto kern) {
    kern<<<kv4_grid(units, 16), 256, 0, stream>>>((const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (uint8_t*)c.k, (uint8_t*)c.v,
                                                  c.block_table, positions, seq_ids, units, c.kv_heads, c.page_size, c.max_pages,
                                                  c.n_seqs, c.n_pages, k_stride, v_stride);
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
  const long long units = (long long)tokens * c.kv_heads * (c.head_dim / 8);
  const auto go = [&](auto kern) {
    kern<<<kv4_grid(units, 16), 256, 0, stream>>>((const uint8_t*)c.k, (const uint8_t*)c.v, c.block_table, positions, seq_ids,
                                                  (__nv_bfloat16*)k, (__nv_bfloat16*)v, units, c.kv_heads, c.page_size,
                                                  c.max_pages, c.n_seqs, c.n_pages);
  };
  if (c.head_dim == 128) go(kv_read_int4_kernel<128>);
  else go(kv_read_int4_kernel<64>);
  count_launch();
  check_launch();
}

namespace {
void kv4_workspace(const void* workspace, long long bytes) {
  MB_REQUIRE(bytes == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
             "attention over 4-bit pages: workspace missing or not 16-byte aligned");
}
bool p4_few(int max_q, int group) { return (long long)max_q * group <= P4_FEW_COLUMNS; }
}  // namespace

long long paged_attn_int4_workspace(const KvInt4Cache& c, int batch, int total_q, int max_q, int max_kv, int heads) {
  if (batch == 0 || max_q == 0 || c.kv_heads <= 0) return 0;
  const int G = heads / c.kv_heads;
  if (!p4_few(max_q, G)) return prompt_int4_workspace(batch, total_q, max_kv, heads, c.kv_heads, c.head_dim);
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
  kv4_workspace(workspace, paged_attn_int4_workspace(c, batch, batch, 1, 0, heads));
  few_query_int4(c, q, q_stride, nullptr, context_lens, out, (long long)heads * c.head_dim, batch, batch, 1, heads, scale, workspace,
                 status, stream);
}

void paged_attn_prefill_int4(const KvInt4Cache& c, const void* q, long long q_stride, const int* cu_q, const int* kv_lens, void* out,
                             long long o_stride, int batch, int total_q, int max_q, int max_kv, int heads, float scale,
                             void* workspace, int* status, cudaStream_t stream) {
  kv4_check(c, "paged_attn_prefill_int4");
  MB_REQUIRE(heads > 0 && heads % c.kv_heads == 0, "paged_attn_prefill_int4: heads must be a multiple of kv_heads");
  MB_REQUIRE(q_stride % 8 == 0 && o_stride % 8 == 0 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
             "paged_attn_prefill_int4: q and out must be 16-byte aligned with token strides of multiples of 8 elements");
  MB_REQUIRE(scale > 0.f, "paged_attn_prefill_int4: scale must be positive");
  if (batch == 0 || total_q == 0 || max_q == 0) return;
  kv4_workspace(workspace, paged_attn_int4_workspace(c, batch, total_q, max_q, max_kv, heads));
  if (p4_few(max_q, heads / c.kv_heads)) {
    few_query_int4(c, q, q_stride, cu_q, kv_lens, out, o_stride, batch, total_q, max_q, heads, scale, workspace, status, stream);
    return;
  }
  prompt_int4(c, q, q_stride, cu_q, kv_lens, out, o_stride, batch, total_q, max_q, max_kv, heads, scale, workspace, status, stream);
}

}  // namespace mb
