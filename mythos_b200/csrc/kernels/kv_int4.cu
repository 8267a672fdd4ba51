// 4-bit paged KV cache: writing, reading back, and attention over it (format: kv_int4.cuh).
//
//   kv_append_int4            new K / V rows -> codes, scales and lows in their pages
//   kv_read_int4              tokens of the cache -> bf16 rows
//   paged_attn_decode_int4    one query token per sequence
//   paged_attn_prefill_int4   several new query tokens per sequence, causal, over everything in the pages
#include <cuda_fp16.h>

#include <algorithm>

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

// ------------------------------------------------------------------------------------------------ attention
// One (sequence, kv head, block of COLS query columns) per cluster; the CTAs of the cluster split its tokens. A column
// is one (query token, head of the group) pair: column c is head c % G of token c / G. Four warps per CTA; warp w
// takes every fourth chunk (32 tokens, two tiles) of its CTA's range through a ring of its own, filled with one bulk copy per
// tile for K and one for V.
//
// What bounds it is the integer pipe (half rate) that takes the codes apart, so operands are formed by one AND each:
// the low eleven bits of an fp16 are linear in its value (subnormals and the first normal binade share one step,
// 2^-24), so a nibble anywhere in them is its code times a power of two. Keys: bits 3-6 (code 2^-21) and 7-10 (code 2^-17)
// of a rotated word, then the word rotated by eight; queries of the second kind are multiplied by 2^-4. Values: bits 0-3
// (2^-24) and 4-7 (2^-20) of two tokens' halves side by side; they are different output values, scaled at the end.
//
// Scores: q . k = sum over groups of scale (q_g . c_g) + low sum(q_g), the product exact in fp16 (a query column is divided
// by a power of two first, so that its bf16 values fit). Values: o = sum_t (p_t scale_t) (c_t - 8) + sum_t p_t (low_t + 8
// scale_t): the codes are centred (one packed subtraction on the idle FMA pipe), because this sum runs over the whole
// context and the tensor cores truncate what they add; the second sum is a scalar per column and group in fp32.
// p_t scale_t is rounded to fp16 (2^-12 of each term); the running reference M is the maximum of the scores plus the
// exponent of the chunk's values, so it fits whatever the values' size. Everything else is fp32. mma.sync rather than tcgen05:
// with 8 columns a 128-row tile would be filled to a sixteenth, and the codes would have to go through shared memory
// once more.
//
// The CTAs of a cluster merge their partial softmax states through distributed shared memory: no scratch, no
// counters, one result for the same inputs, and calls on several streams share nothing.
constexpr int P4_WARPS = 4;
constexpr int P4_THREADS = 32 * P4_WARPS;
constexpr int P4_CHUNK = 32;      // tokens

template <int D, int COLS>
struct P4Cfg {
  using L = KvInt4<D>;
  static constexpr int STAGES = 3;
  static constexpr int HALF = 2 * L::TILE_BYTES;              // K (or V) of a chunk
  static constexpr int STAGE = 2 * HALF;
  static constexpr int WARP_BYTES = STAGES * STAGE;
  static constexpr int OFF_BAR = P4_WARPS * WARP_BYTES;
  static constexpr int OFF_ML = OFF_BAR + P4_WARPS * STAGES * 8 + 16;               // m, l: [warps][COLS] each
  static constexpr int OFF_Z = OFF_ML + 2 * P4_WARPS * COLS * 4;                    // [warps][COLS][groups]
  static constexpr int OFF_CTA = OFF_Z + P4_WARPS * COLS * L::GROUPS * 4;           // m, l of the CTA
  static constexpr int BYTES = OFF_CTA + 2 * COLS * 4 + 128;
  static_assert(COLS * D * 4 <= WARP_BYTES, "a warp's output state is staged in its own (drained) ring");
};

__device__ __forceinline__ void p4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void p4_bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t p4_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void p4_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t p4_mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float p4_ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t p4_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float p4_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
struct P4Args {
  const __nv_bfloat16* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const int* block_table;
  const int* kv_lens;
  const int* cu_q;          // first query row of every sequence, or null: one query token per sequence
  __nv_bfloat16* out;
  long long q_stride, o_stride;
  int G, kv_heads, total_q, page_size, max_pages, n_pages, splits;
  float scale_log2;
  int* status;
};

// A warp's running state. Thread (r, t) of the warp holds columns 2 t and 2 t + 1 of every block of eight.
template <int D, int COLS>
struct P4State {
  static constexpr int NB = COLS / 8, GR = KvInt4<D>::GROUPS;
  uint32_t qb[NB][GR][8];                 // B operand: column r
  float qsum[NB][GR][2], factor[NB][2];   // of columns 2 t, 2 t + 1, as everything below
  int limit[NB][2];
  float o[NB][GR][4][4];                  // units of 2^-24 (even i) and 2^-20
  float z[NB][GR][2], m[NB][2], l[NB][2];
};

__device__ __forceinline__ uint32_t p4_transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// One chunk: tile u (0, 1) at `at` + u * TILE_BYTES for K, HALF behind for V; tok0: its first token.
// MASK: some token is not seen by some column (visible: those seen by any), or not held at all.
template <int D, int COLS, bool MASK>
__device__ __forceinline__ void p4_chunk(P4State<D, COLS>& s, const uint8_t* at, int tok0, int lane, int visible, uint32_t absent) {
  using L = KvInt4<D>;
  using C = P4Cfg<D, COLS>;
  constexpr int GR = L::GROUPS, NB = COLS / 8;
  const int r = lane >> 2, t = lane & 3;
  // ---- scores: rows of the product are key rows 8 j + r of a tile, columns 2 t + c
  float sc[2][NB][GR][4];                         // [tile][block][group][2 j + c]
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t kw[2][GR][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* kp = at + u * L::TILE_BYTES + (8 * j + r) * L::ROW + t * (8 * GR);
      if constexpr (GR == 2) {
        const uint4 x = *reinterpret_cast<const uint4*>(kp);
        kw[j][0][0] = x.x; kw[j][0][1] = x.y; kw[j][1][0] = x.z; kw[j][1][1] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(kp);
        kw[j][0][0] = x.x; kw[j][0][1] = x.y;
      }
    }
#pragma unroll
    for (int g = 0; g < GR; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w0 = kw[0][g][h], w1 = kw[1][g][h], v0 = __funnelshift_r(w0, w0, 8), v1 = __funnelshift_r(w1, w1, 8);
        const uint32_t a0 = w0 & 0x00780078u, a1 = w1 & 0x00780078u, a2 = w0 & 0x07800780u, a3 = w1 & 0x07800780u;
        const uint32_t b0 = v0 & 0x00780078u, b1 = v1 & 0x00780078u, b2 = v0 & 0x07800780u, b3 = v1 & 0x07800780u;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float (&c)[4] = sc[u][nb][g];
          if (h == 0) c[0] = c[1] = c[2] = c[3] = 0.f;
          p4_mma(c, a0, a1, a2, a3, s.qb[nb][g][4 * h], s.qb[nb][g][4 * h + 1]);
          p4_mma(c, b0, b1, b2, b3, s.qb[nb][g][4 * h + 2], s.qb[nb][g][4 * h + 3]);
        }
      }
  }
  // ---- exponent of the chunk's values: one group of one token per thread and tile
  float mag = 0.f;
#pragma unroll
  for (int u = 0; u < GR; ++u) {                  // (one group a token: the warp's halves take the two tiles)
    const int tile = GR == 2 ? u : lane >> 4, row = GR == 2 ? lane >> 1 : lane & 15, g = GR == 2 ? lane & 1 : 0;
    const uint32_t p = *reinterpret_cast<const uint32_t*>(at + C::HALF + tile * L::TILE_BYTES + L::OFF_PAIR + row * L::PAIR + 4 * g);
    const float top = fmaf(15.f, kv4_scale(p), kv4_low(p));
    bool use = true;                              // (what every column sees may be infinite: the result is no number then)
    if (MASK) {                                   // a place behind the context may hold anything
      const int n = (row & 8) + ((row >> 1) & 3) + ((row & 1) << 2);       // token at this pair row
      use = kv4_finite(p) && tok0 + 16 * tile + n < visible && !(absent >> tile & 1u);
    }
    mag = fmax3(mag, use ? fabsf(top) : 0.f, use ? fabsf(kv4_low(p)) : 0.f);
  }
  // p is kept up to 2^8 (and 2^6 more until the reference moves) times the inverse of the largest magnitude, which is at
  // least 7 scales: p times a scale then stays below 2^13, and is exact to 2^-12 over 24 octaves below. Bounded so that p, its
  // sum and its product with any value stay within fp32.
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(mag));
  const float ev = fminf(fmaxf(__uint_as_float(0x4B000000u | (bits >> 23)) - (8388608.f + 127.f), -80.f), 112.f) - 8.f;
  // ---- online softmax: scores relative to the reference; it moves only when one of them passes it by 2^6
  float x[2][NB][2][2];                           // [tile][block][j][c]
  float top = -INFINITY;
  const int tok_r = tok0 + ((r >> 1) & 3) + ((r & 1) << 2);                // token of key row r of the first tile; row r + 8: 8 on
  float mm[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 2; ++c) mm[nb][c] = s.m[nb][c] == -INFINITY ? 0.f : s.m[nb][c];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t kq[GR];
      const uint8_t* kp = at + u * L::TILE_BYTES + L::OFF_PAIR + (8 * j + r) * L::PAIR;
      if constexpr (GR == 2) {
        const uint2 y = *reinterpret_cast<const uint2*>(kp);
        kq[0] = y.x; kq[1] = y.y;
      } else {
        kq[0] = *reinterpret_cast<const uint32_t*>(kp);
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = kv4_low(kq[0]) * s.qsum[nb][0][c];
          if constexpr (GR == 2) v = fmaf(kv4_low(kq[1]), s.qsum[nb][1][c], v);
#pragma unroll
          for (int g = 0; g < GR; ++g) v = fmaf(kv4_scale(kq[g]), sc[u][nb][g][2 * j + c], v);
          v = fmaf(v, s.factor[nb][c], -mm[nb][c]);
          if (MASK && (tok_r + 16 * u + 8 * j >= s.limit[nb][c] || (absent >> u & 1u))) v = -INFINITY;
          x[u][nb][j][c] = v;
        }
    }
  bool first = false;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int c = 0; c < 2; ++c) first = first || s.m[nb][c] == -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) top = fmax3(top, x[u][nb][j][0], x[u][nb][j][1]);
  }
  if (__any_sync(0xffffffffu, first || top + ev > 6.f)) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float mx = fmaxf(fmax3(x[0][nb][0][c], x[0][nb][1][c], x[1][nb][0][c]), x[1][nb][1][c]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        mx += ev;                                 // relative to the reference used so far
        if (s.m[nb][c] == -INFINITY ? mx > -INFINITY : mx > 0.f) {
          const float alpha = s.m[nb][c] == -INFINITY ? 0.f : fast_exp2(-mx);
          s.m[nb][c] = mm[nb][c] + mx;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) x[u][nb][j][c] -= mx;
          s.l[nb][c] *= alpha;
#pragma unroll
          for (int g = 0; g < GR; ++g) {
            s.z[nb][g][c] *= alpha;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s.o[nb][g][i][c] *= alpha;
              s.o[nb][g][i][2 + c] *= alpha;
            }
          }
        }
      }
  }
  // ---- weights p scale as the B operand (k = tokens, n = columns): transposed in blocks of eight by eight. Odd key rows
  // are the tokens that enter with the complement of their codes.
  uint32_t pb[2][NB][GR][2];
  const uint32_t flip = (uint32_t)(r & 1) << 31;
  const float whole = (r & 1) ? -15.f : 0.f;      // low + 15 scale, the scale's sign already turned
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t vq[GR];
      const uint8_t* vp = at + C::HALF + u * L::TILE_BYTES + L::OFF_PAIR + (8 * j + r) * L::PAIR;
      if constexpr (GR == 2) {
        const uint2 y = *reinterpret_cast<const uint2*>(vp);
        vq[0] = y.x; vq[1] = y.y;
      } else {
        vq[0] = *reinterpret_cast<const uint32_t*>(vp);
      }
      float w[GR], b[GR];
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        w[g] = __uint_as_float(vq[g] << 16 ^ flip);
        b[g] = fmaf(whole, w[g], kv4_low(vq[g]));
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float p0 = fast_exp2(x[u][nb][j][0]), p1 = fast_exp2(x[u][nb][j][1]);
        s.l[nb][0] += p0;
        s.l[nb][1] += p1;
        // a token the column does not see may hold anything, behind the sequence's end too: it is left out, not
        // multiplied by zero
        const bool s0 = !MASK || x[u][nb][j][0] != -INFINITY, s1 = !MASK || x[u][nb][j][1] != -INFINITY;
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          if (MASK) {
            s.z[nb][g][0] += s0 ? p0 * b[g] : 0.f;
            s.z[nb][g][1] += s1 ? p1 * b[g] : 0.f;
          } else {
            s.z[nb][g][0] = fmaf(p0, b[g], s.z[nb][g][0]);
            s.z[nb][g][1] = fmaf(p1, b[g], s.z[nb][g][1]);
          }
          pb[u][nb][g][j] = p4_transpose(p4_half2(s0 ? p0 * w[g] : 0.f, s1 ? p1 * w[g] : 0.f));
        }
      }
    }
  // ---- values: the A operand holds values x tokens (t, t + 4, t + 8, t + 12: those of key rows 2 t, 2 t + 1 and 8 on)
  const int chunk = r ^ ((t >> 1) << 2);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t vw[2][2][GR];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint8_t* vp = at + C::HALF + u * L::TILE_BYTES + (t + 4 * (2 * j + e)) * L::ROW + chunk * (4 * GR);
        if constexpr (GR == 2) {
          const uint2 w = *reinterpret_cast<const uint2*>(vp);
          vw[j][e][0] = w.x; vw[j][e][1] = w.y;
        } else {
          vw[j][e][0] = *reinterpret_cast<const uint32_t*>(vp);
        }
      }
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      // halves of the two tokens' words side by side: lo holds values 0, 2, 4, 6 and hi values 1, 3, 5, 7 of both
      uint32_t lo0 = __byte_perm(vw[0][0][g], vw[0][1][g], 0x5410), hi0 = __byte_perm(vw[0][0][g], vw[0][1][g], 0x7632);
      uint32_t lo1 = __byte_perm(vw[1][0][g], vw[1][1][g], 0x5410), hi1 = __byte_perm(vw[1][0][g], vw[1][1][g], 0x7632);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i == 2) {
          lo0 >>= 8; hi0 >>= 8; lo1 >>= 8; hi1 >>= 8;
        }
        const uint32_t mask = (i & 1) ? 0x00F000F0u : 0x000F000Fu;
        const uint32_t a0 = (lo0 ^ 0xFFFF0000u) & mask, a1 = (hi0 ^ 0xFFFF0000u) & mask, a2 = (lo1 ^ 0xFFFF0000u) & mask,
                       a3 = (hi1 ^ 0xFFFF0000u) & mask;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) p4_mma(s.o[nb][g][i], a0, a1, a2, a3, pb[u][nb][g][0], pb[u][nb][g][1]);
      }
    }
  }
}

template <int D, int COLS>
__global__ void __launch_bounds__(P4_THREADS, COLS == 8 ? 4 : 2)
paged_attn_int4_kernel(const __grid_constant__ P4Args a) {
  using L = KvInt4<D>;
  using C = P4Cfg<D, COLS>;
  constexpr int GR = L::GROUPS, NB = COLS / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int b = blockIdx.x, hkv = blockIdx.y % a.kv_heads, col0 = blockIdx.y / a.kv_heads * COLS, split = blockIdx.z;
  const int row0 = a.cu_q ? a.cu_q[b] : b, q_len = a.cu_q ? a.cu_q[b + 1] - row0 : 1;
  const int n_cols = min(COLS, q_len * a.G - col0);
  if (n_cols <= 0) return;                       // the same for every CTA of the cluster
  const int kv_len = a.kv_lens[b];

  uint8_t* ring = smem + warp * C::WARP_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR) + warp * C::STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_BAR + P4_WARPS * C::STAGES * 8);
  float* s_m = reinterpret_cast<float*>(smem + C::OFF_ML);
  float* s_l = s_m + P4_WARPS * COLS;
  float* s_z = reinterpret_cast<float*>(smem + C::OFF_Z);
  float* s_cta = reinterpret_cast<float*>(smem + C::OFF_CTA);      // m[COLS], l[COLS]
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncthreads();

  // chunks of this CTA: what the last query of the block sees, cut into equal ranges
  const int first_q = col0 / a.G, last_q = (col0 + n_cols - 1) / a.G;
  const int visible = max(0, min(kv_len, kv_len - q_len + last_q + 1));       // to some column
  const int common = min(kv_len, kv_len - q_len + first_q + 1);               // to every column
  const int n_chunks = (visible + P4_CHUNK - 1) / P4_CHUNK;
  const int per = (n_chunks + a.splits - 1) / a.splits;
  const int chunk0 = split * per + warp, chunk_end = min(n_chunks, split * per + per);
  const int mine = (chunk_end - chunk0 + P4_WARPS - 1) / P4_WARPS;            // chunk0, + 4, ... (<= 0: none)
  const int* table = a.block_table + (long long)b * a.max_pages;

  // lane l holds tile l % 2 of the warp's chunk 16 n + l / 2 for the block n being issued, and of the next block:
  // its index, -1 without a page, -2 behind the visible tokens
  auto locate = [&](int i) {
    const int token = (chunk0 + P4_WARPS * i) * P4_CHUNK + (lane & 1) * 16;
    return i < mine && token < visible ? kv4_tile(table, token, a.max_pages, a.n_pages, a.page_size, a.kv_heads, hkv) : -2;
  };
  int ids = locate(lane >> 1), ids_next = locate(16 + (lane >> 1));
  uint32_t absent = 0u;                           // bits 2 s, 2 s + 1: tiles of stage s that were not loaded
  // lanes 0 .. 3 start one copy each: tile l % 2, K (l < 2) or V
  const uint8_t* base = (lane & 2) ? a.v_cache : a.k_cache;
  const uint32_t dst0 = smem_u32(ring) + ((lane & 2) ? C::HALF : 0) + (lane & 1) * L::TILE_BYTES;
  auto issue = [&](int i, int st) {               // all lanes: the warp's chunk i into stage st
    if (i > 0 && (i & 15) == 0) {
      ids = ids_next;
      ids_next = locate(i + 16 + (lane >> 1));
    }
    const int id = __shfl_sync(0xffffffffu, ids, 2 * (i & 15) + (lane & 1));
    const uint32_t gone = __ballot_sync(0xffffffffu, id < 0) & 3u;
    absent = (absent & ~(3u << (2 * st))) | gone << (2 * st);
    if (lane == 0) {
      if (gone == 3u) mbar_arrive(&full[st]);
      else mbar_arrive_expect_tx(&full[st], gone ? C::STAGE / 2 : C::STAGE);
    }
    if (lane < 4) {
      if (id >= 0) p4_bulk_load(dst0 + st * C::STAGE, base + (long long)id * L::TILE_BYTES, L::TILE_BYTES, &full[st]);
      else if (id == -1 && a.status) atomicCAS(a.status, 0, ST_BAD_ARG | (92 << 16));   // a token of the context without a page
    }
  };
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i)
    if (i < mine) issue(i, i);

  // Queries: the B operand, column r of every block; word h of group g holds values 64 g + 16 t + 8 h ..
  P4State<D, COLS> s;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int col = col0 + nb * 8 + r;
    const int qi = col / a.G, g_head = col % a.G;
    const bool live = nb * 8 + r < n_cols && (unsigned)(row0 + qi) < (unsigned)a.total_q;
    const int limit = live ? min(kv_len, kv_len - q_len + qi + 1) : 0;
    const __nv_bfloat16* qp = a.q + (long long)(row0 + qi) * a.q_stride + (long long)(hkv * a.G + g_head) * D + 16 * t;
    uint32_t raw[GR][8];
    float big = 0.f;
#pragma unroll
    for (int g = 0; g < GR; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (live) v = *reinterpret_cast<const uint4*>(qp + 64 * g + 8 * h);
        raw[g][4 * h] = v.x; raw[g][4 * h + 1] = v.y; raw[g][4 * h + 2] = v.z; raw[g][4 * h + 3] = v.w;
#pragma unroll
        for (int e = 0; e < 4; ++e)               // (both halves of a word)
          big = fmax3(big, fabsf(kv4_scale(raw[g][4 * h + e])), fabsf(kv4_low(raw[g][4 * h + e])));
      }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // the column's largest value in 2^14 .. 2^15
    const int eq = big > 0.f ? max(-100, min(113, (int)(__float_as_uint(big) >> 23) - 127 - 14)) : 0;
    const float down = p4_pow2(-eq), down4 = p4_pow2(-eq - 4), factor = a.scale_log2 * 0x1p21f * p4_pow2(eq);
    float qsum[GR];
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q0 = kv4_scale(raw[g][e]), q1 = kv4_low(raw[g][e]), f = (e & 1) ? down4 : down;
        s.qb[nb][g][e] = p4_half2(q0 * f, q1 * f);
        sum += q0 * down + q1 * down;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qsum[g] = sum * 0x1p-21f;                   // the products are in units of 2^-21
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {                 // what concerns columns 2 t + c sits in the threads of r = 2 t + c
      const int from = 8 * t + 4 * c;
      s.limit[nb][c] = __shfl_sync(0xffffffffu, limit, from);
      s.factor[nb][c] = __shfl_sync(0xffffffffu, factor, from);
      s.m[nb][c] = -INFINITY;
      s.l[nb][c] = 0.f;
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        s.qsum[nb][g][c] = __shfl_sync(0xffffffffu, qsum[g], from);
        s.z[nb][g][c] = 0.f;
      }
    }
#pragma unroll
    for (int g = 0; g < GR; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) s.o[nb][g][i][0] = s.o[nb][g][i][1] = s.o[nb][g][i][2] = s.o[nb][g][i][3] = 0.f;
  }

  bool ok = true;
  int st = 0, st_issue = C::STAGES - 1;
  uint32_t parity = 0u;
  int i = 0;
  for (; i < mine; ++i) {
    // the stage read in the step before is free now: every value read from it has gone through a product
    if (i + C::STAGES - 1 < mine) {
      issue(i + C::STAGES - 1, st_issue);
      st_issue = st_issue == C::STAGES - 1 ? 0 : st_issue + 1;
    }
    if (!__all_sync(0xffffffffu, mbar_try_wait(&full[st], parity))) {
      ok = mbar_wait(&full[st], parity, abort_flag, a.status, 93);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
    }
    const int tok = (chunk0 + P4_WARPS * i) * P4_CHUNK;
    const uint32_t gone = absent >> (2 * st) & 3u;
    const uint8_t* at = ring + st * C::STAGE;
    if (gone == 0u && tok + P4_CHUNK <= common) p4_chunk<D, COLS, false>(s, at, tok, lane, visible, 0u);
    else p4_chunk<D, COLS, true>(s, at, tok, lane, visible, gone);
    __syncwarp();
    if (++st == C::STAGES) {
      st = 0;
      parity ^= 1u;
    }
  }
  if (!ok)                                        // copies in flight land before the ring's memory goes away
    for (int k = 0; k < C::STAGES && i < mine; ++k, ++i) {
      mbar_drain(&full[st], parity);
      if (++st == C::STAGES) {
        st = 0;
        parity ^= 1u;
      }
    }

  // ---- the warp's state: row c of w_acc is column c, values in order
  float* w_acc = reinterpret_cast<float*>(ring);
  __syncwarp();
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = nb * 8 + 2 * t + c;
      float l = s.l[nb][c];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      if (r == 0) {
        s_m[warp * COLS + col] = ok ? s.m[nb][c] : -INFINITY;
        s_l[warp * COLS + col] = ok ? l : 0.f;
      }
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        float z = s.z[nb][g][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
        if (r == 0) s_z[(warp * COLS + col) * GR + g] = z;
        // values 64 g + 8 r + (0 .. 7), out of their units
        float (&o)[4][4] = s.o[nb][g];
        float* dst = w_acc + col * D + 64 * g + 8 * r;
        *reinterpret_cast<float4*>(dst) = make_float4(o[0][c] * 0x1p24f, o[0][2 + c] * 0x1p24f, o[1][c] * 0x1p20f, o[1][2 + c] * 0x1p20f);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(o[2][c] * 0x1p24f, o[2][2 + c] * 0x1p24f, o[3][c] * 0x1p20f, o[3][2 + c] * 0x1p20f);
      }
    }
  __syncthreads();

  // ---- the CTA's state, in the first warp's ring: every element is read and written by one thread
  float* acc = reinterpret_cast<float*>(smem);
  for (int idx = threadIdx.x; idx < COLS * D; idx += P4_THREADS) {
    const int c = idx / D, g = (idx % D) / 64;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < P4_WARPS; ++w) M = fmaxf(M, s_m[w * COLS + c]);
    float A = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < P4_WARPS; ++w) {
      const float lw = s_l[w * COLS + c];
      if (lw == 0.f) continue;                    // nothing seen (a NaN is not nothing)
      const float e = fast_exp2(s_m[w * COLS + c] - M);
      l += e * lw;
      A += e * (reinterpret_cast<const float*>(smem + w * C::WARP_BYTES)[idx] + s_z[(w * COLS + c) * GR + g]);
    }
    acc[idx] = A;
    if (idx % D == 0) {
      s_cta[c] = M;
      s_cta[COLS + c] = l;
    }
  }
  const int splits = a.splits;
  if (splits > 1) p4_cluster_sync();
  else __syncthreads();
  // ---- the cluster's state: every CTA writes a share of the block's outputs
  const uint32_t rank = splits > 1 ? p4_rank() : 0u;
  const int share = (COLS * D / 2 + splits - 1) / splits;        // in pairs of values
  const int end = min(COLS * D / 2, (int)(rank + 1) * share);
  for (int idx = rank * share + threadIdx.x; idx < end; idx += P4_THREADS) {
    const int c = 2 * idx / D, d = 2 * idx % D;
    if (c >= n_cols) break;
    float A0 = 0.f, A1 = 0.f, l = 0.f, M = -INFINITY;
    if (splits == 1) {
      A0 = acc[2 * idx];
      A1 = acc[2 * idx + 1];
      l = s_cta[COLS + c];
    } else {
      const uint32_t m_at = smem_u32(s_cta + c), l_at = smem_u32(s_cta + COLS + c), a_at = smem_u32(acc + 2 * idx);
#pragma unroll 4
      for (int p = 0; p < splits; ++p) {
        const float m = p4_ld_cluster(p4_mapa(m_at, p)), lp = p4_ld_cluster(p4_mapa(l_at, p));
        const float b0 = p4_ld_cluster(p4_mapa(a_at, p)), b1 = p4_ld_cluster(p4_mapa(a_at + 4, p));
        if (lp == 0.f) continue;
        const float Mn = fmaxf(M, m);
        const float e0 = fast_exp2(M - Mn), e1 = fast_exp2(m - Mn);
        A0 = A0 * e0 + e1 * b0;
        A1 = A1 * e0 + e1 * b1;
        l = l * e0 + e1 * lp;
        M = Mn;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;                  // nothing visible: zeros
    const int col = col0 + c, qi = col / a.G;
    if ((unsigned)(row0 + qi) >= (unsigned)a.total_q) break;
    __nv_bfloat16* dst = a.out + (long long)(row0 + qi) * a.o_stride + (long long)(hkv * a.G + col % a.G) * D + d;
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(A0 * inv, A1 * inv);
  }
  if (splits > 1) p4_cluster_sync();               // nobody leaves while a peer still reads its shared memory
}

// A kernel's shared-memory and cluster limits, raised once per device.
template <typename K>
void p4_configure(K kern, int smem, unsigned long long& seen) {
  int dev = 0;
  MB_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 64 && (seen >> dev & 1ull)) return;
  MB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  MB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (dev < 64) seen |= 1ull << dev;
}

template <int D, int COLS>
void p4_launch(P4Args& a, int batch, int max_q, cudaStream_t stream) {
  static unsigned long long seen = 0;
  p4_configure(paged_attn_int4_kernel<D, COLS>, P4Cfg<D, COLS>::BYTES, seen);
  const long long blocks = ((long long)max_q * a.G + COLS - 1) / COLS;
  MB_REQUIRE(blocks * a.kv_heads <= 65535, "paged attention over 4-bit pages: too many query columns for one launch");
  // As many CTAs as fit the GPU at once, four per SM, with a chunk or more per warp if the table were full.
  const long long pairs = (long long)batch * a.kv_heads * blocks;
  const long long chunks = ((long long)a.max_pages * a.page_size + P4_CHUNK - 1) / P4_CHUNK;
  const long long fit = 4LL * sm_count() / pairs, use = (chunks + P4_WARPS - 1) / P4_WARPS;
  const int splits = (int)std::max(1LL, std::min({16LL, fit, use}));
  a.splits = splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(batch, (unsigned)(blocks * a.kv_heads), splits);
  cfg.blockDim = dim3(P4_THREADS);
  cfg.dynamicSmemBytes = P4Cfg<D, COLS>::BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = splits;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_attn_int4_kernel<D, COLS>, a));
  count_launch();
}

void p4_attention(P4Args& a, int head_dim, int batch, int max_q, cudaStream_t stream) {
  const bool wide = max_q * a.G > 8;
  if (head_dim == 128) {
    if (wide) p4_launch<128, 16>(a, batch, max_q, stream);
    else p4_launch<128, 8>(a, batch, max_q, stream);
  } else {
    if (wide) p4_launch<64, 16>(a, batch, max_q, stream);
    else p4_launch<64, 8>(a, batch, max_q, stream);
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

void paged_attn_decode_int4(const KvInt4Cache& c, const void* q, long long q_stride, const int* context_lens, void* out, int batch,
                            int heads, float scale, int* status, cudaStream_t stream) {
  kv4_check(c, "paged_attn_decode_int4");
  MB_REQUIRE(heads > 0 && heads % c.kv_heads == 0, "paged_attn_decode_int4: heads must be a multiple of kv_heads");
  MB_REQUIRE(q_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0,
             "paged_attn_decode_int4: q must be 16-byte aligned with a token stride of a multiple of 8 elements");
  MB_REQUIRE(scale > 0.f, "paged_attn_decode_int4: scale must be positive");
  if (batch == 0) return;
  P4Args a{(const __nv_bfloat16*)q, (const uint8_t*)c.k, (const uint8_t*)c.v, c.block_table, context_lens, nullptr,
           (__nv_bfloat16*)out, q_stride, (long long)heads * c.head_dim, heads / c.kv_heads, c.kv_heads, batch, c.page_size,
           c.max_pages, c.n_pages, 1, scale * 1.4426950408889634f, status};
  p4_attention(a, c.head_dim, batch, 1, stream);
}

namespace {
bool p4_few(int max_q, int group) { return (long long)max_q * group <= P4_FEW_COLUMNS; }
}  // namespace

long long paged_attn_prefill_int4_workspace(int batch, int total_q, int max_q, int max_kv, int heads, int kv_heads, int head_dim) {
  return p4_few(max_q, heads / kv_heads) ? 0 : prompt_int4_workspace(batch, total_q, max_kv, heads, kv_heads, head_dim);
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
  if (p4_few(max_q, heads / c.kv_heads)) {
    P4Args a{(const __nv_bfloat16*)q, (const uint8_t*)c.k, (const uint8_t*)c.v, c.block_table, kv_lens, cu_q, (__nv_bfloat16*)out,
             q_stride, o_stride, heads / c.kv_heads, c.kv_heads, total_q, c.page_size, c.max_pages, c.n_pages, 1,
             scale * 1.4426950408889634f, status};
    p4_attention(a, c.head_dim, batch, max_q, stream);
    return;
  }
  MB_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "paged_attn_prefill_int4: workspace missing or not aligned");
  prompt_int4(c, q, q_stride, cu_q, kv_lens, out, o_stride, batch, total_q, max_q, max_kv, heads, scale, workspace, status, stream);
}

}  // namespace mb
