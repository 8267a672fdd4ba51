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

// ------------------------------------------------------------------------------------------------ attention
// One (sequence, kv head, block of COLS query columns) per cluster; the CTAs of the cluster split its tiles. A column
// is one (query token, head of the group) pair: column c is head c % G of token c / G. Four warps per CTA; warp w
// takes every fourth tile of its CTA's range through a ring of its own, filled with one bulk copy per tile
// for K and one for V.
//
// Scores: q . k = sum over groups of scale (q_g . c_g) + low sum(q_g). The matrix product runs on 16 + code, exact in
// bf16, one AND-OR per pair of values; the offset leaves with (low - 16 scale) sum(q_g) in fp32. Values:
// o = sum_t (p_t scale_t) (c_t - 8) + sum_t p_t (low_t + 8 scale_t): the codes are centred here, because this sum runs
// over the whole context and the tensor cores truncate what they add; the second sum is a scalar per column and group.
// p_t scale_t is rounded to bf16 (half a step, 2^-9 of each term; the rounding errors of the terms are independent),
// everything else is fp32. mma.sync rather than tcgen05: at 8 columns the tile would be 128 rows for 8 useful ones,
// and the codes would have to be expanded through shared memory.
//
// The CTAs of a cluster merge their partial softmax states through distributed shared memory: no scratch, no
// counters, one result for the same inputs, and calls on several streams share nothing.
constexpr int P4_WARPS = 4;
constexpr int P4_THREADS = 32 * P4_WARPS;

template <int D, int COLS>
struct P4Cfg {
  using L = KvInt4<D>;
  static constexpr int STAGES = D == 128 ? 6 : 8;
  static constexpr int STAGE = 2 * L::TILE_BYTES;             // K tile, V tile
  static constexpr int WARP_BYTES = STAGES * STAGE;
  static constexpr int OFF_BAR = P4_WARPS * WARP_BYTES;
  static constexpr int OFF_ML = OFF_BAR + P4_WARPS * STAGES * 8 + 16;              // m, l: [warps][COLS] each
  static constexpr int OFF_Z = OFF_ML + 2 * P4_WARPS * COLS * 4;                    // [warps][COLS][groups]
  static constexpr int OFF_CTA = OFF_Z + P4_WARPS * COLS * L::GROUPS * 4;           // m, l of the CTA, weight, 1 / l
  static constexpr int BYTES = OFF_CTA + 2 * COLS * 4 + 128;
  static_assert(COLS * D * 4 <= WARP_BYTES, "a warp's output state is staged in its own (drained) ring");
};

__device__ __forceinline__ void p4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void p4_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
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
// The pair of values 2 i, 2 i + 1 of a rotated key word as the bf16 numbers 16 + code.
template <int I>
__device__ __forceinline__ uint32_t p4_key_pair(uint32_t w) {
  const uint32_t s = I == 0 ? w : (I == 3 ? __funnelshift_r(w, w, 12) : w >> (4 * I));
  return (s & 0x00780078u) | 0x41804180u;
}
// Nibble i of both halves as the bf16 numbers code - 8: 128 + code by bit pattern, minus 136 (exact).
template <int I>
__device__ __forceinline__ uint32_t p4_value_pair(uint32_t w) {
  const uint32_t x = ((w >> (4 * I)) & 0x000F000Fu) | 0x43004300u;
  const __nv_bfloat162 y = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)));
  return *reinterpret_cast<const uint32_t*>(&y);
}

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

template <int D, int COLS>
__global__ void __launch_bounds__(P4_THREADS)
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

  // tiles of this CTA: what the last query of the block sees, cut into equal ranges
  const int last_q = (col0 + n_cols - 1) / a.G;
  const int visible = min(kv_len, kv_len - q_len + last_q + 1);
  const int n_tiles = (max(0, visible) + 15) >> 4;
  const int per = (n_tiles + a.splits - 1) / a.splits;
  const int tile0 = split * per, tile1 = min(n_tiles, tile0 + per);
  const int my_tiles = (tile1 - tile0 - warp + P4_WARPS - 1) / P4_WARPS;      // tile0 + warp, + 4, ... (<= 0: none)
  const int* table = a.block_table + (long long)b * a.max_pages;

  // lane l holds the tile index of the warp's tile 32 n + l for the block n being issued, and of the next block
  auto locate = [&](int i) {
    return i < my_tiles ? kv4_tile(table, (tile0 + warp + P4_WARPS * i) * 16, a.max_pages, a.n_pages, a.page_size, a.kv_heads, hkv) : -1;
  };
  int ids = locate(lane), ids_next = locate(32 + lane);
  uint32_t present = 0u;                          // bit s: stage s holds a tile
  auto issue = [&](int i) {                       // all lanes; lane 0 starts the copies of the warp's tile i
    if (i > 0 && (i & 31) == 0) {
      ids = ids_next;
      ids_next = locate(i + 32 + lane);
    }
    const int id = __shfl_sync(0xffffffffu, ids, i & 31), st = i % C::STAGES;
    if (id >= 0) {
      present |= 1u << st;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[st], C::STAGE);
        p4_bulk_load(ring + st * C::STAGE, a.k_cache + (long long)id * L::TILE_BYTES, L::TILE_BYTES, &full[st]);
        p4_bulk_load(ring + st * C::STAGE + L::TILE_BYTES, a.v_cache + (long long)id * L::TILE_BYTES, L::TILE_BYTES, &full[st]);
      }
    } else {                                      // a token of the context without a page: reported, left out
      present &= ~(1u << st);
      if (lane == 0) {
        if (a.status) atomicCAS(a.status, 0, ST_BAD_ARG | (92 << 16));
        mbar_arrive(&full[st]);
      }
    }
  };
  for (int i = 0; i < C::STAGES - 1 && i < my_tiles; ++i) issue(i);

  // Queries: the A operand, columns r and r + 8; k-step j of group g holds values 64 g + 16 t + 4 j .. + 3.
  uint32_t qa[NB][GR][8];
  float qsum[NB][GR];
  int limit[NB];                                  // tokens the column sees
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int col = col0 + nb * 8 + r;
    const int qi = col / a.G, g_head = col % a.G;
    const bool live = nb * 8 + r < n_cols && (unsigned)(row0 + qi) < (unsigned)a.total_q;
    limit[nb] = live ? min(kv_len, kv_len - q_len + qi + 1) : 0;
    const __nv_bfloat16* qp = a.q + (long long)(row0 + qi) * a.q_stride + (long long)(hkv * a.G + g_head) * D + 16 * t;
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (live) x = *reinterpret_cast<const uint4*>(qp + 64 * g + 8 * h);
        qa[nb][g][4 * h] = x.x; qa[nb][g][4 * h + 1] = x.y; qa[nb][g][4 * h + 2] = x.z; qa[nb][g][4 * h + 3] = x.w;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += kv4_scale(qa[nb][g][4 * h + e]) + kv4_low(qa[nb][g][4 * h + e]);   // both halves
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      qsum[nb][g] = sum + __shfl_xor_sync(0xffffffffu, sum, 2);
    }
  }
  float o[NB][GR][4][4];
  float z[NB][GR], m_ref[NB], l_run[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m_ref[nb] = -INFINITY;
    l_run[nb] = 0.f;
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      z[nb][g] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nb][g][i][0] = o[nb][g][i][1] = o[nb][g][i][2] = o[nb][g][i][3] = 0.f;
    }
  }

  bool ok = true;
  int done = 0;
  for (int i = 0; i < my_tiles; ++i) {
    // the stage read in the step before is free now: every value read from it has gone through a product
    if (i + C::STAGES - 1 < my_tiles) issue(i + C::STAGES - 1);
    const int st = i % C::STAGES;
    ok = mbar_wait(&full[st], (i / C::STAGES) & 1, abort_flag, a.status, 93);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    done = i + 1;
    if (!(present >> st & 1u)) continue;
    const uint8_t* kt = ring + st * C::STAGE;
    const uint8_t* vt = kt + L::TILE_BYTES;

    // ---- scores of tokens t + 4 (2 j + e): sc[j][g][2 nb' + e] over the matrix product's rows r and r + 8
    float sc[2][GR][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t kw[GR][2];
      const uint8_t* kp = kt + (8 * j + r) * L::ROW + t * (8 * GR);
      if constexpr (GR == 2) {
        const uint4 x = *reinterpret_cast<const uint4*>(kp);
        kw[0][0] = x.x; kw[0][1] = x.y; kw[1][0] = x.z; kw[1][1] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(kp);
        kw[0][0] = x.x; kw[0][1] = x.y;
      }
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        sc[j][g][0] = sc[j][g][1] = sc[j][g][2] = sc[j][g][3] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = kw[g][h];
          const uint32_t p0 = p4_key_pair<0>(w), p1 = p4_key_pair<1>(w), p2 = p4_key_pair<2>(w), p3 = p4_key_pair<3>(w);
          p4_mma(sc[j][g], qa[0][g][4 * h], NB > 1 ? qa[NB - 1][g][4 * h] : 0u, qa[0][g][4 * h + 1], NB > 1 ? qa[NB - 1][g][4 * h + 1] : 0u, p0, p1);
          p4_mma(sc[j][g], qa[0][g][4 * h + 2], NB > 1 ? qa[NB - 1][g][4 * h + 2] : 0u, qa[0][g][4 * h + 3], NB > 1 ? qa[NB - 1][g][4 * h + 3] : 0u, p2, p3);
        }
      }
    }
    // ---- scales and lows of this thread's four tokens
    const int tok0 = (tile0 + warp + P4_WARPS * i) * 16 + t;
    float ks[2][2][GR], kl[2][2][GR], vs[2][2][GR], vl[2][2][GR];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t kq[2][GR], vq[2][GR];
      const uint8_t* kp = kt + L::OFF_PAIR + (8 * j + 2 * t) * L::PAIR;
      const uint8_t* vp = vt + L::OFF_PAIR + (8 * j + 2 * t) * L::PAIR;
      if constexpr (GR == 2) {
        const uint4 x = *reinterpret_cast<const uint4*>(kp), y = *reinterpret_cast<const uint4*>(vp);
        kq[0][0] = x.x; kq[0][1] = x.y; kq[1][0] = x.z; kq[1][1] = x.w;
        vq[0][0] = y.x; vq[0][1] = y.y; vq[1][0] = y.z; vq[1][1] = y.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(kp), y = *reinterpret_cast<const uint2*>(vp);
        kq[0][0] = x.x; kq[1][0] = x.y;
        vq[0][0] = y.x; vq[1][0] = y.y;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          ks[j][e][g] = kv4_scale(kq[e][g]);
          kl[j][e][g] = fmaf(-16.f, ks[j][e][g], kv4_low(kq[e][g]));
          vs[j][e][g] = kv4_scale(vq[e][g]);
          vl[j][e][g] = fmaf(8.f, vs[j][e][g], kv4_low(vq[e][g]));
        }
    }
    // ---- online softmax per column; the reference maximum moves only when it grew by more than 2^8
    uint32_t pb[NB][GR][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float x[2][2], mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = 0.f;
#pragma unroll
          for (int g = 0; g < GR; ++g) v += fmaf(ks[j][e][g], sc[j][g][2 * nb + e], kl[j][e][g] * qsum[nb][g]);
          x[j][e] = tok0 + 4 * (2 * j + e) < limit[nb] ? v * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, x[j][e]);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const bool need = mx > m_ref[nb] + 8.f || (m_ref[nb] == -INFINITY && mx > -INFINITY);
      if (__any_sync(0xffffffffu, need)) {
        const float alpha = need ? fast_exp2(m_ref[nb] - mx) : 1.f;
        if (need) m_ref[nb] = mx;
        l_run[nb] *= alpha;
        const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          z[nb][g] *= alpha;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            o[nb][g][q][0] *= a0; o[nb][g][q][1] *= a1; o[nb][g][q][2] *= a0; o[nb][g][q][3] *= a1;
          }
        }
      }
      const float m_use = m_ref[nb] == -INFINITY ? 0.f : m_ref[nb];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float p0 = fast_exp2(x[j][0] - m_use), p1 = fast_exp2(x[j][1] - m_use);
        l_run[nb] += p0 + p1;
        // a token the column does not see may hold anything, behind the sequence's end too: it is left out, not
        // multiplied by zero
        const bool s0 = tok0 + 8 * j < limit[nb], s1 = tok0 + 8 * j + 4 < limit[nb];
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          z[nb][g] += (s0 ? p0 * vl[j][0][g] : 0.f) + (s1 ? p1 * vl[j][1][g] : 0.f);
          pb[nb][g][j] = pack_bf16x2(s0 ? p0 * vs[j][0][g] : 0.f, s1 ? p1 * vs[j][1][g] : 0.f);
        }
      }
    }
    // ---- values: the A operand holds values x tokens, B the probabilities
    uint32_t vw[2][2][GR];
    const int chunk = r ^ ((t >> 1) << 2);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint8_t* vp = vt + (t + 4 * (2 * j + e)) * L::ROW + chunk * (4 * GR);
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
      const uint32_t lo0 = __byte_perm(vw[0][0][g], vw[0][1][g], 0x5410), hi0 = __byte_perm(vw[0][0][g], vw[0][1][g], 0x7632);
      const uint32_t lo1 = __byte_perm(vw[1][0][g], vw[1][1][g], 0x5410), hi1 = __byte_perm(vw[1][0][g], vw[1][1][g], 0x7632);
#define P4_PV(I)                                                                                              \
  do {                                                                                                        \
    const uint32_t a0 = p4_value_pair<I>(lo0), a1 = p4_value_pair<I>(hi0), a2 = p4_value_pair<I>(lo1),        \
                   a3 = p4_value_pair<I>(hi1);                                                                \
    _Pragma("unroll") for (int nb = 0; nb < NB; ++nb) p4_mma(o[nb][g][I], a0, a1, a2, a3, pb[nb][g][0], pb[nb][g][1]); \
  } while (0)
      P4_PV(0);
      P4_PV(1);
      P4_PV(2);
      P4_PV(3);
#undef P4_PV
    }
    __syncwarp();
  }
  if (!ok)                                        // copies in flight land before the ring's memory goes away
    for (int i = done; i < my_tiles && i < done + C::STAGES; ++i) mbar_drain(&full[i % C::STAGES], (i / C::STAGES) & 1);

  // ---- the warp's state: row c of w_acc is column c, values in order
  float* w_acc = reinterpret_cast<float*>(ring);
  __syncwarp();
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float l = l_run[nb];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
      s_m[warp * COLS + nb * 8 + r] = ok ? m_ref[nb] : -INFINITY;
      s_l[warp * COLS + nb * 8 + r] = ok ? l : 0.f;
    }
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      float zz = z[nb][g];
      zz += __shfl_xor_sync(0xffffffffu, zz, 1);
      zz += __shfl_xor_sync(0xffffffffu, zz, 2);
      if (t == 0) s_z[(warp * COLS + nb * 8 + r) * GR + g] = zz;
      // thread (r, t): columns 2 t and 2 t + 1, values 64 g + 8 r + (0 .. 7)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* dst = w_acc + (nb * 8 + 2 * t + c) * D + 64 * g + 8 * r;
        *reinterpret_cast<float4*>(dst) = make_float4(o[nb][g][0][c], o[nb][g][0][2 + c], o[nb][g][1][c], o[nb][g][1][2 + c]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(o[nb][g][2][c], o[nb][g][2][2 + c], o[nb][g][3][c], o[nb][g][3][2 + c]);
      }
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
  // Enough CTAs for two to four per SM, each with two tiles or more per warp if the table were full.
  const long long pairs = (long long)batch * a.kv_heads * blocks;
  const long long tiles = (long long)a.max_pages * (a.page_size >> 4);
  int splits = 1;
  while (splits < 16 && pairs * splits < 2LL * sm_count() && tiles > 8LL * splits) splits *= 2;
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
