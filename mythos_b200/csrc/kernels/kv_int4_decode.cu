// Attention over the 4-bit paged KV cache for one or a few query tokens per sequence (format: kv_int4.cuh).
//
// Queries of one (sequence, kv head) are columns: column c is head c % G of token c / G. A warp takes chunks of 32 tokens
// (two tiles) for a block of COLS columns through a ring of its own. The ring is filled by 16-byte asynchronous copies, eight
// lanes to a tile: a bulk copy takes its addresses from uniform registers, and four lanes with a copy each cost 61 instructions
// a chunk, of 675, where these nine take twelve.
//
// Most of its instructions take codes apart, on the integer pipe (half rate), so operands are formed by one AND each:
// the low eleven bits of an fp16 are linear in its value (subnormals and the first normal binade share one step,
// 2^-24), so a nibble anywhere in them is its code times a power of two. Keys: bits 3-6 (code 2^-21) and 7-10 (code 2^-17)
// of a rotated word, then the word rotated by eight; queries of the second kind are multiplied by 2^-4. Values: bits 0-3
// (2^-24) and 4-7 (2^-20) of two tokens' halves side by side; they are different output values, scaled at the end.
//
// Scores: q . k = sum over groups of scale (q_g . c_g) + low sum(q_g), the product exact in fp16 (a query column is
// divided by a power of two first, so that its bf16 values fit). Values: o = sum_t (p_t scale_t) c_t + sum_t p_t low_t, the
// second sum a scalar per column and group in fp32. The tensor cores truncate what they add, and the codes are all
// positive: over a long context that would drift. So every second token (the upper halves of the operand) enters as
// -(p scale) (15 - c) + p (low + 15 scale): complementing costs one NOT per word, and the running sum stays near zero.
// p_t scale_t is rounded to fp16 (2^-11 of each term); the running reference M is the maximum of score plus exponent of the values
// over the tokens, so it fits whatever the values' size. Everything else is fp32. mma.sync rather than tcgen05:
// with 8 columns a 128-row tile would be filled to a sixteenth, and the codes would have to go through shared memory
// once more.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "api.h"
#include "common.cuh"
#include "host_util.h"
#include "kv_int4.cuh"
#include "tc.cuh"

namespace mb {
namespace {

constexpr int P4_WARPS = 4;
constexpr int P4_THREADS = 32 * P4_WARPS;
constexpr int P4_CHUNK = 32;      // tokens

template <int D, int COLS>
struct P4Cfg {
  using L = KvInt4<D>;
  // One chunk ahead: sixteen warps keep 74 KB (D = 128) in flight per SM, about twice what its share of the memory rate
  // times the latency asks for.
  static constexpr int STAGES = 2;
  static constexpr int HALF = 2 * L::TILE_BYTES;              // K (or V) of a chunk
  static constexpr int STAGE = 2 * HALF;
  static constexpr int WARP_BYTES = STAGES * STAGE;
  static constexpr int PART = COLS * D * 4;                   // a part's sums, [COLS][D]
  static_assert(PART <= WARP_BYTES, "a warp's last part is staged in its own (drained) ring");
};

__device__ __forceinline__ void p4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same into a fresh accumulator.
__device__ __forceinline__ void p4_mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void p4_copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t p4_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float p4_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t p4_transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

struct P4Args {
  const __nv_bfloat16* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  Kv4Pages pages;
  const int* kv_lens;
  const int* cu_q;          // first query row of every sequence, or null: one query token per sequence
  __nv_bfloat16* out;
  long long q_stride, o_stride;
  int batch, G, kv_heads, total_q;
  int max_q, max_kv;        // what the call announced of a sequence
  int most_chunks;          // a sequence's: the tables' tokens, and one chunk more, which reports what lies behind them
  Kv4Div by_group, by_heads;
  float scale_log2;
  int* status;
};

// Chunks of a sequence, whatever stands in its length: counts and sums of them stay within the launch's limits.
__device__ __forceinline__ int p4_chunks(int kv_len, int most) {
  return (int)min(((unsigned)max(kv_len, 0) + P4_CHUNK - 1u) / P4_CHUNK, (unsigned)most);
}
// A unit: one (sequence, kv head, block of columns).
struct P4Unit {
  int b, hkv, col0, n_cols, row0, q_len, kv_len;
  int to_some, to_all;      // tokens that some column sees, and that all see
  __device__ __forceinline__ int chunks(const P4Args& a) const { return p4_chunks(kv_len, a.most_chunks); }
  __device__ __forceinline__ P4Unit(const P4Args& a, int cols, int b_, int y) : b(b_) {
    const int block = a.by_heads(y);
    hkv = y - block * a.kv_heads;
    col0 = block * cols;
    row0 = a.cu_q ? a.cu_q[b] : b;
    q_len = a.cu_q ? a.cu_q[b + 1] - row0 : 1;
    kv_len = a.kv_lens[b];
    n_cols = min(cols, min(q_len, a.max_q) * a.G - col0);
    to_some = min(kv_len, kv_len - q_len + a.by_group(col0 + max(n_cols, 1) - 1) + 1);
    to_all = min(kv_len, kv_len - q_len + a.by_group(col0) + 1);
  }
  // Where the value d of column c goes, or null: a row that the output does not have.
  __device__ __forceinline__ __nv_bfloat16* out(const P4Args& a, int D, int c, int d) const {
    const int col = col0 + c, qi = a.by_group(col), row = row0 + qi;
    if (c >= n_cols || (unsigned)row >= (unsigned)a.total_q) return nullptr;
    return a.out + row * a.o_stride + (hkv * a.G + col - qi * a.G) * D + d;
  }
};

// A sequence with more new tokens or keys than the call announced is reported. Rows behind max_q have no unit and are left as they
// were; keys are all dealt with.
__device__ __forceinline__ void p4_announced(const P4Args& a, int q_len, int kv_len) {
  if (a.status && (q_len > a.max_q || kv_len > a.max_kv)) atomicCAS(a.status, 0, ST_BAD_ARG | (90 << 16));
}

// A warp's running state. Thread (r, t) of the warp holds columns 2 t and 2 t + 1 of every block of eight.
template <int D, int COLS>
struct P4State {
  static constexpr int NB = COLS / 8, GR = KvInt4<D>::GROUPS;
  uint32_t qb[NB][GR][8];                 // B operand: column r
  float qsum[NB][GR][2], factor[NB][2];   // of columns 2 t, 2 t + 1, as everything below
  int limit[NB][2];
  float o[NB][GR][4][4];                  // units of 2^-(24 + P4_DOWN) (even i) and 2^-(20 + P4_DOWN)
  float z[NB][GR][2], m[NB][2], l[NB][2];
  uint32_t unseen;                        // bit 2 nb + c: the column has seen no score yet (its reference is 0)
};

// Exponent that values of magnitude `mag` enter the reference with. p is kept up to 2^19 (and 2^6 more until the reference moves) times
// the inverse of the token's largest magnitude, which is at least 7 scales: p times a scale times 2^-P4_DOWN then stays below 2^12, and is
// exact to 2^-11 over 19 octaves below the reference. Every bf16 magnitude from 2^-81 on has its own: p is 2^-108 at least at the reference, so
// that 18 octaves of weights below it count, and 2^106 at most, so that a million of them stay within fp32, and so does a product with any
// value. Smaller magnitudes lose bits, below 2^-110 all. (With 2^8 and without P4_DOWN magnitudes ended at 2^112, and p times a scale
// overflowed above 2^117.)
constexpr int P4_DOWN = 11;
__device__ __forceinline__ float p4_exponent(float mag) {
  return fminf(fmaxf(__uint_as_float(0x4B000000u | (__float_as_uint(mag) >> 23)) - (8388608.f + 127.f), -81.f), 127.f) - 19.f;
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
    // (groups innermost: products of one sum wait for one another; 8 x 32768 tokens: 53.1 -> 51.9 us)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const uint32_t k0 = kw[0][g][h], k1 = kw[1][g][h];
          const uint32_t w0 = e ? __funnelshift_r(k0, k0, 8) : k0, w1 = e ? __funnelshift_r(k1, k1, 8) : k1;
          const uint32_t a0 = w0 & 0x00780078u, a1 = w1 & 0x00780078u, a2 = w0 & 0x07800780u, a3 = w1 & 0x07800780u;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float (&c)[4] = sc[u][nb][g];
            if (h == 0 && e == 0) p4_mma0(c, a0, a1, a2, a3, s.qb[nb][g][0], s.qb[nb][g][1]);
            else p4_mma(c, a0, a1, a2, a3, s.qb[nb][g][4 * h + 2 * e], s.qb[nb][g][4 * h + 2 * e + 1]);
          }
        }
  }
  // ---- largest exponent of the chunk's values, which decides whether the reference may have to move: one group of one token per thread and tile
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
  const float ev = p4_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mag))));
  // ---- online softmax: scores relative to the reference; it moves only when one of them passes it by 2^6
  float x[2][NB][2][2];                           // [tile][block][j][c]
  float top = -INFINITY;
  const int tok_r = tok0 + ((r >> 1) & 3) + ((r & 1) << 2);                // token of key row r of the first tile; row r + 8: 8 on
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
          v = fmaf(v, s.factor[nb][c], -s.m[nb][c]);
          if (MASK && (tok_r + 16 * u + 8 * j >= s.limit[nb][c] || (absent >> u & 1u))) v = -INFINITY;
          x[u][nb][j][c] = v;
        }
    }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) top = fmax3(top, x[u][nb][j][0], x[u][nb][j][1]);
  if (__any_sync(0xffffffffu, s.unseen != 0u || top + ev > 6.f)) {
    // where it moves to goes by every token's own score and exponent: with the chunk's exponent, one large token that a column
    // hardly weighs or does not see took the others' products below what fp16 holds (8 x 32768 tokens: 49.6 -> 50.7 us for it)
    float most[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) most[nb][0] = most[nb][1] = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t w[2];
        const uint32_t vp = smem_u32(at) + C::HALF + u * L::TILE_BYTES + L::OFF_PAIR + (8 * j + r) * L::PAIR;
        if constexpr (GR == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(vp));
        else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(vp));
        float m = 0.f;
#pragma unroll
        for (int g = 0; g < GR; ++g) m = fmax3(m, fabsf(fmaf(15.f, kv4_scale(w[g]), kv4_low(w[g]))), fabsf(kv4_low(w[g])));
        const float own = p4_exponent(m);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          most[nb][0] = fmaxf(most[nb][0], x[u][nb][j][0] + own);
          most[nb][1] = fmaxf(most[nb][1], x[u][nb][j][1] + own);
        }
      }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float mx = most[nb][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const bool first = s.unseen >> (2 * nb + c) & 1u;
        // (by the column's own scores alone: what the others hold, a NaN say, does not reach its bits)
        if (first ? mx > -INFINITY : mx > 6.f) {
          const float half = first ? 0.f : fast_exp2(-0.5f * mx), alpha = half * half;
          s.unseen &= ~(1u << (2 * nb + c));
          s.m[nb][c] += mx;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) x[u][nb][j][c] -= mx;
          s.l[nb][c] = s.l[nb][c] * half * half;  // (the sum may outlast what the products are: exponents of values are in them only)
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
  const float sign = ((r & 1) ? -1.f : 1.f) / (1 << P4_DOWN), whole = (r & 1) ? 15.f : 0.f;
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
        w[g] = kv4_scale(vq[g]) * sign;
        b[g] = fmaf(whole, kv4_scale(vq[g]), kv4_low(vq[g]));
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
      // halves of the two tokens' words side by side: lo holds values 0, 2, 4, 6 and hi values 1, 3, 5, 7 of both; the
      // second token's codes enter as 15 - code
      const uint32_t n0 = ~vw[0][1][g], n1 = ~vw[1][1][g];
      uint32_t lo0 = __byte_perm(vw[0][0][g], n0, 0x5410), hi0 = __byte_perm(vw[0][0][g], n0, 0x7632);
      uint32_t lo1 = __byte_perm(vw[1][0][g], n1, 0x5410), hi1 = __byte_perm(vw[1][0][g], n1, 0x7632);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i == 2) {
          lo0 >>= 8; hi0 >>= 8; lo1 >>= 8; hi1 >>= 8;
        }
        const uint32_t mask = (i & 1) ? 0x00F000F0u : 0x000F000Fu;
        const uint32_t a0 = lo0 & mask, a1 = hi0 & mask, a2 = lo1 & mask, a3 = hi1 & mask;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) p4_mma(s.o[nb][g][i], a0, a1, a2, a3, pb[u][nb][g][0], pb[u][nb][g][1]);
      }
    }
  }
}

// Queries of a unit into the state. The B operand: column r of every block; word h of group g holds values 64 g + 16 t + 8 h ..
template <int D, int COLS>
__device__ __forceinline__ void p4_queries(P4State<D, COLS>& s, const P4Args& a, const P4Unit& u, int lane) {
  constexpr int GR = KvInt4<D>::GROUPS, NB = COLS / 8;
  const int r = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int col = u.col0 + nb * 8 + r, qi = a.by_group(col);
    const bool live = nb * 8 + r < u.n_cols && (unsigned)(u.row0 + qi) < (unsigned)a.total_q;
    const int limit = live ? min(u.kv_len, u.kv_len - u.q_len + qi + 1) : 0;
    const __nv_bfloat16* qp = a.q + (u.row0 + qi) * a.q_stride + (u.hkv * a.G + col - qi * a.G) * D + 16 * t;
    uint32_t raw[GR][8];
    __nv_bfloat162 top = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
    for (int g = 0; g < GR; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (live) v = *reinterpret_cast<const uint4*>(qp + 64 * g + 8 * h);
        raw[g][4 * h] = v.x; raw[g][4 * h + 1] = v.y; raw[g][4 * h + 2] = v.z; raw[g][4 * h + 3] = v.w;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&raw[g][4 * h + e])));
      }
    top = __hmax2(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = __hmax2(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float big = fmaxf(__low2float(top), __high2float(top));
    // the column's largest value in 2^14 .. 2^15
    const int eq = big > 0.f ? max(-100, min(113, (int)(__float_as_uint(big) >> 23) - 127 - 14)) : 0;
    const float down = p4_pow2(-eq), down4 = p4_pow2(-eq - 4);
#pragma unroll
    for (int g = 0; g < GR; ++g) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = (e & 1) ? down4 : down;
        s.qb[nb][g][e] = p4_half2(kv4_scale(raw[g][e]) * f, kv4_low(raw[g][e]) * f);     // (both halves of a word)
      }
      // sum(q_g) in the scores' units of 2^-21: the product with a key whose codes are all one
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 8; e += 2) p4_mma(c, 0x00080008u, 0x00080008u, 0x00800080u, 0x00800080u, s.qb[nb][g][e], s.qb[nb][g][e + 1]);
      s.qsum[nb][g][0] = c[0];
      s.qsum[nb][g][1] = c[1];
      s.z[nb][g][0] = s.z[nb][g][1] = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) s.o[nb][g][q][0] = s.o[nb][g][q][1] = s.o[nb][g][q][2] = s.o[nb][g][q][3] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {                 // what concerns columns 2 t + c sits in the threads of r = 2 t + c
      const int from = 8 * t + 4 * c;
      s.limit[nb][c] = __shfl_sync(0xffffffffu, limit, from);
      s.factor[nb][c] = a.scale_log2 * 0x1p21f * p4_pow2(__shfl_sync(0xffffffffu, eq, from));
      s.m[nb][c] = 0.f;
      s.l[nb][c] = 0.f;
    }
  }
  s.unseen = (1u << (2 * NB)) - 1u;
}

// The state's sums, complete over the warp: into `out` (whole) or as a part to w_acc [COLS][D] with references and row sums
// in ml [2][COLS]. Thread (r, t) has columns 2 t and 2 t + 1 of every block, values 64 g + 8 r + (0 .. 7).
template <int D, int COLS>
__device__ __forceinline__ void p4_result(const P4State<D, COLS>& s, const P4Args& a, const P4Unit& u, bool whole, float* w_acc, float* ml,
                                          int lane) {
  constexpr int GR = KvInt4<D>::GROUPS, NB = COLS / 8;
  const int r = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int cc = nb * 8 + 2 * t + c;
      float l = s.l[nb][c];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;      // nothing visible: zeros
      if (!whole && r == 0) {
        ml[cc] = l == 0.f ? -INFINITY : s.m[nb][c];
        ml[COLS + cc] = l;
      }
      __nv_bfloat16* dst = whole ? u.out(a, D, cc, 8 * r) : nullptr;
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        float z = s.z[nb][g][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
        float v[8];                               // out of their units, with the offset sum
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float unit = ((q & 1) ? 0x1p20f : 0x1p24f) * (1 << P4_DOWN);
          v[2 * q] = fmaf(s.o[nb][g][q][c], unit, z) * inv;
          v[2 * q + 1] = fmaf(s.o[nb][g][q][2 + c], unit, z) * inv;
        }
        if (!whole) {
          float* p = w_acc + cc * D + 64 * g + 8 * r;
          *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else if (dst) {
          *reinterpret_cast<uint4*>(dst + 64 * g) =
              make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        }
      }
    }
}

// A warp's chunks 0 .. mine - 1 through its ring. locate(i) gives the tile of the lane's half (lane & 1) of chunk i: -1 without
// a page (reported, left out), -2 behind the keys. Lanes 8 n .. 8 n + 7 copy tile n % 2 of K (n < 2) or V.
template <int D, int COLS>
struct P4Feed {
  using L = KvInt4<D>;
  using C = P4Cfg<D, COLS>;
  static constexpr int PIECES = L::TILE_BYTES / 16;
  const uint8_t* ring;
  const uint8_t* from;            // the lane's first piece of tile 0
  uint32_t to;                    // of stage 0
  int* status;
  int lane, mine;
  int ids = -2, ids_next = -2;    // lane l: tile l % 2 of chunk 16 n + l / 2 for the block n being issued, and of the next one
  uint32_t none = 0u;             // bit l: that tile does not exist
  uint32_t gone = 0u, gone_next = 0u;  // bits 0, 1: tiles of the chunk in use, and of the next one, that were not loaded
  int off = 0;                    // of the stage in use (0 or STAGE)
  __device__ __forceinline__ P4Feed(const P4Args& a, uint8_t* ring_, int lane_, int mine_) : ring(ring_), status(a.status), lane(lane_), mine(mine_) {
    from = ((lane & 16) ? a.v_cache : a.k_cache) + (lane & 7) * 16;
    to = smem_u32(ring_) + ((lane & 16) ? C::HALF : 0) + ((lane & 8) ? L::TILE_BYTES : 0) + (lane & 7) * 16;
  }
  template <class F>
  __device__ __forceinline__ void issue(int i, int stage, const F& locate) {
    if (i < mine) {
      const int k = i & 15;
      if (k == 0) {
        ids = i == 0 ? locate(lane >> 1) : ids_next;
        none = __ballot_sync(0xffffffffu, ids < 0);
        if (ids == -1 && status) atomicCAS(status, 0, ST_BAD_ARG | (92 << 16));
      }
      if (k == 4 && i + 12 < mine) ids_next = locate(i + 12 + (lane >> 1));
      const int id = __shfl_sync(0xffffffffu, ids, 2 * k + (lane >> 3 & 1));
      gone_next = none >> (2 * k) & 3u;
      if (id >= 0) {
        const uint8_t* src = from + (long long)id * L::TILE_BYTES;
#pragma unroll
        for (int j = 0; j < PIECES / 8; ++j) p4_copy16(to + stage + 128 * j, src + 128 * j);
        if (PIECES % 8 && (lane & 7) < PIECES % 8) p4_copy16(to + stage + PIECES / 8 * 128, src + PIECES / 8 * 128);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Waits for chunk i, with the next one under way.
  template <class F>
  __device__ __forceinline__ void wait(int i, const F& locate) {
    gone = gone_next;
    issue(i + 1, off ^ C::STAGE, locate);         // (every lane is done with that stage: next())
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
  }
  __device__ __forceinline__ const uint8_t* at() const { return ring + off; }
  __device__ __forceinline__ void next() {
    __syncwarp();
    off ^= C::STAGE;
  }
};
static_assert(P4Cfg<128, 8>::STAGES == 2, "P4Feed alternates between two stages");

// Chunks i .. end - 1 of the warp, which are the unit's chunks chunk, chunk + step, ... Those that every column sees whole come
// first and have a loop of their own: with both forms in one loop the accumulators were copied between them.
template <int D, int COLS, class F>
__device__ __forceinline__ void p4_run(P4State<D, COLS>& s, P4Feed<D, COLS>& feed, const P4Unit& u, int& i, int end, int chunk, int step,
                                       const F& locate) {
  bool waited = false;
  for (; i < end && (chunk + 1) * P4_CHUNK <= u.to_all; ++i, chunk += step) {
    feed.wait(i, locate);
    if (feed.gone != 0u) {
      waited = true;
      break;
    }
    p4_chunk<D, COLS, false>(s, feed.at(), chunk * P4_CHUNK, feed.lane, u.to_some, 0u);
    feed.next();
  }
#pragma unroll 1
  for (; i < end; ++i, chunk += step) {
    if (!waited) feed.wait(i, locate);
    waited = false;
    p4_chunk<D, COLS, true>(s, feed.at(), chunk * P4_CHUNK, feed.lane, u.to_some, feed.gone);
    feed.next();
  }
}

// Joins the parts of a unit that shared memory holds (bits of `parts`), column c, values d .. d + 3: sums, and the column's
// reference and row sum. References may lie further apart than 2^126 where values do: row sums are scaled in two steps, here and below.
template <int D, int COLS, class At>
__device__ __forceinline__ float4 p4_join(uint32_t parts, const float* ml, const At& at, int c, int d, float& M, float& l) {
  M = -INFINITY;
  for (uint32_t w = parts; w; w &= w - 1) M = fmaxf(M, ml[(__ffs(w) - 1) * 2 * COLS + c]);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  l = 0.f;
  for (uint32_t w = parts; w; w &= w - 1) {
    const int k = __ffs(w) - 1;
    const float lk = ml[(2 * k + 1) * COLS + c];
    if (lk == 0.f) continue;                      // nothing seen (a NaN is not nothing)
    const float half = fast_exp2(0.5f * (ml[2 * k * COLS + c] - M)), e = half * half;
    const float4 v = *reinterpret_cast<const float4*>(at(k) + c * D + d);
    l = fmaf(half, half * lk, l);
    acc.x = fmaf(e, v.x, acc.x);
    acc.y = fmaf(e, v.y, acc.y);
    acc.z = fmaf(e, v.z, acc.z);
    acc.w = fmaf(e, v.w, acc.w);
  }
  return acc;
}
__device__ __forceinline__ void p4_store(__nv_bfloat16* dst, const float4& v, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (dst) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
}

// ------------------------------------------------------------------------------------------------ short contexts
// One unit per cluster, whose CTAs split its chunks and join their sums through distributed shared memory: one launch, which
// counts where the whole call takes a few microseconds.
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
__device__ __forceinline__ float4 p4_ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int D, int COLS>
struct P4SmemCluster {
  using C = P4Cfg<D, COLS>;
  static constexpr int OFF_CTA = P4_WARPS * C::WARP_BYTES;                  // the CTA's sums
  static constexpr int OFF_ML = OFF_CTA + C::PART;                          // [warps][m, l][COLS]
  static constexpr int OFF_CML = OFF_ML + P4_WARPS * 2 * COLS * 4;          // of the CTA: [m, l][COLS]
  static constexpr int BYTES = OFF_CML + 2 * COLS * 4;
};

template <int D, int COLS>
__global__ void __launch_bounds__(P4_THREADS, COLS == 8 ? 4 : 2)
paged_attn_int4_cluster_kernel(const __grid_constant__ P4Args a) {
  using C = P4Cfg<D, COLS>;
  using S = P4SmemCluster<D, COLS>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, splits = gridDim.z;
  const P4Unit u(a, COLS, blockIdx.x, blockIdx.y);
  if (blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) p4_announced(a, u.q_len, u.kv_len);
  if (u.n_cols <= 0) return;                      // the same for every CTA of the cluster
  float* s_ml = reinterpret_cast<float*>(smem + S::OFF_ML);
  float* s_cml = reinterpret_cast<float*>(smem + S::OFF_CML);
  float* s_cta = reinterpret_cast<float*>(smem + S::OFF_CTA);
  const int n = u.chunks(a), per = (n + splits - 1) / splits;
  const int chunk0 = blockIdx.z * per + warp, end = min(n, (int)blockIdx.z * per + per);
  const int mine = max(0, (end - chunk0 + P4_WARPS - 1) / P4_WARPS);        // chunk0, + 4, ...
  const auto locate = [&](int i) {
    const int token = (chunk0 + P4_WARPS * i) * P4_CHUNK + (lane & 1) * 16;
    return i < mine && token < u.kv_len ? a.pages.tile(u.b, token, u.hkv) : -2;
  };
  P4Feed<D, COLS> feed(a, smem + warp * C::WARP_BYTES, lane, mine);
  feed.issue(0, 0, locate);
  P4State<D, COLS> s;
  p4_queries(s, a, u, lane);
  int i = 0;
  p4_run(s, feed, u, i, mine, chunk0, P4_WARPS, locate);
  p4_result(s, a, u, false, reinterpret_cast<float*>(smem + warp * C::WARP_BYTES), s_ml + warp * 2 * COLS, lane);
  __syncthreads();
  for (int k = threadIdx.x; k < COLS * D / 4; k += P4_THREADS) {
    const int c = 4 * k / D, d = 4 * k % D;
    float M, l;
    const float4 v = p4_join<D, COLS>((1u << P4_WARPS) - 1u, s_ml, [&](int w) { return reinterpret_cast<const float*>(smem + w * C::WARP_BYTES); }, c, d, M, l);
    *reinterpret_cast<float4*>(s_cta + 4 * k) = v;
    if (d == 0) {
      s_cml[c] = M;
      s_cml[COLS + c] = l;
    }
  }
  p4_cluster_sync();
  // every CTA writes a share of the block's outputs, four values a thread
  const int share = (COLS * D / 4 + splits - 1) / splits, rank = p4_rank();
  for (int k = rank * share + threadIdx.x; k < min(COLS * D / 4, (rank + 1) * share); k += P4_THREADS) {
    const int c = 4 * k / D, d = 4 * k % D;
    if (c >= u.n_cols) break;
    const uint32_t m_at = smem_u32(s_cml + c), l_at = smem_u32(s_cml + COLS + c), v_at = smem_u32(s_cta + 4 * k);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f, M = -INFINITY;
#pragma unroll 4
    for (int p = 0; p < splits; ++p) {
      const float m = p4_ld_cluster(p4_mapa(m_at, p)), lp = p4_ld_cluster(p4_mapa(l_at, p));
      const float4 v = p4_ld_cluster4(p4_mapa(v_at, p));
      if (lp == 0.f) continue;
      const float Mn = fmaxf(M, m), h0 = M == -INFINITY ? 0.f : fast_exp2(0.5f * (M - Mn)), h1 = fast_exp2(0.5f * (m - Mn));
      const float e0 = h0 * h0, e1 = h1 * h1;
      acc.x = fmaf(e1, v.x, acc.x * e0);
      acc.y = fmaf(e1, v.y, acc.y * e0);
      acc.z = fmaf(e1, v.z, acc.z * e0);
      acc.w = fmaf(e1, v.w, acc.w * e0);
      l = fmaf(h1, h1 * lp, h0 * (h0 * l));
      M = Mn;
    }
    p4_store(u.out(a, D, c, d), acc, l);
  }
  p4_cluster_sync();                              // nobody leaves while a peer still reads its shared memory
}

// ------------------------------------------------------------------------------------------------ long contexts
// A unit has n = ceil(keys / 32) chunks. All chunks of all units stand in one line, units of a sequence side by side, and every
// warp takes an equal stretch of it, so that ragged batches and any number of units load the GPU evenly (with equal splits
// of each unit, 148 SMs x 16 warps were filled to three quarters: 8 x 32768 tokens and 5 kv heads took 73 us, 60 this way). A
// warp that meets a whole unit writes its outputs; parts of units go to shared memory and are joined by the CTA, and what
// crosses a CTA's border goes to a scratch buffer of the call (two slots a CTA) and is joined by p4_merge_kernel.
struct P4Line {
  int batch, G, kv_heads, cols, max_q, most_chunks;
  const int* kv_lens;
  const int* cu_q;
  __device__ __forceinline__ P4Line(const P4Args& a, int cols_)
      : batch(a.batch), G(a.G), kv_heads(a.kv_heads), cols(cols_), max_q(a.max_q), most_chunks(a.most_chunks), kv_lens(a.kv_lens), cu_q(a.cu_q) {}
  __device__ __forceinline__ int chunks(int b) const { return p4_chunks(kv_lens[b], most_chunks); }
  __device__ __forceinline__ int units(int b) const {
    const int q = cu_q ? max(min(cu_q[b + 1] - cu_q[b], max_q), 0) : 1;
    return kv_heads * ((q * G + cols - 1) / cols);
  }
  __device__ __forceinline__ int size(int b) const { return b < batch ? chunks(b) * units(b) : 0; }
};
// Equal stretches: the first `rem` of them one chunk longer. No more stretches than leave each two chunks: every part costs the
// merge more than a chunk costs a warp.
struct P4Share {
  int workers, per, rem;
  __device__ __forceinline__ P4Share(int total, int most)
      : workers(max(1, min(most, total / 2))), per(total / workers), rem(total - per * workers) {}
  __device__ __forceinline__ int start(int worker) const {
    const int w = min(worker, workers);            // (the warps that are left have none)
    return w * per + min(w, rem);
  }
  __device__ __forceinline__ int worker(int place) const {       // whose stretch holds it
    const int longer = rem * (per + 1);
    return place < longer ? place / (per + 1) : rem + (place - longer) / max(per, 1);
  }
};
// What a warp knows of the line: the size of sequence `lane` (of the first 32) and the sum of those up to it.
struct P4Scan {
  int size, sum, total;
  __device__ __forceinline__ P4Scan(const P4Line& line, int lane) {
    size = line.size(lane);
    sum = size;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    total = __shfl_sync(0xffffffffu, sum, 31);
    for (int b0 = 32; b0 < line.batch; b0 += 32) total += __reduce_add_sync(0xffffffffu, (unsigned)line.size(b0 + lane));
  }
  // The sequence that holds a place below the total, and where it begins.
  __device__ __forceinline__ int find(const P4Line& line, int place, int lane, int& begin) const {
    int base = 0, n = size, up = sum;
    for (int b0 = 0;; b0 += 32) {
      const unsigned past = __ballot_sync(0xffffffffu, base + up > place);
      if (past || b0 + 32 >= line.batch) {
        const int l = past ? __ffs(past) - 1 : 31;
        begin = base + __shfl_sync(0xffffffffu, up - n, l);
        return b0 + l;
      }
      base += __shfl_sync(0xffffffffu, up, 31);
      n = line.size(b0 + 32 + lane);
      up = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
      }
    }
  }
  // Where sequence b begins.
  __device__ __forceinline__ int begin(const P4Line& line, int b, int lane) const {
    if (b < 32) return __shfl_sync(0xffffffffu, sum - size, b);
    int s = __shfl_sync(0xffffffffu, sum, 31);
    for (int b0 = 32; b0 < b; b0 += 32) s += __reduce_add_sync(0xffffffffu, (unsigned)(b0 + lane < b ? line.size(b0 + lane) : 0));
    return s;
  }
};

template <int D, int COLS>
struct P4SmemLine {
  using C = P4Cfg<D, COLS>;
  static constexpr int OFF_HEAD = P4_WARPS * C::WARP_BYTES;                 // head parts; tail parts lie in the drained rings
  static constexpr int OFF_ML = OFF_HEAD + P4_WARPS * C::PART;              // [warps][head, tail][m, l][COLS]
  static constexpr int OFF_UNIT = OFF_ML + P4_WARPS * 4 * COLS * 4;         // [warps][head, tail] int4: sequence, unit, begins, ends
  static constexpr int OFF_LEAD = OFF_UNIT + P4_WARPS * 2 * 16;             // int2: sequence and unit of the CTA's first chunk
  static constexpr int BYTES = OFF_LEAD + 16;
};

template <int D, int COLS>
__global__ void __launch_bounds__(P4_THREADS, COLS == 8 ? 4 : 2)
paged_attn_int4_line_kernel(const __grid_constant__ P4Args a, float* __restrict__ scratch) {
  using C = P4Cfg<D, COLS>;
  using S = P4SmemLine<D, COLS>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* s_ml = reinterpret_cast<float*>(smem + S::OFF_ML);
  int4* s_unit = reinterpret_cast<int4*>(smem + S::OFF_UNIT);
  int2* s_lead = reinterpret_cast<int2*>(smem + S::OFF_LEAD);
  // the merge may start as soon as there is room; it waits for this grid's end before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (lane < 2) s_unit[warp * 2 + lane] = make_int4(-1, 0, 0, 0);
  __syncwarp();                                   // (the warp's own, until the CTA meets)

  const P4Line line(a, COLS);
  const P4Scan scan(line, lane);
  const P4Share share(scan.total, gridDim.x * P4_WARPS);
  const int worker = blockIdx.x * P4_WARPS + warp;
  const int f0 = share.start(worker), mine = share.start(worker + 1) - f0;
  int begin = 0, b = 0, n = 1, left_units = 0, y = 0, chunk = 0;
  if (mine > 0) {
    b = scan.find(line, f0, lane, begin);
    n = line.chunks(b);
    y = (f0 - begin) / n;
    chunk = f0 - begin - y * n;
    left_units = line.units(b) - y;
    if (warp == 0 && lane == 0) *s_lead = make_int2(b, y);       // (where the first warp has nothing, no warp has)
  }
  // Every lane walks the line from where it was.
  int lb = b, ln = n, lbegin = begin, lsize = mine > 0 ? line.size(b) : 0;
  const auto locate = [&](int i) {
    if (i >= mine) return -2;
    const int f = f0 + i;
    while (f >= lbegin + lsize) {
      lbegin += lsize;
      lsize = line.size(++lb);
      ln = line.chunks(lb);
    }
    const int at = f - lbegin, ly = at / ln, token = (at - ly * ln) * P4_CHUNK + (lane & 1) * 16;
    return token < a.kv_lens[lb] ? a.pages.tile(lb, token, ly - a.by_heads(ly) * a.kv_heads) : -2;
  };
  P4Feed<D, COLS> feed(a, smem + warp * C::WARP_BYTES, lane, mine);
  feed.issue(0, 0, locate);
  P4State<D, COLS> s;
  int i = 0;
  while (i < mine) {
    // ---- one unit, or the part of it in this warp's stretch
    const P4Unit u(a, COLS, b, y);
    const bool begins = chunk == 0;
    p4_queries(s, a, u, lane);
    const int part = min(n - chunk, mine - i);
    p4_run(s, feed, u, i, i + part, chunk, 1, locate);
    chunk += part;
    const bool ends = chunk == n;
    const int slot = ends ? 0 : 1;                // (a part that does not end its unit is the warp's last)
    p4_result(s, a, u, begins && ends, reinterpret_cast<float*>(smem + (slot ? warp * C::WARP_BYTES : S::OFF_HEAD + warp * C::PART)),
              s_ml + (warp * 2 + slot) * 2 * COLS, lane);
    if (!(begins && ends) && lane == 0) s_unit[warp * 2 + slot] = make_int4(b, y, begins ? 1 : 0, ends ? 1 : 0);
    if (ends) {
      chunk = 0;
      ++y;
      if (--left_units == 0 && i < mine) {
        do {
          ++b;
          n = line.chunks(b);
          left_units = line.units(b);
        } while (n == 0 || left_units == 0);      // (the line has mine chunks: some later sequence holds the next)
        y = 0;
      }
    }
  }
  __syncthreads();

  // ---- parts of one unit follow each other in the order (warp, head / tail): joined by the CTA
  const auto at = [&](int k) {
    return reinterpret_cast<const float*>((k & 1) ? smem + (k >> 1) * C::WARP_BYTES : smem + S::OFF_HEAD + (k >> 1) * C::PART);
  };
  for (int p = 0; p < 2 * P4_WARPS;) {
    const int4 g = s_unit[p];
    if (g.x < 0) {
      ++p;
      continue;
    }
    uint32_t parts = 1u << p;
    int e = p + 1, last_end = g.w;
    for (; e < 2 * P4_WARPS; ++e) {
      const int4 v = s_unit[e];
      if (v.x < 0) continue;
      if (v.x != g.x || v.y != g.y) break;
      parts |= 1u << e;
      last_end = v.w;
    }
    p = e;
    const bool whole = g.z && last_end;
    const P4Unit u(a, COLS, g.x, g.y);
    // the unit that holds the CTA's first chunk goes to the first slot
    float* dst = scratch + (blockIdx.x * 2 + (s_lead->x == g.x && s_lead->y == g.y ? 0 : 1)) * COLS * (D + 2);
    for (int k = threadIdx.x; k < u.n_cols * D / 4; k += P4_THREADS) {
      const int c = 4 * k / D, d = 4 * k % D;
      float M, l;
      const float4 v = p4_join<D, COLS>(parts, s_ml, at, c, d, M, l);
      if (whole) {
        p4_store(u.out(a, D, c, d), v, l);
      } else {
        *reinterpret_cast<float4*>(dst + 4 * k) = v;
        if (d == 0) {
          dst[COLS * D + c] = M;
          dst[COLS * D + COLS + c] = l;
        }
      }
    }
  }
}

// One CTA per unit and 32 of its values: joins the parts of a unit that lies in several CTAs' stretches; zeros for a sequence
// without keys. First the weights of the parts (one thread per part and column), then the sums: slices of the CTA share
// the parts, with their loads in flight (one slice takes 0.3 us a part: one sequence of 16384 tokens, one kv head, in a wide table: 44.6
// us with a part for every chunk, 11.7 with four slices and two chunks a stretch; 8 x 32768 of 5 heads: 54.7 -> 49.9).
constexpr int P4_MERGE = 64;      // parts whose weights are held at a time
template <int D, int COLS, int SLICES>
__global__ void __launch_bounds__(COLS * 8 * SLICES)
p4_merge_kernel(const __grid_constant__ P4Args a, const float* __restrict__ scratch, int ctas) {
  constexpr int PART = COLS * (D + 2), THREADS = COLS * 8 * SLICES;
  __shared__ float s_w[P4_MERGE][COLS], s_lw[P4_MERGE][COLS], s_l[SLICES][COLS];
  __shared__ float4 s_acc[SLICES][COLS * 8];
  __shared__ int s_at[P4_MERGE];
  const int b = blockIdx.x, y = blockIdx.y, lane = threadIdx.x & 31;
  const P4Line line(a, COLS);
  const P4Scan scan(line, lane);
  const P4Share share(scan.total, ctas * P4_WARPS);
  const int u0 = scan.begin(line, b, lane) + y * line.chunks(b), n = line.chunks(b);
  const bool here = y < line.units(b);
  int c0 = 0, c1 = -1;
  if (n > 0 && here) {
    c0 = share.worker(u0) / P4_WARPS;
    c1 = share.worker(u0 + n - 1) / P4_WARPS;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");             // every CTA, so that this grid ends behind the one before
  if (y == 0 && blockIdx.z == 0 && threadIdx.x == 0 && a.cu_q) p4_announced(a, a.cu_q[b + 1] - a.cu_q[b], a.kv_lens[b]);
  if (!here || (n > 0 && c0 == c1)) return;       // no such unit, or written by that CTA
  const P4Unit u(a, COLS, b, y);
  const int slice = threadIdx.x / (COLS * 8), at_col = threadIdx.x % (COLS * 8), c = at_col >> 3, part_of = threadIdx.x & 7;
  const int d = blockIdx.z * 32 + part_of * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f, M = -INFINITY;
  for (int k0 = c0; k0 <= c1; k0 += P4_MERGE) {   // (a unit of more than 64 CTAs: joined in turns)
    const int parts = min(P4_MERGE, c1 - k0 + 1);
    __syncthreads();
    for (int i = threadIdx.x; i < parts * COLS; i += THREADS) {
      const int p = i / COLS, cc = i % COLS, k = k0 + p;
      // the first CTA has the unit in its first slot only where the unit holds the first chunk of its stretch; a CTA's stretch is
      // never empty between others
      const int at = (2 * k + (u0 > share.start(k * P4_WARPS) ? 1 : 0)) * PART;
      if (cc == 0) s_at[p] = at;
      s_w[p][cc] = scratch[at + COLS * D + cc];
      s_lw[p][cc] = scratch[at + COLS * D + COLS + cc];
    }
    __syncthreads();
    float Mn = M;                                 // the eight threads of a column look through every eighth part
    for (int p = part_of; p < parts; p += 8)
      if (s_lw[p][c] != 0.f) Mn = fmaxf(Mn, s_w[p][c]);          // nothing seen is left out, a NaN is not
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, o));
    const float half = M == -INFINITY ? 0.f : fast_exp2(0.5f * (M - Mn)), e = half * half;
    acc.x *= e; acc.y *= e; acc.z *= e; acc.w *= e;
    l = l * half * half;
    M = Mn;
    if (c < u.n_cols) {
#pragma unroll 8
      for (int p = slice; p < parts; p += SLICES) {
        const float lw = s_lw[p][c];
        const float4 v = lw != 0.f ? *reinterpret_cast<const float4*>(scratch + s_at[p] + c * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float half = lw != 0.f ? fast_exp2(0.5f * (s_w[p][c] - M)) : 0.f, w = half * half;
        l = fmaf(half, half * lw, l);
        acc.x = fmaf(w, v.x, acc.x);
        acc.y = fmaf(w, v.y, acc.y);
        acc.z = fmaf(w, v.z, acc.z);
        acc.w = fmaf(w, v.w, acc.w);
      }
    }
  }
  if constexpr (SLICES > 1) {
    s_acc[slice][at_col] = acc;
    if (part_of == 0) s_l[slice][c] = l;
    __syncthreads();
    if (slice > 0) return;
#pragma unroll
    for (int k = 1; k < SLICES; ++k) {
      const float4 v = s_acc[k][at_col];
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      l += s_l[k][c];
    }
  }
  p4_store(u.out(a, D, c, d), acc, l);
}

// A kernel's limits, raised once per device.
template <typename K>
void p4_configure(K kern, int smem, bool cluster, std::atomic<unsigned long long>& seen) {
  int dev = 0;
  MB_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 64 && (seen >> dev & 1ull)) return;
  MB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (cluster) MB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (dev < 64) seen |= 1ull << dev;
}

// Clusters of `splits` CTAs that run side by side. A cluster lies within one of the GPU's partitions, which are not of one size: 40
// clusters of 14 CTAs are fewer CTAs than fit, but take two turns (8 x 2048 tokens, 5 kv heads: 18.5 us, 10.7 in smaller ones).
template <int D, int COLS>
int p4_capacity(int splits) {
  static std::atomic<int> known[64][17];          // per device
  static std::atomic<unsigned long long> seen{0};
  int n = 0, dev = 0;
  MB_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 64 && (n = known[dev][splits]) > 0) return n;
  p4_configure(paged_attn_int4_cluster_kernel<D, COLS>, P4SmemCluster<D, COLS>::BYTES, true, seen);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(1, 1, splits);
  cfg.blockDim = dim3(P4_THREADS);
  cfg.dynamicSmemBytes = P4SmemCluster<D, COLS>::BYTES;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = splits;
  MB_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, paged_attn_int4_cluster_kernel<D, COLS>, &cfg));
  n = std::max(1, n);
  if (dev < 64) known[dev][splits] = n;
  return n;
}
int p4_capacity(int D, int cols, int splits) {
  if (D == 128) return cols == 16 ? p4_capacity<128, 16>(splits) : p4_capacity<128, 8>(splits);
  return cols == 16 ? p4_capacity<64, 16>(splits) : p4_capacity<64, 8>(splits);
}

// How a call runs, by its sizes (the table's width stands for the contexts, which only the device knows).
struct P4Plan {
  int cols, ctas, splits;         // splits > 0: clusters; else stretches of the line over that many CTAs
  long long blocks, units, chunks, resident;      // resident: CTAs side by side
};
P4Plan p4_plan(int batch, int max_q, int G, int kv_heads, int D, long long max_tokens) {
  P4Plan p;
  max_q = std::max(1, max_q);       // (a call that announces no new tokens still looks at the lengths)
  p.cols = (long long)max_q * G > 8 ? 16 : 8;
  p.blocks = ((long long)max_q * G + p.cols - 1) / p.cols;
  p.units = (long long)batch * kv_heads * p.blocks;
  p.chunks = std::max(1LL, (max_tokens + P4_CHUNK - 1) / P4_CHUNK);
  p.resident = (p.cols == 8 ? 4LL : 2LL) * sm_count();
  p.ctas = (int)std::max(1LL, std::min(p.resident, (p.units * p.chunks + P4_WARPS - 1) / P4_WARPS));
  // A cluster per unit, of as many CTAs as the units leave room for, while no warp gets more than sixteen chunks (eight, where a
  // larger cluster would have been of use). One launch, no scratch and no walk along the line: 64 x 1024 tokens (8 kv heads, one
  // query) take 22.1 us (27.4 as a line), 64 x 2048 37.2 (41.1), 64 ragged x 1280 24.2 (27.3), 1 x 1024 6.8 (9.3), 8 x 8192 23.9
  // (26.8). Longer contexts want the line's evenness: 1 x 32768 take 23.1 there (24.2 before as clusters), 2 x 32768 27.5 (31.3), and what
  // lies between is even: 1 x 16384 16.1 (15.5).
  const long long want = std::min(16LL, (p.chunks + P4_WARPS - 1) / P4_WARPS);
  long long room = std::max(1LL, std::min(want, p.resident / std::max(1LL, p.units)));
  while (room > 1 && p4_capacity(D, p.cols, (int)room) < p.units) --room;
  p.splits = p.chunks <= (room == 16 ? 8 : 16) * P4_WARPS * room ? (int)room : 0;
  return p;
}

template <int D, int COLS>
void p4_launch(P4Args& a, const P4Plan& plan, float* scratch, cudaStream_t stream) {
  MB_REQUIRE(plan.blocks * a.kv_heads <= 65535, "paged attention over 4-bit pages: too many query columns for one launch");
  MB_REQUIRE(plan.units * (plan.chunks + 1) < (1LL << 31), "paged attention over 4-bit pages: too many chunks for one launch");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (plan.splits > 0) {
    static std::atomic<unsigned long long> seen{0};
    p4_configure(paged_attn_int4_cluster_kernel<D, COLS>, P4SmemCluster<D, COLS>::BYTES, true, seen);
    cfg.gridDim = dim3(a.batch, (unsigned)(plan.blocks * a.kv_heads), plan.splits);
    cfg.blockDim = dim3(P4_THREADS);
    cfg.dynamicSmemBytes = P4SmemCluster<D, COLS>::BYTES;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = plan.splits;
    MB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_attn_int4_cluster_kernel<D, COLS>, a));
    count_launch();
    return;
  }
  static std::atomic<unsigned long long> seen{0};
  p4_configure(paged_attn_int4_line_kernel<D, COLS>, P4SmemLine<D, COLS>::BYTES, false, seen);
  paged_attn_int4_line_kernel<D, COLS><<<plan.ctas, P4_THREADS, P4SmemLine<D, COLS>::BYTES, stream>>>(a, scratch);
  count_launch();
  check_launch();
  cfg.gridDim = dim3(a.batch, (unsigned)(plan.blocks * a.kv_heads), D / 32);
  const auto merge = [&](auto kern, int slices) {
    cfg.blockDim = dim3(COLS * 8 * slices);
    MB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a, (const float*)scratch, plan.ctas));
  };
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  // (units of a few parts each want no slices: 64 x 1024 tokens, 8 kv heads, in a wide table: 27.6 us with one, 34.6 with four)
  if (plan.ctas >= 8 * plan.units) merge(p4_merge_kernel<D, COLS, 4>, 4);
  else merge(p4_merge_kernel<D, COLS, 1>, 1);
  count_launch();
}

}  // namespace

bool few_query_int4_takes(int batch, int max_q, int max_kv, int heads, int kv_heads, int head_dim) {
  const P4Plan p = p4_plan(batch, max_q, heads / kv_heads, kv_heads, head_dim, max_kv);
  return max_q == 0 || p.blocks * p.cols <= 64 || (p.units <= p.resident && p.units * p.chunks <= 8 * P4_WARPS * p.resident);
}

long long few_query_int4_workspace(const KvInt4Cache& c, int batch, int max_q, int heads) {
  const P4Plan p = p4_plan(batch, max_q, heads / c.kv_heads, c.kv_heads, c.head_dim, (long long)c.max_pages * c.page_size);
  return p.splits > 0 ? 0 : 2LL * p.ctas * p.cols * (c.head_dim + 2) * 4;
}

void few_query_int4(const KvInt4Cache& c, const void* q, long long q_stride, const int* cu_q, const int* kv_lens, void* out,
                    long long o_stride, int batch, int total_q, int max_q, int max_kv, int heads, float scale, void* workspace,
                    int* status, cudaStream_t stream) {
  const int G = heads / c.kv_heads;
  const P4Plan plan = p4_plan(batch, max_q, G, c.kv_heads, c.head_dim, (long long)c.max_pages * c.page_size);
  P4Args a{(const __nv_bfloat16*)q, (const uint8_t*)c.k, (const uint8_t*)c.v,
           {c.block_table, c.n_seqs, c.max_pages, c.n_pages, c.kv_heads, c.page_size, kv4_div(c.page_size)}, kv_lens, cu_q,
           (__nv_bfloat16*)out, q_stride, o_stride, batch, G, c.kv_heads, total_q, max_q, max_kv, (int)(plan.chunks + 1), kv4_div(G), kv4_div(c.kv_heads),
           scale * 1.4426950408889634f, status};
  float* scratch = (float*)workspace;
  if (c.head_dim == 128) {
    if (plan.cols == 16) p4_launch<128, 16>(a, plan, scratch, stream);
    else p4_launch<128, 8>(a, plan, scratch, stream);
  } else {
    if (plan.cols == 16) p4_launch<64, 16>(a, plan, scratch, stream);
    else p4_launch<64, 8>(a, plan, scratch, stream);
  }
}

}  // namespace mb
