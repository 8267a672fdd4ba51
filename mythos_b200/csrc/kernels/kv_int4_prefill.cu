// Attention of prompts over the 4-bit paged KV cache: tcgen05 products on fp16 images of the pages.
//
// kv4_expand_kernel turns every sequence's pages into 128-token tiles [batch, kv_heads, tokens, D] of
// fp16 in a workspace, once for all the queries that read them, and the queries into fp16 rows; fa_int4_kernel is the
// persistent two-tile flash attention kernel of attention_fwd2.cu over those images (128 x 128 score tiles, P in tensor memory).
//
// Why fp16 and not bf16: a value scale * code + low has up to 20 significant bits. Rounded to bf16 (half a step, 2^-8)
// every key moves its score by up to 2^-8 of sum |q k|, which is several times the error of all other roundings together
// (measured 4.5e-3 of the output in bf16 against 1.7e-3 here, of which 1.65e-3 is the output's own rounding). fp16
// has three bits more but a range of 2^-14 .. 2^15, so exponents are factored out, all powers of two (exact):
//   * a query row is divided by 2^eq (its largest value then lies in 2^14 .. 2^15); the thread that owns the row's softmax
//     multiplies it back with the softmax scale;
//   * a tile of keys (128 tokens of one head) is divided by 2^ek, which joins the same factor per step;
//   * a tile of values is divided by 2^ev, and the probabilities of the step are multiplied by it: the running reference
//     M is the maximum of score + ev, so that p 2^(ev - M) stays within fp16, and the row sum is taken back by 2^-ev. What it
//     is taken back to is sum 2^(score - M), between 2^-113 and 2^116 a key for ev of -110 to 113: it is kept in units of 2^10 (units of the
//     first tile's ev overflowed where later values were 2^130 times as large). Values below 2^-124 lose bits.
// Tokens of a tile whose magnitudes lie more than 2^8 apart get exponents of their own (PF_SPREAD), so that a large token takes no
// bits from the others for the queries that give it no weight or do not see it: the softmax then adds every key's own to its score
// first. Such tiles, and tiles whose values lie 2^100 below the largest, take a step of their own (four times as long: 2048 tokens over 6144 with
// one such token in every tile 850 us, not 226).
// The matrix product multiplies masked probabilities of zero by whatever the value rows hold, so nothing that is not
// finite goes there: tokens behind a sequence's end are zeros, and a token with a scale that is not finite gets values of
// zero and NaN keys, which reach the queries that see it through their scores, and no others.
//
// The work is a line of (item, key tile) steps, an item being 256 query rows of one kv head, cut into equal stretches, one per
// CTA: with whole items per CTA the 256 items of 2048 new tokens left every fourth SM idle for half of the time. What a border
// cuts is written as an unnormalised part and joined by a third kernel.
//
// Rows of a query tile are (token, head) pairs of one kv head when the group divides 128 (a box of GP heads x 128 / GP tokens
// in one TMA load), so that short prompts fill their tiles and the heads of a group read a K / V tile once; other groups run one
// head at a time.
#include <cuda_fp16.h>

#include <algorithm>

#include "api.h"
#include "host_util.h"
#include "kv_int4.cuh"
#include "tc.cuh"

namespace mb {
namespace {

constexpr int PF_TILE = 128;      // tokens of a K / V tile, rows of a query tile
constexpr int PF_EXPAND = 256;    // threads of the expansion
constexpr int PF_Q_ROWS = 4;      // query rows a thread takes part in, loads first (one, with a 64-bit division: 4 prompts of 2048 tokens, 32 heads, took 198 us, not 187)

// Exponent e so that a value of magnitude m lies in 2^14 .. 2^15 after division by 2^e. Bounded so that 2^-e is a number.
__device__ __forceinline__ int pf_exponent(float m) {
  if (!(m > 0.f)) return 0;
  const int e = (int)(__float_as_uint(m) >> 23) - 127 - 14;      // subnormals: -141 -> bounded
  return max(-126, min(113, e));
}
constexpr int PF_EV_MIN = -110;   // of a tile of values
constexpr int PF_SPREAD = 8;      // octaves between the tokens of a tile that share an exponent: p keeps 2^-17 of the largest term
// Octaves between the values' exponents of a part's tiles up to which row sums are taken from p, which goes with them: 26 are left for the scores
// before fp32 ends. What lies below counts for nothing in the products, but would in the sum where it is the values that are small.
constexpr int PF_ALIKE = 100;
constexpr float PF_SUM_UNIT = 0x1p10f;      // of a row sum
__device__ __forceinline__ float pf_pow2(int e) { return __uint_as_float((uint32_t)(max(-126, min(127, e)) + 127) << 23); }
// Of values: zeros must not raise the reference (with an exponent of 0 they took thirteen bits and more from the other tiles' p).
__device__ __forceinline__ int pf_value_exponent(float m) { return m > 0.f ? max(PF_EV_MIN, pf_exponent(m)) : PF_EV_MIN; }
__device__ __forceinline__ uint32_t pf_half2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// tcgen05.mma on fp16 with the descriptors' low words (address / 16) in registers and their high words constant: formed anew for
// every product, they took the issuing thread longer than the product takes.
constexpr uint32_t PF_DESC_HI = 1024 / 16 | 1u << 14 | 2u << 29;      // atoms 1024 bytes apart, version, 128-byte swizzle
template <uint32_t IDESC, uint32_t A_HI, uint32_t B_HI>
__device__ __forceinline__ void pf_mma(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 a, b;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "mov.b64 a, {%1, %2};\n"
      "mov.b64 b, {%3, %4};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n"
      "}\n" ::"r"(d), "r"(a_lo), "n"(A_HI), "r"(b_lo), "n"(B_HI), "r"(IDESC), "r"(accumulate)
      : "memory");
}
template <uint32_t IDESC, uint32_t B_HI>
__device__ __forceinline__ void pf_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 b;\n"
      "setp.ne.b32 p, %5, 0;\n"
      "mov.b64 b, {%2, %3};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n"
      "}\n" ::"r"(d), "r"(a), "r"(b_lo), "n"(B_HI), "r"(IDESC), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pf_store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// Eight values times inv (a power of two) as fp16. 0x4300 | code is the bf16 number 128 + code; the 128 scale leaves with the low
// (both exact to 2^-17 of a step, far below fp16's rounding).
__device__ __forceinline__ uint4 pf_expand8(uint32_t w, uint32_t pair, float inv) {
  const float s = kv4_scale(pair) * inv, low = fmaf(-128.f, s, kv4_low(pair) * inv);
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = (w >> (4 * i) & 0x000F000Fu) | 0x43004300u;
    y[i] = pf_half2(fmaf(kv4_scale(x), s, low), fmaf(kv4_low(x), s, low));           // (both halves of a word)
  }
  return make_uint4(y[0], y[1], y[2], y[3]);
}

// ------------------------------------------------------------------------------------------------ the line of steps
// A pair is (sequence, block of 256 query rows); its items, one per unit (`pack` heads of a kv head), stand side by side, each
// with as many steps as its last row sees key tiles (at least one, so that rows that see nothing get their zeros), behind
// PF_SETUP places that stand for what an item costs beside its steps (8500 cycles of 3350 a step: equal numbers of steps alone
// gave the stretches of short items 40 of them, and 4 prompts of 2048 tokens took 296 us instead of 195).
constexpr int PF_SETUP = 2;
struct PfLine {
  const int* cu_q;
  const int* kv_lens;
  int batch, pack, log_pack, units, n_qb, tiles;
  int per_item;                     // query tiles of an item: two, one where that fills the GPU
  Kv4Div by_blocks, by_share;       // query blocks of a sequence; units of a kv head
};
struct PfItem {
  int b, row0, q_len, q_off, kv_len, tok[2], J[2], steps;   // tok: first token of each tile; J: its key tiles
  bool live[2];
  __device__ __forceinline__ int places() const { return steps > 0 ? steps + PF_SETUP : 0; }
  __device__ __forceinline__ PfItem(const PfLine& a, int pair) {
    b = a.by_blocks(pair);
    const int blk = pair - b * a.n_qb, per = PF_TILE >> a.log_pack;     // tokens of a tile
    row0 = a.cu_q[b];
    q_len = a.cu_q[b + 1] - row0;
    kv_len = a.kv_lens[b];
    q_off = kv_len - q_len;
    steps = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      tok[t] = (a.per_item * blk + t) * per;
      live[t] = t < a.per_item && tok[t] < q_len;
      const int hi = live[t] ? min(kv_len, q_off + min(q_len, tok[t] + per)) : 0;
      J[t] = min(a.tiles, (max(hi, 0) + PF_TILE - 1) / PF_TILE);
      if (live[t]) steps = max(steps, max(1, J[t]));
    }
  }
};
// Written by the expansion, read by the attention and the merge: [0] places of a stretch, [1] how many stretches have one more,
// [2] stretches; then (pair, unit, place in the item, places) of every stretch's start.
struct PfPlan {
  int* p;
  __device__ __forceinline__ int per() const { return p[0]; }
  __device__ __forceinline__ int rem() const { return p[1]; }
  __device__ __forceinline__ int count() const { return p[2]; }
  __device__ __forceinline__ int* start(int c) const { return p + 4 + 4 * c; }
};
__device__ __forceinline__ int pf_start(int per, int rem, int c) { return c * per + min(c, rem); }
__device__ __forceinline__ int pf_owner(int per, int rem, int place) {       // whose stretch holds it
  const int longer = rem * (per + 1);
  return place < longer ? place / (per + 1) : rem + (place - longer) / max(per, 1);
}

struct PfExpand {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  Kv4Pages pages;
  const int* kv_lens;
  const __nv_bfloat16* q;
  long long q_stride;
  __half* k;            // [batch * kv_heads, tokens, D]
  __half* v;
  __half* qh;           // [total_q, heads, D]
  float* q_factor;      // [total_q, heads]: 2^eq
  int* exponents;       // [batch * kv_heads, tiles]: from the low byte on ek, a bit per 16 tokens that have no page, ev, 1 where tokens have their own
  int16_t* own;         // [batch * kv_heads, tiles, 128]: there, ek and ev of every token
  int kv_heads, heads, tiles, kv_blocks, q_blocks, q_rows;     // q_rows: total_q * heads
  Kv4Div by_heads;
  int pairs;
  int max_q, max_kv;    // what the call announced of a sequence
  PfLine line;
  PfPlan plan;
  int ctas;
  int* status;
};

constexpr int PF_MIN_STEPS = 6;   // places of a stretch: a step is about 2 us, setting up and writing a part five
static_assert(PF_MIN_STEPS > PF_SETUP, "a stretch holds a step");
// Where there are no more items than CTAs and none has more steps than this, every CTA takes a whole one, and there is no merge:
// 3 prompts of 500 over up to 500 tokens (8 steps) take 31 us so and 35 with equal stretches, one of 700 over 700 (11) 33 and 31.
constexpr int PF_WHOLE_STEPS = 8;
// The same for items of a single query tile, whose steps are shorter (2400 cycles to 3350): 6 ragged prompts of up to 700 tokens
// (6 steps) take 20.7 us so and 22.9 with two tiles, 700 over 700 (11) 29.3 and 31.0, 1500 (12) 30.4 and 29.4.
constexpr int PF_SINGLE_STEPS = 11;

// One block: the plan. Every thread takes a run of pairs.
__device__ void pf_make_plan(const PfExpand& a) {
  __shared__ int s_sum[PF_EXPAND / 32], s_total;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (a.pairs + PF_EXPAND - 1) / PF_EXPAND, p0 = min(a.pairs, (int)threadIdx.x * each), p1 = min(a.pairs, p0 + each);
  for (int b = threadIdx.x; b < a.line.batch; b += PF_EXPAND)     // more tokens than the caller said: not all may be dealt with
    if (a.status && (a.line.kv_lens[b] > a.max_kv || a.line.cu_q[b + 1] - a.line.cu_q[b] > a.max_q))
      atomicCAS(a.status, 0, ST_BAD_ARG | (90 << 16));
  int sum = 0;
  for (int p = p0; p < p1; ++p) sum += PfItem(a.line, p).places() * a.line.units;
  int up = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += v;
  }
  if (lane == 31) s_sum[warp] = up;
  __syncthreads();
  if (threadIdx.x == 0) {
    int t = 0;
    for (int w = 0; w < PF_EXPAND / 32; ++w) {
      const int v = s_sum[w];
      s_sum[w] = t;
      t += v;
    }
    s_total = t;
  }
  __syncthreads();
  const int total = s_total;
  const int count = max(1, min(a.ctas, total / PF_MIN_STEPS)), per = total / count, rem = total - per * count;
  int place = s_sum[warp] + up - sum;
  for (int p = p0; p < p1; ++p) {
    const int places = PfItem(a.line, p).places(), end = place + places * a.line.units;
    for (int c = place > 0 ? pf_owner(per, rem, place - 1) + 1 : 0; c < count && pf_start(per, rem, c) < end; ++c) {
      const int at = pf_start(per, rem, c) - place;
      int* s = a.plan.start(c);
      s[0] = p;
      s[1] = at / places;
      s[2] = at - at / places * places;
      s[3] = per + (c < rem ? 1 : 0);
    }
    place = end;
  }
  if (threadIdx.x == 0) {
    a.plan.p[0] = per;
    a.plan.p[1] = rem;
    a.plan.p[2] = total > 0 ? count : 0;
  }
}

// Blocks [0, kv_blocks): one 128-token tile of one (sequence, kv head). Then query rows, one per D / 8 lanes; then the plan.
template <int D>
__global__ void __launch_bounds__(PF_EXPAND)
kv4_expand_kernel(const __grid_constant__ PfExpand a) {
  using L = KvInt4<D>;
  constexpr int WORDS = D / 8;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the attention waits for this grid's end before it reads
  if ((int)blockIdx.x == a.kv_blocks + a.q_blocks) {
    pf_make_plan(a);
    return;
  }
  if ((int)blockIdx.x >= a.kv_blocks) {
    constexpr int ROWS = PF_EXPAND / WORDS;        // PF_Q_ROWS of them in turn, loads first
    const int row0 = ((int)blockIdx.x - a.kv_blocks) * (ROWS * PF_Q_ROWS) + threadIdx.x / WORDS, c = threadIdx.x % WORDS;
    bf16x8 x[PF_Q_ROWS];
#pragma unroll
    for (int k = 0; k < PF_Q_ROWS; ++k) {
      const int row = min(row0 + k * ROWS, a.q_rows - 1), token = a.by_heads(row);
      x[k] = ldg8(a.q, token * a.q_stride + (row - token * a.heads) * D + c * 8);
    }
#pragma unroll
    for (int k = 0; k < PF_Q_ROWS; ++k) {
      const long long row = row0 + k * ROWS;
      float f[8];
      unpack8(x[k], f);
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(f[e]));
#pragma unroll
      for (int o = WORDS / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (row >= a.q_rows) continue;               // (the lanes of a row go together; every lane has shuffled)
      const int e = pf_exponent(m);
      const float inv = pf_pow2(-e);
      *reinterpret_cast<uint4*>(a.qh + row * D + c * 8) =
          make_uint4(pf_half2(f[0] * inv, f[1] * inv), pf_half2(f[2] * inv, f[3] * inv), pf_half2(f[4] * inv, f[5] * inv),
                     pf_half2(f[6] * inv, f[7] * inv));
      if (c == 0) a.q_factor[row] = pf_pow2(e);
    }
    return;
  }
  __shared__ uint32_t s_pair[2][PF_TILE][L::GROUPS];
  __shared__ int s_tile[8];
  __shared__ uint32_t s_ext[4][PF_EXPAND / 32];       // largest magnitudes of K and V, smallest
  __shared__ int8_t s_own[2][PF_TILE];
  const int j = blockIdx.x % a.tiles, bh = blockIdx.x / a.tiles, b = bh / a.kv_heads, head = bh % a.kv_heads;
  const int len = a.kv_lens[b], n0 = j * PF_TILE;
  if (n0 >= len) return;
  if (threadIdx.x < 8) {
    int tile = -1;
    if (n0 + 16 * (int)threadIdx.x < len) {
      tile = a.pages.tile(b, n0 + 16 * threadIdx.x, head);
      if (tile < 0 && a.status) atomicCAS(a.status, 0, ST_BAD_ARG | (91 << 16));
    }
    s_tile[threadIdx.x] = tile;
  }
  __syncthreads();
  // pairs of both tensors; the largest magnitude a group can stand for lies at one of its ends
  static_assert(PF_TILE * L::GROUPS <= PF_EXPAND && PF_TILE * L::GROUPS % 32 == 0, "a thread holds one group at most, and warps go together");
  float km = 0.f, vm = 0.f;            // of the thread's token
  bool held = false;                   // with values that are numbers
  if (const int i = threadIdx.x; i < PF_TILE * L::GROUPS) {
    const int n = i / L::GROUPS, g = i % L::GROUPS, tile = s_tile[n >> 4];
    uint32_t kp = 0u, vp = 0u;
    if (tile >= 0 && n0 + n < len) {
      const long long at = (long long)tile * L::TILE_BYTES;
      kp = *reinterpret_cast<const uint32_t*>(a.k_cache + at + kv4_pair<D>(n & 15, g));
      bool finite = true;
#pragma unroll
      for (int gg = 0; gg < L::GROUPS; ++gg) {
        const uint32_t p = *reinterpret_cast<const uint32_t*>(a.v_cache + at + kv4_pair<D>(n & 15, gg));
        finite = finite && kv4_finite(p);
        if (gg == g) vp = p;
      }
      held = finite;
      if (!finite) {
        kp = 0x7FFF7FFFu;
        vp = 0u;
      }
    }
    s_pair[0][n][g] = kp;
    s_pair[1][n][g] = vp;
    if (kv4_finite(kp)) km = fmaxf(fabsf(kv4_low(kp)), fabsf(fmaf(15.f, kv4_scale(kp), kv4_low(kp))));
    vm = fmaxf(fabsf(kv4_low(vp)), fabsf(fmaf(15.f, kv4_scale(vp), kv4_low(vp))));
    if constexpr (L::GROUPS == 2) {
      km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, 1));
      vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, 1));
    }
    if (g == 0) {
      s_own[0][n] = (int8_t)pf_exponent(km);
      s_own[1][n] = (int8_t)pf_value_exponent(vm);
    }
  }
  // (As integers: they are not negative. Values of zero count as the smallest there are: a token of them that takes nearly all the weight
  // must not push the others' p out of fp16. Keys of zero do no harm.)
  {
    const uint32_t kb = __float_as_uint(km), vb = __float_as_uint(vm);
    const uint32_t k1 = __reduce_max_sync(0xffffffffu, kb), v1 = __reduce_max_sync(0xffffffffu, vb);
    const uint32_t k0 = __reduce_min_sync(0xffffffffu, kb ? kb : ~0u), v0 = __reduce_min_sync(0xffffffffu, held ? vb : ~0u);
    if ((threadIdx.x & 31) == 0) {
      s_ext[0][threadIdx.x >> 5] = k1;
      s_ext[1][threadIdx.x >> 5] = v1;
      s_ext[2][threadIdx.x >> 5] = k0;
      s_ext[3][threadIdx.x >> 5] = v0;
    }
  }
  __syncthreads();
  uint32_t k1 = 0u, v1 = 0u, k0 = ~0u, v0 = ~0u;
#pragma unroll
  for (int w = 0; w < PF_EXPAND / 32; ++w) {
    k1 = max(k1, s_ext[0][w]);
    v1 = max(v1, s_ext[1][w]);
    k0 = min(k0, s_ext[2][w]);
    v0 = min(v0, s_ext[3][w]);
  }
  const int ek = pf_exponent(__uint_as_float(k1)), ev = pf_value_exponent(__uint_as_float(v1));
  const bool apart = (int)(k1 >> 23) - (int)(min(k0, k1) >> 23) > PF_SPREAD || (int)(v1 >> 23) - (int)(min(v0, v1) >> 23) > PF_SPREAD;
  if (threadIdx.x == 0) {
    int absent = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) absent |= (s_tile[u] < 0 && n0 + 16 * u < len ? 1 : 0) << u;
    a.exponents[blockIdx.x] = (ek & 0xFF) | absent << 8 | (ev & 0xFF) << 16 | (apart ? 1 : 0) << 24;
  }
  if (apart && threadIdx.x < PF_TILE)
    a.own[(long long)blockIdx.x * PF_TILE + threadIdx.x] = (int16_t)((s_own[0][threadIdx.x] & 0xFF) | s_own[1][threadIdx.x] * 256);
  const long long out = ((long long)bh * a.tiles + j) * PF_TILE * D;
#pragma unroll 4
  for (int i = threadIdx.x; i < PF_TILE * WORDS; i += PF_EXPAND) {
    const int n = i / WORDS, c = i % WORDS, g = c >> 3, u = c & 7, tile = s_tile[n >> 4];
    const uint32_t kp = s_pair[0][n][g], vp = s_pair[1][n][g];
    uint32_t kw = 0u, vw = 0u;
    if (tile >= 0 && n0 + n < len) {
      const long long at = (long long)tile * L::TILE_BYTES;
      kw = kv4_unrotate(*reinterpret_cast<const uint32_t*>(a.k_cache + at + kv4_key_word<D>(n & 15, g, u)));
      vw = *reinterpret_cast<const uint32_t*>(a.v_cache + at + kv4_value_word<D>(n & 15, g, u));
    }
    *reinterpret_cast<uint4*>(a.k + out + (long long)i * 8) = pf_expand8(kw, kp, pf_pow2(apart ? -s_own[0][n] : -ek));
    *reinterpret_cast<uint4*>(a.v + out + (long long)i * 8) = pf_expand8(vw, vp, pf_pow2(apart ? -s_own[1][n] : -ev));
  }
}

// ------------------------------------------------------------------------------------------------ attention
constexpr int PF_THREADS = 384;   // service warps, softmax of tile 0, softmax of tile 1

template <int D>
struct PfCfg {
  static constexpr int KS = D == 128 ? 2 : 4, VS = D == 128 ? 3 : 4;    // K and V stages
  static constexpr int CHUNKS = D / 64;
  static constexpr int TILE_BYTES = PF_TILE * D * 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = 2 * TILE_BYTES;
  static constexpr int OFF_V = OFF_K + KS * TILE_BYTES;
  static constexpr int OFF_BAR = OFF_V + VS * TILE_BYTES;
  static constexpr int NUM_BARS = 4 + 2 * KS + 2 * VS + 8;
  static constexpr int SMEM_BYTES = OFF_BAR + NUM_BARS * 8 + 16 + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory per CTA");
  static constexpr int COL_S = 0;     // S_t at t * 128 (P_t over its first 64 columns)
  static constexpr int COL_O = 256;   // O_t at 256 + t * D
};

struct PfArgs {
  PfLine line;
  PfPlan plan;
  const float* q_factor;
  const int* exponents;
  const int16_t* own;
  __nv_bfloat16* out;
  float* parts;         // [stretches][2 slots][2 tiles]: see pf_part_floats
  long long o_stride;
  int heads, group, total_q;
  float scale_log2;
  int* status;
  bool whole;           // a whole item per CTA
  Kv4Div by_units;
};
// A part of a query tile: sums [D / 4][128 rows][4], reference and row sum per row.
template <int D>
__host__ __device__ constexpr int pf_part_floats() { return PF_TILE * (D + 2); }

// The parts of a CTA's stretch, in order: the steps j0 .. j1 of an item.
struct PfCursor {
  int pair, unit, at, left, slot = -1;
  int j0, j1;           // of the part
  int of_pair, of_unit;
  __device__ __forceinline__ explicit PfCursor(const PfArgs& a) {
    const int c = blockIdx.x;
    left = 0;
    pair = unit = at = 0;
    if (a.whole) {                        // one item per stretch, which needs no plan
      pair = a.by_units(c);
      unit = c - pair * a.line.units;
      left = PfItem(a.line, pair).places();
    } else if (c < a.plan.count()) {
      const int* s = a.plan.start(c);
      left = s[3];
      pair = s[0];
      unit = s[1];
      at = s[2];
    }
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  // The item of the next part, and past it.
  __device__ __forceinline__ PfItem next(const PfArgs& a) {
    PfItem it(a.line, pair);
    while (it.steps == 0) it = PfItem(a.line, ++pair);     // (a later pair holds the steps that are left)
    slot = slot < 0 ? 0 : 1;
    of_pair = pair;
    of_unit = unit;
    const int end = min(it.places(), at + left);
    j0 = max(0, at - PF_SETUP);
    j1 = end - PF_SETUP;          // (more than j0: a stretch is longer than PF_SETUP)
    left -= end - at;
    at = 0;
    if (left <= PF_SETUP) left = 0;                        // no step of the next item
    if (j1 == it.steps) {
      if (++unit == a.line.units) {
        unit = 0;
        ++pair;
      }
    }
    return it;
  }
};

// Where every CTA has an item of its own the kernel is launched ahead of the expansion's end, and finds its item meanwhile (6 ragged
// prompts of up to 700 tokens: 20.7 us -> 19.7; with stretches, which wait for the plan first, it gains nothing).
__device__ __forceinline__ void pf_wait_expansion() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__host__ __device__ constexpr uint32_t pf_idesc(int M, int N, bool b_mn_major) {   // fp16 operands, fp32 accumulator
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// One step of the softmax for parts whose exponents lie far apart, whatever they are: a row's scores over the tile at t_s are replaced by score +
// ev of the token - ev of the tile (e), as they enter the softmax, and their sum goes without the tokens' exponents, from the scores as they were
// rounded. `own`: the tokens' ek and ev, or null where all have the tile's. Four scores at a time, then 32: little code and few registers, since
// the loops of ordinary parts must not pay for it (one loop with both cost 4 prompts of 2048 tokens 188 -> 195 us, 16 of 1024 with narrow heads
// 196 -> 212). O_t is at t_o; `first`: the part's first step, which finds none.
template <int D>
__device__ __forceinline__ void pf_special_step(uint32_t t_s, uint32_t t_o, uint64_t* p_full, const int16_t* own, float row_f, int limit,
                                                uint32_t absent, int ek, int e, bool first, float& m_ref, float& l) {
  float sum = 0.f, top = -1e30f, m_new = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < PF_TILE; c += 4) {
    uint32_t x[4];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(t_s + c) : "memory");
    const uint32_t all = ((uint32_t)(ek & 0xFF) | (uint32_t)(e & 0xFF) << 8) * 0x10001u;
    const uint2 w = own ? *reinterpret_cast<const uint2*>(own + c) : make_uint2(all, all);
    tmem_ld_wait();
    float y[4];
    const float before = top;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int both = (int16_t)((i < 2 ? w.x : w.y) >> (16 * (i & 1)));          // ek, ev
      const bool seen = c + i <= limit && !(absent >> (c >> 4) & 1u);
      const float more = (float)((both >> 8) - e);
      // (the factor is never zero: a masked score of minus infinity has to stay one)
      const float z = seen ? fmaf(__uint_as_float(x[i]), fmaxf(row_f * pf_pow2((signed char)both), 1e-37f), more) : -INFINITY;
      x[i] = __float_as_uint(z);
      y[i] = z - more;
      m_new = fmaxf(m_new, z);
      top = fmaxf(top, y[i]);
    }
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(t_s + c), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
    sum *= fast_exp2(before - top);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += fast_exp2(y[i] - top);
  }
  tmem_st_wait();
  const float ev = (float)e;
  m_new += ev;
  const bool need = m_new - m_ref > 6.f;         // as below
  if (__any_sync(0xffffffffu, need)) {
    // (the sum may outlast what the products are: exponents of values are in them only)
    const float half = need ? fast_exp2(0.5f * (m_ref - m_new)) : 1.f, alpha = half * half;
    if (need) m_ref = m_new;
    l = l * half * half;
    if (!first) {
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        tmem_ld16(t_o + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        tmem_st16(t_o + c, o);
      }
    }
  }
  if (sum != 0.f) {                              // (nothing seen: the reference may be infinite)
    // in two factors: beside the largest values the sum lies near fp32's smallest numbers, where ex2 gives zero
    const float half = fast_exp2(0.5f * (top - m_ref));
    l += sum * half * (1.f / PF_SUM_UNIT) * half;
  }
  const float shift = m_ref == -INFINITY ? 0.f : ev - m_ref;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {                  // P_t over columns of S_t that have been read
    uint32_t x[32], pk[16];
    tmem_ld32(t_s + c * 32, x);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) pk[i] = pf_half2(fast_exp2(__uint_as_float(x[2 * i]) + shift), fast_exp2(__uint_as_float(x[2 * i + 1]) + shift));
    tmem_st16(t_s + c * 16, pk);
    if (c & 1) {
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[c >> 1]);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(PF_THREADS, 1)
fa_int4_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PfArgs a) {
  using Cfg = PfCfg<D>;
  constexpr int KS = Cfg::KS, VS = Cfg::VS, CHUNKS = Cfg::CHUNKS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* q_full = bars;                 // [2]
  uint64_t* q_free = bars + 2;             // [2]
  uint64_t* k_full = bars + 4;             // [KS]
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;         // [VS]
  uint64_t* v_empty = v_full + VS;
  uint64_t* s_full = v_empty + VS;         // [2]
  uint64_t* p_full = s_full + 2;           // [2 tiles][2 halves of the keys]
  uint64_t* o_full = p_full + 4;           // [2]
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  int* status = a.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv_heads = a.heads / a.group;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the merge waits for this grid's end before it reads

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_free[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[2 * t], 128);
      mbar_init(&p_full[2 * t + 1], 128);
      mbar_init(&o_full[t], 1);
    }
    for (int s = 0; s < KS; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
    for (int s = 0; s < VS; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_ptr, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr;
  // 384 threads start with 168 registers each (64512); 128 x 96 + 256 x 200 = 63488
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 2) {
      // ------------------------------------------------------------------ Q loader
      if (lane == 0) {
        uint32_t n_q[2] = {0, 0};   // loads issued per tile (phase of q_free / q_full)
        bool ok = true;
        PfCursor c(a);
        pf_wait_expansion();
        while (c.more() && ok) {
          const PfItem it = c.next(a);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (min(c.j1, it.J[t]) <= c.j0 || !ok) continue;
            if (!mbar_wait(&q_free[t], (n_q[t] & 1) ^ 1, abort_flag, status, 94)) { ok = false; break; }
            mbar_arrive_expect_tx(&q_full[t], Cfg::TILE_BYTES);
            for (int k = 0; k < CHUNKS; ++k)
              tma_load_3d(smem + Cfg::OFF_Q + t * Cfg::TILE_BYTES + k * (PF_TILE * 128), &tm_q, &q_full[t], k * 64,
                          c.of_unit * a.line.pack, it.row0 + it.tok[t]);
            ++n_q[t];
          }
        }
      }
    } else if (warp == 0) {
      // ------------------------------------------------------------------ K / V loader
      if (lane == 0) {
        uint32_t kc = 0, vc = 0;
        bool ok = true;
        PfCursor c(a);
        pf_wait_expansion();
        while (c.more() && ok) {
          const PfItem it = c.next(a);
          const int bh = it.b * kv_heads + a.line.by_share(c.of_unit), end = min(c.j1, max(it.J[0], it.J[1]));
          for (int j = c.j0; j < end; ++j) {
            const int ks = kc % KS, vs = vc % VS;
            if (!mbar_wait(&k_empty[ks], ((kc / KS) & 1) ^ 1, abort_flag, status, 95)) { ok = false; break; }
            mbar_arrive_expect_tx(&k_full[ks], Cfg::TILE_BYTES);
            for (int k = 0; k < CHUNKS; ++k)
              tma_load_3d(smem + Cfg::OFF_K + ks * Cfg::TILE_BYTES + k * (PF_TILE * 128), &tm_k, &k_full[ks], k * 64, j * PF_TILE, bh);
            ++kc;
            if (!mbar_wait(&v_empty[vs], ((vc / VS) & 1) ^ 1, abort_flag, status, 96)) { ok = false; break; }
            mbar_arrive_expect_tx(&v_full[vs], Cfg::TILE_BYTES);
            for (int k = 0; k < CHUNKS; ++k)
              tma_load_3d(smem + Cfg::OFF_V + vs * Cfg::TILE_BYTES + k * (PF_TILE * 128), &tm_v, &v_full[vs], k * 64, j * PF_TILE, bh);
            ++vc;
          }
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer
      if (lane == 0) {
        constexpr uint32_t IDESC_S = pf_idesc(PF_TILE, PF_TILE, false);
        constexpr uint32_t IDESC_O = pf_idesc(PF_TILE, D, true);
        const uint32_t q_addr = smem_u32(smem + Cfg::OFF_Q) / 16;
        const uint32_t k_addr = smem_u32(smem + Cfg::OFF_K) / 16;
        // (V: keys are rows; the halves of its columns lie PF_TILE * 128 bytes apart)
        const uint32_t v_addr = smem_u32(smem + Cfg::OFF_V) / 16 + ((PF_TILE * 128 / 16) << 16);
        uint32_t kc = 0, vc = 0;              // K / V tiles consumed so far (ring position and phase)
        uint32_t n_q[2] = {0, 0}, n_p[2] = {0, 0};
        bool ok = true;
        auto issue_s = [&](int t, uint32_t kpos) {
          const uint32_t qa = q_addr + t * (Cfg::TILE_BYTES / 16);
          const uint32_t ka = k_addr + (kpos % KS) * (Cfg::TILE_BYTES / 16);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const int c = k >> 2, kk = k & 3;
            pf_mma<IDESC_S, PF_DESC_HI, PF_DESC_HI>(tmem_base + Cfg::COL_S + t * 128, qa + (c * (PF_TILE * 128) + kk * 32) / 16,
                                        ka + (c * (PF_TILE * 128) + kk * 32) / 16, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[t]);
        };
        PfCursor c(a);
        pf_wait_expansion();
        while (c.more() && ok) {
          const PfItem it = c.next(a);
          const int j0 = c.j0;
          int end[2];                         // steps of each tile in this part: j0 .. end - 1
#pragma unroll
          for (int t = 0; t < 2; ++t) end[t] = min(c.j1, it.J[t]);
          const int last = max(end[0], end[1]);
          if (last <= j0) continue;
          // scores of the first step for both tiles
          if (!mbar_wait(&k_full[kc % KS], (kc / KS) & 1, abort_flag, status, 97)) { ok = false; break; }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (end[t] <= j0 || !ok) continue;
            if (!mbar_wait(&q_full[t], n_q[t] & 1, abort_flag, status, 98)) { ok = false; break; }
            tc_fence_after();
            issue_s(t, kc);
            if (end[t] == j0 + 1) umma_commit(&q_free[t]);
          }
          if (!ok) break;
          umma_commit(&k_empty[kc % KS]);   // every score product of the first key tile has been issued
          ++kc;
          for (int j = j0; j < last && ok; ++j) {
            bool v_ready = false, k_ready = false;
            const bool have_next = j + 1 < last;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (j >= end[t] || !ok) continue;
              if (!mbar_wait(&p_full[2 * t], n_p[t] & 1, abort_flag, status, 99)) { ok = false; break; }
              if (!v_ready) {
                if (!mbar_wait(&v_full[vc % VS], (vc / VS) & 1, abort_flag, status, 100)) { ok = false; break; }
                v_ready = true;
              }
              tc_fence_after();
              const uint32_t va = v_addr + (vc % VS) * (Cfg::TILE_BYTES / 16);
#pragma unroll
              for (int k = 0; k < PF_TILE / 16; ++k) {   // O_t += P_t(tmem) V, the second half while its exponentials run
                if (k == PF_TILE / 32) {
                  if (!mbar_wait(&p_full[2 * t + 1], n_p[t] & 1, abort_flag, status, 104)) { ok = false; break; }
                  tc_fence_after();
                }
                pf_mma_ts<IDESC_O, PF_DESC_HI>(tmem_base + Cfg::COL_O + t * D, tmem_base + Cfg::COL_S + t * 128 + k * 8, va + k * 128,
                                     (j > j0 || k > 0) ? 1u : 0u);
              }
              if (!ok) break;
              ++n_p[t];
              if (j == end[t] - 1) umma_commit(&o_full[t]);
              if (j + 1 < end[t]) {
                if (!k_ready) {
                  if (!mbar_wait(&k_full[kc % KS], (kc / KS) & 1, abort_flag, status, 101)) { ok = false; break; }
                  tc_fence_after();
                  k_ready = true;
                }
                issue_s(t, kc);               // overwrites S_t / P_t: ordered behind the PV product just issued
                if (j + 2 == end[t]) umma_commit(&q_free[t]);   // that was the tile's last score product
              }
            }
            if (!ok) break;
            umma_commit(&v_empty[vc % VS]);
            ++vc;
            if (have_next) {
              umma_commit(&k_empty[kc % KS]);
              ++kc;
            }
          }
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (end[t] > j0) ++n_q[t];
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ------------------------------------------------------------------ softmax + epilogue
    const int t = (warp - 4) >> 2;           // query tile
    const int quarter = warp & 3;            // TMEM lane quarter this warp may access
    const int r = quarter * 32 + lane;
    const uint32_t lane_sel = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem_base + Cfg::COL_S + t * 128 + lane_sel;
    const uint32_t t_o = tmem_base + Cfg::COL_O + t * D + lane_sel;
    const bool wide = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.o_stride * 2)) & 31) == 0;
    uint32_t n_s = 0, n_o = 0;
    bool ok = true;
    PfCursor c(a);
    pf_wait_expansion();
    while (c.more() && ok) {
      const PfItem it = c.next(a);
      // (selects, not indexing: the item stays in registers)
      const int Jt = t ? it.J[1] : it.J[0], j0 = c.j0, end = min(c.j1, Jt);
      const bool whole = j0 == 0 && end == Jt && (t ? it.live[1] : it.live[0]);     // the tile's outputs are complete here
      if (end <= j0 && !whole) continue;
      const int tok = (t ? it.tok[1] : it.tok[0]) + (r >> a.line.log_pack), head = c.of_unit * a.line.pack + (r & (a.line.pack - 1));
      const int row = it.row0 + tok;
      const bool live = tok < it.q_len && (unsigned)row < (unsigned)a.total_q;
      const int limit = min(it.kv_len - 1, it.q_off + tok);
      const int* ex = a.exponents + (long long)(it.b * kv_heads + a.line.by_share(c.of_unit)) * a.line.tiles;
      const float row_f = live ? a.q_factor[(long long)row * a.heads + head] * a.scale_log2 : 0.f;      // (other rows: no spread)
      float m_ref = -INFINITY, l = 0.f;       // (no key seen yet)
      // The exponents of the part's tiles. Where some take a special step (tokens with their own, or far below the largest), the others are run
      // stretch by stretch; otherwise nothing more is looked at.
      int e_min = 127, e_max = -128, own = 0;
#pragma unroll 1
      for (int j = j0 + lane; j < end; j += 32) {
        const int w = ex[j], e = (signed char)(w >> 16);
        e_min = min(e_min, e);
        e_max = max(e_max, e);
        own |= w >> 24;
      }
      e_max = __reduce_max_sync(0xffffffffu, e_max);
      const bool plain = !__any_sync(0xffffffffu, own || e_max - e_min > PF_ALIKE);
      for (int j = j0; j < end && ok;) {
        int stop = end;                       // the next tile that takes a special step
        if (!plain) {
          for (int b = j; b < stop; b += 32) {
            const int w = ex[min(b + lane, end - 1)], e = (signed char)(w >> 16);
            const uint32_t found = __ballot_sync(0xffffffffu, b + lane < end && (w >> 24 || e < e_max - PF_ALIKE));
            if (found) stop = b + __ffs(found) - 1;
          }
          if (stop == j) {
            ok = mbar_wait(&s_full[t], n_s & 1, abort_flag, status, 102);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ++n_s;
            tc_fence_after();
            const int w = ex[j];
            pf_special_step<D>(t_s, t_o, &p_full[2 * t], w >> 24 ? a.own + (ex + j - a.exponents) * PF_TILE : nullptr, row_f, limit - j * PF_TILE,
                               (uint32_t)w >> 8 & 0xFFu, (signed char)w, (signed char)(w >> 16), j == j0, m_ref, l);
            ++j;
            continue;
          }
        }
        int e_next = ex[j];
        for (; j < stop && ok; ++j) {
          const int ek = (signed char)e_next, e = (signed char)(e_next >> 16);
          const uint32_t absent = (uint32_t)e_next >> 8 & 0xFFu;     // sixteens of keys without a page: no query sees them
          if (j + 1 < end) e_next = ex[j + 1];
          // (never zero: a masked score of minus infinity has to stay one)
          const float sc = fmaxf(row_f * pf_pow2(ek), 1e-37f), ev = (float)e;
          ok = mbar_wait(&s_full[t], n_s & 1, abort_flag, status, 102);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          ++n_s;
          tc_fence_after();
          uint32_t sr[4][32];
          float* s = reinterpret_cast<float*>(&sr[0][0]);
          const int kv0 = j * PF_TILE;
          const auto hide = [&](int from, int to) {
            if (kv0 + to - 1 > limit) {
#pragma unroll
              for (int i = from; i < to; ++i)
                if (kv0 + i > limit) s[i] = -INFINITY;
            }
            if (absent) {
#pragma unroll
              for (int i = from; i < to; ++i)
                if (absent >> (i >> 4) & 1u) s[i] = -INFINITY;
            }
          };
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, sr[c]);
          tmem_ld_wait();
          hide(0, 128);
          uint64_t rs2[4] = {0ull, 0ull, 0ull, 0ull};
          uint32_t pk[2][32];
          const auto exponentials = [&](int h) {   // of half h of the keys: fp16 pairs to pk[h], sums to rs2
            const float shift = m_ref == -INFINITY ? 0.f : ev - m_ref;      // (without a key every score is minus infinity)
            const uint64_t sc2 = f32x2(sc, sc), nm2 = f32x2(shift, shift);
#pragma unroll
            for (int i = 64 * h; i < 64 * h + 64; i += 2) {
              float e0f, e1f;
              f32x2_unpack(fma_f32x2(f32x2(s[i], s[i + 1]), sc2, nm2), e0f, e1f);
              const float p0 = fast_exp2(e0f), p1 = fast_exp2(e1f);
              rs2[(i >> 1) & 3] = add_f32x2(rs2[(i >> 1) & 3], f32x2(p0, p1));
              pk[h][(i >> 1) & 31] = pf_half2(p0, p1);
            }
          };
          const auto publish = [&](int h) {        // P_t: fp16 pairs over the first 64 columns of S_t
            tmem_st32(t_s + 32 * h, pk[h]);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&p_full[2 * t + h]);
          };
          // The reference rarely moves: the first half's exponentials are taken with the one there is, with the maximum of all
          // 128 scores in their shadow, and again where it does (257 us -> 242 at 2048 over 6144; the registers that takes come from
          // the service warps).
          if (j > j0) exponentials(0);
          float mx4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int i = 4; i < 124; i += 8) {
            mx4[0] = fmax3(mx4[0], s[i], s[i + 1]);
            mx4[1] = fmax3(mx4[1], s[i + 2], s[i + 3]);
            mx4[2] = fmax3(mx4[2], s[i + 4], s[i + 5]);
            mx4[3] = fmax3(mx4[3], s[i + 6], s[i + 7]);
          }
          mx4[0] = fmax3(mx4[0], s[124], s[125]);
          mx4[1] = fmax3(mx4[1], s[126], s[127]);
          const float m_new = fmaf(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), sc, ev);
          // p up to 2^6 until the reference moves. The first score that is seen always sets it, in whatever tile it stands: a
          // reference of zero kept from a tile without a visible key left p as 2^(score + ev), which fp16 may not hold.
          const bool need = m_new - m_ref > 6.f;
          if (j == j0 || __any_sync(0xffffffffu, need)) {
            const float half = need ? fast_exp2(0.5f * (m_ref - m_new)) : 1.f, alpha = half * half;
            if (need) m_ref = m_new;
            if (j > j0) {
              l = l * half * half;             // (in two steps, as in special ones)
              // S_t(j) complete implies PV_t(j-1) complete (same issuing thread, commit covers earlier MMAs):
              // O_t is quiescent until this warpgroup arrives on p_full, so a rescale can happen right here.
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                tmem_ld32(t_o + c * 32, pk[0]);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) pk[0][i] = __float_as_uint(__uint_as_float(pk[0][i]) * alpha);
                tmem_st32(t_o + c * 32, pk[0]);
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) rs2[q] = 0ull;
              tmem_ld32(t_s, sr[0]);               // (the first half again: its registers need not outlive the exponentials)
              tmem_ld32(t_s + 32, sr[1]);
              tmem_ld_wait();
              hide(0, 64);
            }
            exponentials(0);
          }
          publish(0);
          exponentials(1);
          publish(1);
          float rs[8];
#pragma unroll
          for (int q = 0; q < 4; ++q) f32x2_unpack(rs2[q], rs[2 * q], rs[2 * q + 1]);
          l += (((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]))) * pf_pow2(-e) * (1.f / PF_SUM_UNIT);
        }
      }
      if (!ok) break;
      if (end > j0) {
        ok = mbar_wait(&o_full[t], n_o & 1, abort_flag, status, 103);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++n_o;
        tc_fence_after();
      }
      // p 2^ev and the values' 2^-ev cancel in O
      const float inv_l = l == 0.f ? 0.f : 1.f / PF_SUM_UNIT / l;
      __nv_bfloat16* orow = a.out + (long long)row * a.o_stride + (long long)head * D;
      float* part = a.parts + (long long)((blockIdx.x * 2 + c.slot) * 2 + t) * pf_part_floats<D>();
#pragma unroll 1
      for (int k = 0; k < D / 32; ++k) {
        uint32_t orr[32];                 // (without a key: whatever the columns hold, not used)
        tmem_ld32(t_o + k * 32, orr);
        tmem_ld_wait();
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(part + ((k * 8 + i) * PF_TILE + r) * 4) =
                make_uint4(orr[4 * i], orr[4 * i + 1], orr[4 * i + 2], orr[4 * i + 3]);
        } else if (live) {
          uint32_t v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            v[i] = l == 0.f ? 0u : pack_bf16x2(__uint_as_float(orr[2 * i]) * inv_l, __uint_as_float(orr[2 * i + 1]) * inv_l);
          // rows lie far apart: a lane writes whole 32-byte sectors where they are aligned
          __nv_bfloat16* at = orow + k * 32;
          if (wide) {
            pf_store32(at, v);
            pf_store32(at + 16, v + 8);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(at)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
      }
      if (!whole) {
        part[PF_TILE * D + r] = m_ref;
        part[PF_TILE * (D + 1) + r] = l;
      }
      // The TMEM loads above have completed (tmem_ld_wait); the next part's first PV product waits for
      // this warpgroup's next arrives on p_full, so O_t is not overwritten before it was read.
      tc_fence_before();
    }
  }

  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 10000000LL) {}
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// Joins the parts of query tiles that lie in several stretches: blockIdx.x names the border (the start of a stretch) that cuts
// the item first; 16 values of 128 rows of one of its tiles per block, two threads per row.
template <int D>
__global__ void __launch_bounds__(256)
pf_merge_kernel(const __grid_constant__ PfArgs a) {
  const int border = blockIdx.x + 1, t = blockIdx.y & 1;
  asm volatile("griddepcontrol.wait;" ::: "memory");             // every CTA, so that this grid ends behind the one before
  if (border >= a.plan.count()) return;
  const int* start = a.plan.start(border);
  const int per = a.plan.per(), rem = a.plan.rem(), pair = start[0], unit = start[1], u0 = pf_start(per, rem, border) - start[2];
  if (start[2] == 0 || pf_start(per, rem, border - 1) > u0) return;      // no cut, or not the item's first
  const PfItem it(a.line, pair);
  const int Jt = t ? it.J[1] : it.J[0];
  if (!(t ? it.live[1] : it.live[0]) || Jt == 0) return;
  const int first = u0 + PF_SETUP, c0 = pf_owner(per, rem, first), c1 = pf_owner(per, rem, first + Jt - 1);
  if (c0 == c1) return;                           // written by that CTA
  const int r = threadIdx.x >> 1, v0 = (blockIdx.y >> 1) * 4 + (threadIdx.x & 1) * 2;      // row, first group of four values
  const auto part = [&](int c) {
    return a.parts + (long long)((c * 2 + (u0 > pf_start(per, rem, c) ? 1 : 0)) * 2 + t) * pf_part_floats<D>();
  };
  float M = -INFINITY, l = 0.f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 2
  for (int c = c0; c <= c1; ++c) {
    const float* p = part(c);
    const float m = p[PF_TILE * D + r], lc = p[PF_TILE * (D + 1) + r];
    float4 v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) v[k] = *reinterpret_cast<const float4*>(p + ((v0 + k) * PF_TILE + r) * 4);
    if (lc == 0.f) continue;                      // nothing seen (a NaN is not nothing)
    const float Mn = fmaxf(M, m), h0 = l == 0.f ? 0.f : fast_exp2(0.5f * (M - Mn)), h = fast_exp2(0.5f * (m - Mn)), w0 = h0 * h0, w = h * h;
    M = Mn;
    l = fmaf(h, h * lc, h0 * (h0 * l));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      acc[k].x = fmaf(w, v[k].x, acc[k].x * w0);
      acc[k].y = fmaf(w, v[k].y, acc[k].y * w0);
      acc[k].z = fmaf(w, v[k].z, acc[k].z * w0);
      acc[k].w = fmaf(w, v[k].w, acc[k].w * w0);
    }
  }
  const int tok = (t ? it.tok[1] : it.tok[0]) + (r >> a.line.log_pack), head = unit * a.line.pack + (r & (a.line.pack - 1)), row = it.row0 + tok;
  if (tok >= it.q_len || (unsigned)row >= (unsigned)a.total_q) return;
  const float inv = l == 0.f ? 0.f : 1.f / PF_SUM_UNIT / l;
  uint32_t y[4];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    y[2 * k] = l == 0.f ? 0u : pack_bf16x2(acc[k].x * inv, acc[k].y * inv);
    y[2 * k + 1] = l == 0.f ? 0u : pack_bf16x2(acc[k].z * inv, acc[k].w * inv);
  }
  *reinterpret_cast<uint4*>(a.out + (long long)row * a.o_stride + (long long)head * D + v0 * 4) = make_uint4(y[0], y[1], y[2], y[3]);
}

// Sizes of a call's workspace and launches.
// Bytes of the images of keys and values: every sequence has room for the longest, so a batch that holds a long one beside many
// short ones would ask for far more than it reads. What does not fit is dealt with in slices of the batch, one after the other.
constexpr long long PF_IMAGES = 1LL << 31;
struct PfSizes {
  int tiles, pack, units, n_qb, ctas;
  int per_item;
  int slice;                            // sequences at a time; the rest is for one slice
  bool whole;
  long long kv_tiles, pairs, steps;     // steps: places on the line, at most
  long long kv, q, factor, exponents, own, plan, parts, total;    // bytes, each a multiple of 256
};
PfSizes pf_sizes(int batch, int total_q, int max_q, int max_kv, int heads, int kv_heads, int D) {
  const auto align = [](long long n) { return (n + 255) / 256 * 256; };
  PfSizes z;
  const int G = heads / kv_heads;
  z.tiles = std::max(1, (max_kv + PF_TILE - 1) / PF_TILE);
  z.pack = PF_TILE % G == 0 ? G : 1;
  z.units = heads / z.pack;
  z.slice = (int)std::max(1LL, std::min((long long)batch, PF_IMAGES / (4LL * kv_heads * z.tiles * PF_TILE * D)));
  z.kv_tiles = (long long)z.slice * kv_heads * z.tiles;
  const long long q_tiles = ((long long)max_q * z.pack + PF_TILE - 1) / PF_TILE;
  z.per_item = z.slice * q_tiles * z.units <= sm_count() && z.tiles <= PF_SINGLE_STEPS ? 1 : 2;
  z.n_qb = (int)((q_tiles + z.per_item - 1) / z.per_item);
  z.pairs = (long long)z.slice * z.n_qb;
  z.steps = z.pairs * z.units * (z.tiles + PF_SETUP);
  z.whole = z.per_item == 1 || (z.pairs * z.units <= sm_count() && z.tiles <= PF_WHOLE_STEPS);
  z.ctas = (int)(z.whole ? std::max(1LL, z.pairs * z.units) : std::max(1LL, std::min((long long)sm_count(), z.steps / PF_MIN_STEPS)));
  z.kv = align(z.kv_tiles * PF_TILE * D * 2);
  z.q = align((long long)total_q * heads * D * 2);
  z.factor = align((long long)total_q * heads * 4);
  z.exponents = align(z.kv_tiles * 4);
  z.own = align(z.kv_tiles * PF_TILE * 2);
  z.plan = align((4 + 4LL * z.ctas) * 4);
  z.parts = z.whole ? 0 : align(4LL * z.ctas * PF_TILE * (D + 2) * 4);
  z.total = 2 * z.kv + z.q + z.factor + z.exponents + z.own + z.plan + z.parts;
  return z;
}

}  // namespace

long long prompt_int4_workspace(int batch, int total_q, int max_q, int max_kv, int heads, int kv_heads, int head_dim) {
  return pf_sizes(batch, total_q, max_q, max_kv, heads, kv_heads, head_dim).total;
}

void prompt_int4(const KvInt4Cache& c, const void* q, long long q_stride, const int* cu_q, const int* kv_lens, void* out,
                 long long o_stride, int batch, int total_q, int max_q, int max_kv, int heads, float scale, void* workspace,
                 int* status, cudaStream_t stream) {
  const int D = c.head_dim;
  const PfSizes z = pf_sizes(batch, total_q, max_q, max_kv, heads, c.kv_heads, D);
  uint8_t* p = (uint8_t*)workspace;
  const auto take = [&](long long bytes) {
    uint8_t* at = p;
    p += bytes;
    return at;
  };
  PfExpand x{(const uint8_t*)c.k, (const uint8_t*)c.v,
             {c.block_table, c.n_seqs, c.max_pages, c.n_pages, c.kv_heads, c.page_size, kv4_div(c.page_size)}, kv_lens,
             (const __nv_bfloat16*)q, q_stride};
  x.k = (__half*)take(z.kv);
  x.v = (__half*)take(z.kv);
  x.qh = (__half*)take(z.q);
  x.q_factor = (float*)take(z.factor);
  x.exponents = (int*)take(z.exponents);
  x.own = (int16_t*)take(z.own);
  x.plan = {(int*)take(z.plan)};
  float* parts = (float*)take(z.parts);
  x.kv_heads = c.kv_heads;
  x.heads = heads;
  x.tiles = z.tiles;
  x.q_rows = (int)((long long)total_q * heads);
  x.by_heads = kv4_div(heads);
  x.max_q = max_q;
  x.max_kv = max_kv;
  x.status = status;
  int log_pack = 0;
  while (1 << log_pack < z.pack) ++log_pack;
  const int rows_per = PF_EXPAND / (D / 8) * PF_Q_ROWS;
  MB_REQUIRE((long long)total_q * heads < (1LL << 31) - rows_per, "paged_attn_prefill_int4: too many query rows");
  const long long q_blocks = ((long long)total_q * heads + rows_per - 1) / rows_per;
  MB_REQUIRE(z.kv_tiles + q_blocks + 1 < (1LL << 31) && z.steps < (1LL << 31) && z.pairs < (1LL << 31), "paged_attn_prefill_int4: batch too large");
  // (copies only: TMA moves fp16 as it moves bf16)
  uint64_t qd[3] = {(uint64_t)D, (uint64_t)heads, (uint64_t)total_q}, qs[2] = {(uint64_t)D * 2, (uint64_t)heads * D * 2};
  uint32_t qb[3] = {64, (uint32_t)z.pack, (uint32_t)(PF_TILE / z.pack)};
  const CUtensorMap tq = make_tensor_map(x.qh, TmaDType::BF16, 3, qd, qs, qb, true);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;

  for (int b0 = 0; b0 < batch; b0 += z.slice) {
    const int nb = std::min(z.slice, batch - b0);
    const PfSizes s = pf_sizes(nb, total_q, max_q, max_kv, heads, c.kv_heads, D);
    x.pages.block_table = c.block_table + (long long)b0 * c.max_pages;
    x.pages.n_seqs = c.n_seqs - b0;
    x.kv_lens = kv_lens + b0;
    x.line = {cu_q + b0, kv_lens + b0, nb, s.pack, log_pack, s.units, s.n_qb, s.tiles, s.per_item, kv4_div(std::max(1, s.n_qb)), kv4_div(s.units / c.kv_heads)};
    x.pairs = (int)s.pairs;
    x.ctas = s.ctas;
    x.kv_blocks = (int)s.kv_tiles;
    x.q_blocks = b0 == 0 ? (int)q_blocks : 0;
    const unsigned blocks = (unsigned)x.kv_blocks + (unsigned)x.q_blocks + 1u;
    if (D == 128) kv4_expand_kernel<128><<<blocks, PF_EXPAND, 0, stream>>>(x);
    else kv4_expand_kernel<64><<<blocks, PF_EXPAND, 0, stream>>>(x);
    count_launch();
    check_launch();

    uint64_t kd[3] = {(uint64_t)D, (uint64_t)s.tiles * PF_TILE, (uint64_t)nb * c.kv_heads};
    uint64_t ks[2] = {(uint64_t)D * 2, (uint64_t)s.tiles * PF_TILE * D * 2};
    uint32_t kb[3] = {64, PF_TILE, 1};
    const CUtensorMap tk = make_tensor_map(x.k, TmaDType::BF16, 3, kd, ks, kb, true);
    const CUtensorMap tv = make_tensor_map(x.v, TmaDType::BF16, 3, kd, ks, kb, true);
    PfArgs a{x.line, x.plan, x.q_factor, x.exponents, x.own, (__nv_bfloat16*)out, parts, o_stride, heads, heads / c.kv_heads, total_q,
             scale * 1.4426950408889634f, status, s.whole, kv4_div(s.units)};
    const auto go = [&](auto kern, auto merge, int smem) {
      MB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      cfg.gridDim = dim3((unsigned)s.ctas);
      cfg.blockDim = dim3(PF_THREADS);
      cfg.dynamicSmemBytes = smem;
      cfg.numAttrs = s.whole ? 1 : 0;
      MB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, a));
      if (s.whole) return;
      cfg.gridDim = dim3((unsigned)std::max(1, s.ctas - 1), 2 * (D / 16));
      cfg.blockDim = dim3(256);
      cfg.dynamicSmemBytes = 0;
      cfg.numAttrs = 1;
      MB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, merge, a));
    };
    if (D == 128) go(fa_int4_kernel<128>, pf_merge_kernel<128>, PfCfg<128>::SMEM_BYTES);
    else go(fa_int4_kernel<64>, pf_merge_kernel<64>, PfCfg<64>::SMEM_BYTES);
    count_launch(s.whole ? 1 : 2);
  }
}

}  // namespace mb
