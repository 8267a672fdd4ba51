// Format of the 4-bit paged KV cache, shared by the kernels that write and read it.
//
// A row of D values (one token, one kv head, K or V; D = 64 or 128) is cut into groups of 64. A group is
// stored as scale = bf16((max - min) / 15), low = min (a bf16 already, so exact) and 64 codes
// clamp(round_to_even((x - low) / scale), 0, 15); it stands for scale * code + low. The range is kept
// asymmetric because keys carry per-channel offsets: a symmetric scale would spend codes on values that do
// not occur. The scale is rounded to bf16 (half the bytes of fp32): codes are formed against the rounded
// scale, so its rounding moves the grid by at most 2^-8 of a step per code and adds no error of its own.
// 64 values per group cost 4.5 bits a value; groups of 32 would cost 5 (one ninth more bytes to read per
// decoded token). A group with a NaN, an infinity or a range beyond fp32 has a NaN or infinite scale and
// reads back as NaN: nothing finite is made up.
//
// A cache is [pages, kv_heads, page_size / 16 tiles, TILE_BYTES] bytes. A tile is 16 tokens: 16 rows of codes
// (D / 2 bytes each), then 16 rows of (scale, low) pairs (D / 16 bytes each); contiguous, a multiple of 16
// bytes, fetched in 16-byte pieces. The order inside a tile is that of the tensor-core fragments the attention
// kernel builds, so that a thread reads its operands with 16-byte (keys) and 8-byte (values) shared loads,
// without bank conflicts and without ldmatrix:
//   * eight consecutive values share a 32-bit word; value 2 i + j sits in nibble i + 4 j: word >> 4 i masked by
//     0x000F000F is the pair (2 i, 2 i + 1) in the two halves of a register;
//   * token n of a tile has key row (and pair row, K and V) 8 (n / 8) + 2 (n % 4) + (n / 4) % 2 and value row n:
//     the score fragment of a thread (columns 2 t, 2 t + 1 of two 8-token products) then covers tokens t, t + 4,
//     t + 8 and t + 12, whose value rows lie in different banks for the four t;
//   * a key row is [t = 0..3][group][2 words]: values 64 g + 16 t + 8 h ...; the words are rotated left by three
//     bits, so that two nibbles of a half lie within the top bits of a 16-bit float's mantissa;
//   * a value row is [r = 0..7][group][1 word]: values 64 g + 8 r ...; chunk r is stored at place r ^ 4 ((n / 2) % 2).
#pragma once
#include "common.cuh"
#include "tc.cuh"

namespace mb {

template <int D>
struct KvInt4 {
  static constexpr int GROUPS = D / 64;
  static constexpr int ROW = D / 2;                  // code bytes of a token
  static constexpr int PAIR = GROUPS * 4;            // (scale, low) bytes of a token
  static constexpr int OFF_PAIR = 16 * ROW;
  static constexpr int TILE_BYTES = 16 * (ROW + PAIR);
};

// Row of token n (0..15) among the key rows and the pair rows of a tile.
__device__ __forceinline__ int kv4_row(int n) { return (n & 8) + ((n & 3) << 1) + ((n >> 2) & 1); }
// Byte offset of the word that holds values 64 g + 8 u .. (u = 0..7) inside a tile.
template <int D>
__device__ __forceinline__ int kv4_key_word(int n, int g, int u) {
  return kv4_row(n) * KvInt4<D>::ROW + ((u >> 1) * KvInt4<D>::GROUPS + g) * 8 + (u & 1) * 4;
}
template <int D>
__device__ __forceinline__ int kv4_value_word(int n, int g, int u) {
  return n * KvInt4<D>::ROW + ((u ^ (((n >> 1) & 1) << 2)) * KvInt4<D>::GROUPS + g) * 4;
}
template <int D>
__device__ __forceinline__ int kv4_pair(int n, int g) {
  return KvInt4<D>::OFF_PAIR + kv4_row(n) * KvInt4<D>::PAIR + g * 4;
}

// Quotient by a number the host knows: n * mul / 2^shift with mul = ceil(2^shift / d), shift = 31 + ceil(log2 d); exact for
// 0 <= n < 2^31.
struct Kv4Div {
  uint32_t mul;
  int shift;
  __device__ __forceinline__ int operator()(int n) const { return (int)((unsigned long long)(unsigned)n * mul >> shift); }
};
inline Kv4Div kv4_div(int d) {
  int s = 0;
  while ((1LL << s) < d) ++s;
  return {(uint32_t)(((1ULL << (31 + s)) + (unsigned)d - 1) / (unsigned)d), 31 + s};
}

// Where tokens live.
struct Kv4Pages {
  const int* block_table;
  int n_seqs, max_pages, n_pages, kv_heads, page_size;
  Kv4Div by_page;
  // First tile (of head 0) of the token at `pos` of a sequence, or -1 for one without a page: a sequence or position outside
  // the table, a page id outside the cache. Heads of a page are page_size / 16 tiles apart.
  __device__ __forceinline__ int tile0(int seq, int pos) const {
    if ((unsigned)seq >= (unsigned)n_seqs || pos < 0) return -1;
    const int lp = by_page(pos);
    if (lp >= max_pages) return -1;
    const int page = block_table[(long long)seq * max_pages + lp];
    if ((unsigned)page >= (unsigned)n_pages) return -1;
    return page * kv_heads * (page_size >> 4) + ((pos - lp * page_size) >> 4);
  }
  __device__ __forceinline__ int tile(int seq, int pos, int head) const {
    const int t = tile0(seq, pos);
    return t < 0 ? -1 : t + head * (page_size >> 4);
  }
};

// Quotients are formed as a product with the correctly rounded reciprocal and one residual correction, which gives the
// correctly rounded quotient (Markstein, IBM J. Res. Dev. 34, 1990) where nothing over- or underflows: the division's own
// range checks had made the append instruction-bound at 4.6 times its floor. Outside that range the division is taken.
// (scale, low) of a group from its extremes; the low half of the word is the scale.
__device__ __forceinline__ uint32_t kv4_make_pair(__nv_bfloat16 lo, __nv_bfloat16 hi, float& scale, float& low) {
  low = __bfloat162float(lo);
  const float range = __bfloat162float(hi) - low, q = range * (1.f / 15.f);
  float d = fmaf(fmaf(-q, 15.f, range), 1.f / 15.f, q);
  if (!(range > 0x1p-90f && range < 0x1p120f)) d = __fdiv_rn(range, 15.f);
  const __nv_bfloat16 s = __float2bfloat16(d);
  scale = __bfloat162float(s);
  return (uint32_t)__bfloat16_as_ushort(s) | (uint32_t)__bfloat16_as_ushort(lo) << 16;
}
__device__ __forceinline__ uint32_t kv4_code(float x, float scale, float low) {
  // true division: the nearest code, ties to even (a product with the reciprocal would move ties)
  const int c = __float2int_rn(__fdiv_rn(x - low, scale));
  return scale > 0.f ? (uint32_t)max(0, min(15, c)) : 0u;
}
// Word of eight consecutive values (four bf16 pairs). Adding 3 * 2^22 rounds to an integer in the low bits. Packed fp32 pairs
// halve the issue slots, which bound the kernel.
__device__ __forceinline__ uint32_t kv4_word(const bf16x8& x, float scale, float low, float inv) {
  uint32_t w = 0u;
  if (scale > 0x1p-100f && scale < 0x1p110f) {
    const uint64_t s2 = f32x2(-scale, -scale), l2 = f32x2(-low, -low), i2 = f32x2(inv, inv), round2 = f32x2(12582912.f, 12582912.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(x.v[i]);
      const uint64_t t = add_f32x2(f32x2(f.x, f.y), l2), q = mul_f32x2(t, i2);
      float a, b;
      f32x2_unpack(add_f32x2(fma_f32x2(fma_f32x2(q, s2, t), i2, q), round2), a, b);
      w += __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410) * (1u << (4 * i));
    }
    return w;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(x.v[i]);
    w |= (kv4_code(f.x, scale, low) | kv4_code(f.y, scale, low) << 16) << (4 * i);
  }
  return w;
}
__device__ __forceinline__ uint32_t kv4_rotate(uint32_t w) { return __funnelshift_l(w, w, 3); }
__device__ __forceinline__ uint32_t kv4_unrotate(uint32_t w) { return __funnelshift_r(w, w, 3); }
__device__ __forceinline__ float kv4_scale(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float kv4_low(uint32_t pair) { return __uint_as_float(pair & 0xFFFF0000u); }
// Whether a group's scale and low are finite.
__device__ __forceinline__ bool kv4_finite(uint32_t pair) { return (pair & 0x7F80u) != 0x7F80u && (pair & 0x7F800000u) != 0x7F800000u; }

}  // namespace mb
