// The layout of a matrix held in 8-bit floating point, and what its kernels share.
//
// A matrix [rows, K] is held as OCP e4m3 codes with one scale 2^(b - 127), b a byte, for each
// (row, 128 values of K): value = code * scale. b is the least with max |x| <= 448 * scale, so
// the largest value's code lies in (224, 448] and a code is within 2^-4 of its value (relative;
// below 2^-6 of the scale within 2^-10 of it). It is the nearest code but for one: at the largest
// scale, 2^120, a code of 256 would stand for 2^128, past the largest fp32 and bf16, so values
// from 248 * 2^120 on get 240. A power of two costs nothing against a scale of more bits: codes are
// floating point themselves, dividing by it is exact, and the instructions that take codes apply
// it, so sums stay in the accumulators.
// A block with a NaN or an infinity holds NaN codes and b = 255: it reads back as NaN.
//
// Codes lie in the order in which v_mfma_scale_f32_16x16x128_f8f6f4 takes them: a tile of 16 rows
// and 128 values is one block of 2 KB, the blocks of a tile follow one another along K. In a block, lane l of a
// wavefront owns the bytes [16 l, 16 l + 16) of either KB j: row l % 16, values
// 64 j + 16 (l / 16) + 0..15. Loads are 1 KB a wavefront, to registers or LDS alike, and LDS
// holds blocks as they are with no bank conflicts. Any order of K inside a block would do, as
// both factors have the same and all 128 values of a row share a scale.
//
// Two ways to multiply blocks, both with fp32 accumulators:
// - that instruction on the codes (5 PFLOP/s dense at this GPU's peak). Of the 8 products of a
//   lane's 8 neighbouring bytes it keeps what lies above 2^-13 of the largest one's binade
//   (measured with one product 2^k beside one of 1 + 2^-2 + 2^-6: bits below 2^(k - 13) are cut off,
//   across neighbouring eights none): each product loses less than 2^-13 of its eight's largest,
//   where its codes' own rounding is 2^-4. A typical sum is 2^-14 off.
// - the codes times their scale as bf16 (exact: 4 significant bits) on
//   v_mfma_f32_16x16x32_bf16, half the rate, whose sums are fp32 throughout.
// Up to 32 rows wait for memory, not for the matrix cores, and an fp32 result shows its sums' last
// bits: these take the second; more rows with bf16 results, whose step is 2^-8, the first. So a row's
// bf16 result may be another in its last bit among 33 rows than among 32.
//
// Scales: [tile][quad of blocks][16 rows][4 blocks] bytes, so a lane's dword holds its row's
// scales of 4 blocks and the instruction's op_sel picks one. Rows past the end and values past
// K are zeros; so is the padding of scales.
//
// A pair (gate | up, [2 n, K]) has 8 rows of either half in a tile: rows 0..7 of tile t are 8 t.. of
// the first half, rows 8..15 of the second, each half padded to whole eights. A lane and the one 32
// places on then end with the sums of a gate column and of its up column.
#pragma once

#include "ko_common.h"

namespace ko {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int FP8_BLOCK = 2048;   // bytes of a block of codes: 16 rows, 128 values
constexpr int FP8_K_MAX = 1 << 27;   // so that a byte's place in a tile stays below 2^31

// Whether one launch takes as many workgroups: a grid has fewer than 2^32 threads.
inline bool fp8_launchable(long long groups, int threads) { return groups * threads < 1ll << 32; }

__host__ __device__ __forceinline__ int fp8_blocks(int K) { return (K + 127) >> 7; }
__host__ __device__ __forceinline__ int fp8_quads(int K) { return (K + 511) >> 9; }
__host__ __device__ __forceinline__ long long fp8_tiles(int rows, bool pair) {
  return pair ? (rows / 2 + 7ll) / 8 : (rows + 15ll) / 16;
}

// The row of [rows, K] that row r of tile t holds, or -1.
__device__ __forceinline__ int fp8_row(long long t, int r, int rows, bool pair) {
  if (!pair) {
    const long long row = t * 16 + r;
    return row < rows ? (int)row : -1;
  }
  const int n = rows >> 1;
  const long long row = t * 8 + (r & 7);
  return row < n ? (int)((r >> 3) * n + row) : -1;
}

// The scale's byte for a block whose largest |x| has these bits (NaN and infinity sort above
// every number): 448 = 1.75 * 2^8. At most 247, or 255.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23), b = e - 8 + ((amax_bits & 0x7fffffu) > 0x600000u);
  return e == 255 ? 255u : (uint32_t)max(b, 0);
}
// 2^-(b - 127), b <= 247; the product with a value of the block is exact down to fp32's
// subnormals, far below what a code can hold.
__device__ __forceinline__ float fp8_inverse(uint32_t b) { return __uint_as_float((254u - b) << 23); }
__device__ __forceinline__ float fp8_scale(uint32_t b) {
  return b == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(b ? b << 23 : 0x400000u);
}

// Four codes of v * inv (to nearest, ties to even), or of NaN.
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
  return (uint32_t)w;
}

// Four codes of a block whose scale byte is 247 or more: NaN (255), or with 240 for 256, the largest
// that such a block can have.
__device__ __forceinline__ uint32_t fp8_top4(uint32_t w, uint32_t b) {
  return b == 255 ? 0x7f7f7f7fu : w - ((w & w >> 1 & w >> 2 & w >> 3 & 0x08080808u) >> 3);
}

__device__ __forceinline__ uint32_t umax_xor16(uint32_t u) {
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return max((uint32_t)p[0], (uint32_t)p[1]);
}
__device__ __forceinline__ uint32_t umax_xor32(uint32_t u) {
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return max((uint32_t)p[0], (uint32_t)p[1]);
}

// A block in registers: lane l holds the values 64 j + 16 (l / 16) + 0..15, j = 0, 1, of row l % 16.
// Its codes, in the lane's bytes of the layout above; returns the row's scale byte.
__device__ __forceinline__ uint32_t fp8_quantize_block(const float (&v)[2][16], uint4 (&c)[2]) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
  top = umax_xor32(umax_xor16(top));
  const uint32_t b = fp8_scale_byte(top);
  const float inv = fp8_inverse(min(b, 247u));
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = fp8_pack4(v[j][4 * i], v[j][4 * i + 1], v[j][4 * i + 2], v[j][4 * i + 3], inv);
      if (b >= 247) w[i] = fp8_top4(w[i], b);
    }
    c[j] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return b;
}

// The sum of the squares of 8 values, in order.
__device__ __forceinline__ float fp8_squares(const float* v) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += v[i] * v[i];
  return s;
}
// The sum of the squares of a block's row of 128, its eights' sums c = 0..15 added as a tree: c and
// c + 8, then 4, 2 and 1 apart. A row's sum adds its blocks' in order, in 64 bits. Every kernel forms both so,
// whatever its lanes hold, and all find the same norm. Here the block is in registers as above.
__device__ __forceinline__ float fp8_square_sum(const float (&v)[2][16]) {
  float s[2];
#pragma unroll
  for (int p = 0; p < 2; ++p)
    s[p] = sum_xor16(sum_xor32(fp8_squares(v[0] + 8 * p) + fp8_squares(v[1] + 8 * p)));
  return s[0] + s[1];
}

// 8 values of a block's row in each of 16 neighbouring lanes (a DPP row): their codes; returns the
// block's scale byte. q: packed bf16.
__device__ __forceinline__ uint32_t fp8_quantize8(const uint4& q, uint2& c) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t top = 0;   // of 15-bit magnitudes, which compare as the floats do
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
  int m = (int)top;
  m = max(m, dpp_i<0x128>(m));
  m = max(m, dpp_i<0x124>(m));
  m = max(m, dpp_i<0x122>(m));
  m = max(m, dpp_i<0x121>(m));
  const uint32_t b = fp8_scale_byte((uint32_t)m << 16);
  const float inv = fp8_inverse(min(b, 247u));
  c.x = fp8_pack4(bf16lo(w[0]), bf16hi(w[0]), bf16lo(w[1]), bf16hi(w[1]), inv);
  c.y = fp8_pack4(bf16lo(w[2]), bf16hi(w[2]), bf16lo(w[3]), bf16hi(w[3]), inv);
  if (b >= 247) c.x = fp8_top4(c.x, b), c.y = fp8_top4(c.y, b);
  return b;
}

// 1 / sqrt(sum / K + eps), to fp32's nearest but for one in millions: the instruction's, which is up to
// an ulp off, with one of Newton's steps in 64 bits. Every bit of it that is wrong moves that much more of a
// row's values over a bf16 border, and some of their codes with them; a row has one.
__device__ __forceinline__ float fp8_rstd(double sum, int K, float eps) {
  const double v = sum / K + (double)eps;
  const float y = rsqrtf((float)v);
  if (!(v > 1e-37 && v < 1e37)) return y;   // no row's but one of zeros or of huge values
  return (float)(y * (1.5 - 0.5 * v * y * y));
}

// bf16(gain * bf16(x * rstd)) of packed pairs, as the bf16 chain rounds.
__device__ __forceinline__ uint32_t fp8_norm2(uint32_t x, uint32_t w, float rstd) {
  const uint32_t t = pack_bf16x2(bf16lo(x) * rstd, bf16hi(x) * rstd);
  return pack_bf16x2(bf16lo(w) * bf16lo(t), bf16hi(w) * bf16hi(t));
}

// 8 codes (the dwords w0, w1) times 2^(b - 127) as bf16; scale = b << 23.
__device__ __forceinline__ bf16x8 fp8_to_bf16(uint32_t w0, uint32_t w1, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace ko
