// A KV cache held in 4 bits: the block format, and the quantiser that every writer shares.
//
// Groups of d / NG values of a head vector share a scale s and a value c, both bf16:
//   x = c + s (n - 8),  n = 0..15.
// c lies 8/15 of the way from the group's smallest value to its largest, s is the smallest
// step that reaches both ends from the rounded c:
//   c = bf16(7/15 min + 8/15 max),  s = bf16(max((max - c) / 7, (c - min) / 8)),
//   n = clamp(rint((x - c) (1 / s) + 8), 0, 15).
// A step below 2^-126 is taken as 0 (then x = c); a NaN or an infinity anywhere in a group
// makes s and c NaN, so the group reads NaN. Where the roundings of s and c put an end of a group past
// bf16's largest value, a read returns that value. 8 is chosen, rather than the middle 7.5, because
// bf16 holds 128 + n and 136 exactly: a matrix instruction takes the codes as 128 + n, one
// bit operation per pair, and the offset leaves with the constant 136.
//
// 32 consecutive keys of a (sequence, KV head) pair are one block of 32 D + 256 NG bytes,
// so a pass over the cache is one stream:
//   K codes  key k, lane group kg = 0..3, MFMA step i: the dword at k D/2 + kg D/8 + 4 i holds
//            the values 32 i + 8 kg + e, e = 0..7, value e in the 4 bits from 4 (e/2) + 16 (e%2):
//            a lane's load of D/8 bytes is its part of every 16x16x32 operand, and the same
//            shift of a dword gives the bf16 pair (e, e + 1);
//   V codes  16 D bytes on: for keys 8 q .. 8 q + 7 (q = 0..3), plane h = 0..D/64-1 and n = 0..15
//            the 16 bytes at ((q D/64 + h) 16 + n) 16 hold, key pair p in dword p, the key 8 q +
//            2 p in the low half and the next in the high one, the columns 32 (j/2) + 2 n + j%2
//            for j = 4 h + jj in the 4 bits from 4 jj: the pairs that the contraction over
//            keys takes lie side by side, and appending a key writes whole bytes;
//   scales   32 D bytes on: for K, then for V, for each group 32 dwords, s low and c high.
#pragma once

#include "ko_common.h"

namespace ko {

constexpr int KV4_KEYS = 32;  // keys of a block

__host__ __device__ constexpr int kv4_block_bytes(int d, int ng) { return 32 * d + 256 * ng; }

// The head sizes and groups served: d = 64 or 128, groups of 32, 64 or 128 values.
inline bool kv4_served(int d, int group) {
  return (d == 64 || d == 128) && (group == 32 || group == 64 || group == 128) && group <= d;
}

// Quantiser of a group whose smallest and largest values are mn and mx (NaN if any value
// is). No contraction: every step rounds by itself, as torch's float32 operations do.
struct Kv4Group {
  uint32_t sc;  // s | c << 16
  float c, inv;

  __device__ __forceinline__ void from(float mn, float mx) {
#pragma clang fp contract(off)
    c = round_bf16(mn * (float)(7.0 / 15.0) + mx * (float)(8.0 / 15.0));
    // eighths before their difference: c - mn is up to 8/15 2^129 and may pass fp32's range, mx - c
    // at 7/15 2^129 does not; the eighths are exact
    float s = round_bf16(fmaxf((mx - c) * (float)(1.0 / 7.0), c * 0.125f - mn * 0.125f));
    if (!(fabsf(mn) < INFINITY && fabsf(mx) < INFINITY)) c = s = __uint_as_float(0x7fc00000u);
    if (s < 1.1754943508222875e-38f) s = 0.f;
    // 1 / s, rounded correctly: with y = (1 + e) / s from v_rcp_f32, |e| < 2^-22, the inner fma is exact
    // and the outer one rounds (1 - e^2) / s, 2^-44 off; but 1 / s of an 8-bit significand m lies
    // at least 2^-32 of itself from any border between two floats (|2^32 - j m| >= 1 for its
    // denominator m 2^32), a power of two on a float. s, about 1/15 of a span below 2^129, is below 2^126,
    // so y is normal.
    const float y = __builtin_amdgcn_rcpf(s);
    inv = s == 0.f ? 0.f : fmaf(fmaf(-s, y, 1.0f), y, y);
    sc = (__float_as_uint(s) >> 16) | (__float_as_uint(c) & 0xffff0000u);
  }
  // The code in the low 4 bits, zeros up to bit 21: 1.5 2^23 + t is rounded to a whole number. What
  // lies above is shifted out of the way of codes that are put together at bits below 16.
  __device__ __forceinline__ uint32_t raw(float x) const {
#pragma clang fp contract(off)
    const float t = __builtin_amdgcn_fmed3f((x - c) * inv + 8.0f, 0.f, 15.f);
    return __float_as_uint(t + 12582912.0f);
  }
  __device__ __forceinline__ uint32_t code(float x) const { return raw(x) & 15u; }
};

// NaN-propagating minimum and maximum (gfx950's v_minimum3 / v_maximum3).
__device__ __forceinline__ float kv4_min(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float kv4_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float kv4_min_row16(float v) {
  v = kv4_min(v, dpp_f<0x128>(v));
  v = kv4_min(v, dpp_f<0x124>(v));
  v = kv4_min(v, dpp_f<0x122>(v));
  return kv4_min(v, dpp_f<0x121>(v));
}
__device__ __forceinline__ float kv4_max_row16(float v) {
  v = kv4_max(v, dpp_f<0x128>(v));
  v = kv4_max(v, dpp_f<0x124>(v));
  v = kv4_max(v, dpp_f<0x122>(v));
  return kv4_max(v, dpp_f<0x121>(v));
}
// With the lanes 16 and 32 places away (ko_common.h, sum_xor16).
__device__ __forceinline__ void kv4_minmax_xor16(float& mn, float& mx) {
  const unsigned a = __float_as_uint(mn), b = __float_as_uint(mx);
  const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const auto q = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  mn = kv4_min(__uint_as_float((unsigned)p[0]), __uint_as_float((unsigned)p[1]));
  mx = kv4_max(__uint_as_float((unsigned)q[0]), __uint_as_float((unsigned)q[1]));
}
__device__ __forceinline__ void kv4_minmax_xor32(float& mn, float& mx) {
  const unsigned a = __float_as_uint(mn), b = __float_as_uint(mx);
  const auto p = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  mn = kv4_min(__uint_as_float((unsigned)p[0]), __uint_as_float((unsigned)p[1]));
  mx = kv4_max(__uint_as_float((unsigned)q[0]), __uint_as_float((unsigned)q[1]));
}

}  // namespace ko

// CALL(d, groups a head) for the served sizes (kv4_served).
#define KV4_PICK(D_, GROUP_, CALL)                  \
  if ((D_) == 128) {                                \
    if ((GROUP_) == 32) {                           \
      CALL(128, 4)                                  \
    } else if ((GROUP_) == 64) {                    \
      CALL(128, 2)                                  \
    } else {                                        \
      CALL(128, 1)                                  \
    }                                               \
  } else if ((GROUP_) == 32) {                      \
    CALL(64, 2)                                     \
  } else {                                          \
    CALL(64, 1)                                     \
  }
