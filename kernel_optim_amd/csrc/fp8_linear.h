// What the projections' kernels share: arguments, epilogues, the running of loads ahead of their use.
#pragma once

#include "fp8_core.h"

namespace ko {

enum { EPI_F32 = 0, EPI_BF16 = 1, EPI_RESID = 2, EPI_SWIGLU = 3 };

struct LinearArgs {
  const uint8_t *xc, *wc;     // codes
  const uint32_t *xs, *ws;    // scales
  const uint16_t *x, *nw;     // or x in bf16, and the gain of a norm in front of it
  float eps;
  void* y;
  const uint16_t* h;          // RESID: what is added; may be y
  int M, N, K;
  int xt, wt;                 // tiles of x and of W
  float* part;                // scratch: partial sums,
  int* counters;              // and counters, zero before every call and behind it
};

// RESID: columns n .. n + 3 of h's row m as packed bf16, loaded ahead of the sums they are added to.
// Rows and columns past the end read an element that is there (unused): no lane skips the load, so
// what is waited for behind it stays exact.
__device__ __forceinline__ uint2 load4(const LinearArgs& a, int m, int n) {
  const uint16_t* h = a.h + (long long)min(m, a.M - 1) * a.N;
  if ((a.N & 3) == 0) return *reinterpret_cast<const uint2*>(h + min(n, a.N - 4));
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = h[min(n + i, a.N - 1)];
  return make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
}

// The sum of W wavefronts' partial sums, part[i * stride][lane], in order, 4 reads at a time.
__device__ __forceinline__ f32x4 add_parts(const f32x4 (*part)[64], int stride, int W, int lane) {
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < W; i += 4) {
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = part[min(i + j, W - 1) * stride][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < W) sum += v[j];
  }
  return sum;
}

// Steps st = 0 .. steps - 1 with SETS steps' loads in flight: load(st, set) loads, step(st, set)
// computes and then calls its third argument, which loads the step SETS ahead into the set. In all
// groups of SETS steps but the last two no load is under a condition: behind one, a wait for
// an earlier load would have to wait for all.
template <int SETS, class Load, class Step>
__device__ __forceinline__ void pipeline(int steps, Load load, Step step) {
  int st = 0;
  for (; steps - st >= 2 * SETS; st += SETS) {
#pragma unroll
    for (int i = 0; i < SETS; ++i) step(st + i, i, [&]() { load(st + i + SETS, i); });
  }
  if (steps - st > SETS) {
#pragma unroll
    for (int i = 0; i < SETS; ++i)
      step(st + i, i, [&]() {
        if (st + i + SETS < steps) load(st + i + SETS, i);
      });
    st += SETS;
  }
#pragma unroll
  for (int i = 0; i < SETS; ++i)
    if (st + i < steps) step(st + i, i, []() {});
}

// Columns n .. n + 3 of row m; v2: the second half's sums (SWIGLU); hv: load4 (RESID). The roundings
// are those of the bf16 chain: the product, silu(gate) and their product, or the product and the
// sum with h, each to bf16.
template <int EPI>
__device__ __forceinline__ void store4(const LinearArgs& a, int m, int n, f32x4 v, f32x4 v2, uint2 hv) {
  if (m >= a.M || n >= a.N) return;
  const long long o = (long long)m * a.N + n;
  const bool whole = (a.N & 3) == 0;   // n is a multiple of 4: so is every row's beginning
  if constexpr (EPI == EPI_F32) {
    float* y = static_cast<float*>(a.y) + o;
    if (whole) *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
    else
      for (int i = 0; i < 4 && n + i < a.N; ++i) y[i] = v[i];
    return;
  }
  uint16_t* y = static_cast<uint16_t*>(a.y) + o;
  float r[4];
  const float h[4] = {bf16lo(hv.x), bf16hi(hv.x), bf16lo(hv.y), bf16hi(hv.y)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = v[i];
    if constexpr (EPI == EPI_RESID) r[i] = h[i] + round_bf16(v[i]);
    if constexpr (EPI == EPI_SWIGLU) {
      const float g = round_bf16(v[i]), u = round_bf16(v2[i]);
      r[i] = round_bf16(g / (1.0f + expf(-g))) * u;
    }
  }
  if (whole) *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3]));
  else
    for (int i = 0; i < 4 && n + i < a.N; ++i) y[i] = f32_to_bf16(r[i]);
}

// fp8_few.hip: up to 16 rows of x (codes, or bf16 with or without a norm).
bool few_rows_served(const LinearArgs& a);
bool few_rows_quantized(const LinearArgs& a);   // whether it takes this x in bf16
int launch_few_rows(const LinearArgs& a, int epi, hipStream_t s);

// fp8_mid.hip: up to 64 rows of x in codes.
bool mid_rows_served(const LinearArgs& a, int epi);
long long mid_rows_scratch(const LinearArgs& a);   // bytes
int launch_mid_rows(const LinearArgs& a, int epi, hipStream_t s);

}  // namespace ko
