// y[M, N] = x W^T with both factors held in 8-bit floating point (layout: fp8_core.h).
//
// Tiled product: a workgroup stages the blocks of its x and W tiles for one step of 128 values in
// LDS by direct loads and multiplies the step before. W is the matrix instruction's first factor, so
// that a lane ends with 4 neighbouring columns of a row of y.
#include "fp8_linear.h"

namespace {

using namespace ko;

typedef __attribute__((address_space(1))) const void g_void;
typedef __attribute__((address_space(3))) void l_void;

// 1 KB from src + 16 * lane to dst + 16 * lane in LDS.
__device__ __forceinline__ void load_lds(const uint8_t* src, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds((g_void*)src, (l_void*)dst, 16, 0, 0);
}

__device__ __forceinline__ i32x8 frag(const uint8_t* block, int lane) {
  const i32x4 lo = *reinterpret_cast<const i32x4*>(block + 16 * lane);
  const i32x4 hi = *reinterpret_cast<const i32x4*>(block + 1024 + 16 * lane);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int I>
__device__ __forceinline__ f32x4 mfma(i32x8 a, i32x8 b, f32x4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, I, (int)sa, I, (int)sb);
}

// acc += the 16 x 16 products of a block of W and one of x; byte I of sw and sx are their scales.
// WIDE: through bf16 (fp8_core.h).
template <int I, bool WIDE>
struct Frag;
template <int I>
struct Frag<I, false> {
  i32x8 v;
  uint32_t s;
  __device__ __forceinline__ void load(const uint8_t* block, int lane, uint32_t scales) {
    v = frag(block, lane);
    s = scales;
  }
};
template <int I>
struct Frag<I, true> {
  bf16x8 v[4];
  __device__ __forceinline__ void load(const uint8_t* block, int lane, uint32_t scales) {
    const i32x8 c = frag(block, lane);
    const float sc = __uint_as_float(((scales >> (8 * I)) & 255u) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fp8_to_bf16((uint32_t)c[2 * i], (uint32_t)c[2 * i + 1], sc);
  }
};
template <int I>
__device__ __forceinline__ f32x4 multiply(const Frag<I, false>& w, const Frag<I, false>& x, f32x4 c) {
  return mfma<I>(w.v, x.v, c, w.s, x.s);
}
template <int I>
__device__ __forceinline__ f32x4 multiply(const Frag<I, true>& w, const Frag<I, true>& x, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], c, 0, 0, 0);
  return c;
}

template <int EPI, bool WIDE, int WN, int WM, int TN, int TM>
__global__ __launch_bounds__(64 * WN * WM) void gemm_kernel(LinearArgs a, int nblocks) {
  constexpr int W = WN * WM, NT = WN * TN, MT = WM * TM, CH = 2 * (NT + MT) / W;
  static_assert(CH * W == 2 * (NT + MT), "every wavefront loads as much");
  static_assert(EPI != EPI_SWIGLU || TN % 2 == 0, "a wavefront's tiles in twos");
  __shared__ __attribute__((aligned(16))) uint8_t s_buf[2][(NT + MT) * FP8_BLOCK];
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int wn = wv % WN, wm = wv / WN;
  const int KB = fp8_blocks(a.K), Q = fp8_quads(a.K);
  const int nb = blockIdx.x % nblocks, mb = blockIdx.x / nblocks;
  const int n0 = nb * NT, m0 = mb * MT;   // this workgroup's first tiles

  // tiles past the end: the last one, their results unused
  const uint8_t* src[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = wv * CH + i, t = c >> 1;
    const long long tile = t < NT ? min(n0 + t, a.wt - 1) : min(m0 + t - NT, a.xt - 1);
    src[i] = (t < NT ? a.wc : a.xc) + tile * KB * FP8_BLOCK + (c & 1) * 1024 + 16 * lane;
  }
  auto stage = [&](int kb, int buf) {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      load_lds(src[i] + (long long)kb * FP8_BLOCK, s_buf[buf] + (wv * CH + i) * 1024);
  };
  const uint32_t *ws[TN], *xs[TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
    ws[i] = a.ws + (long long)min(n0 + wn * TN + i, a.wt - 1) * Q * 16 + r;
#pragma unroll
  for (int i = 0; i < TM; ++i)
    xs[i] = a.xs + (long long)min(m0 + wm * TM + i, a.xt - 1) * Q * 16 + r;

  f32x4 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  stage(0, 0);
  for (int q = 0; q < Q; ++q) {
    uint32_t sw[TN], sx[TM];
#pragma unroll
    for (int i = 0; i < TN; ++i) sw[i] = ws[i][q * 16];
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[i] = xs[i][q * 16];
#define KO_STEP(I)                                                                       \
  if (4 * q + I < KB) {                                                                  \
    const int kb = 4 * q + I;                                                            \
    __syncthreads(); /* this step's blocks are there, the other buffer is read out */    \
    if (kb + 1 < KB) stage(kb + 1, (I + 1) & 1);                                         \
    const uint8_t* sb = s_buf[I & 1];                                                    \
    Frag<I, WIDE> fw[TN], fx[TM];                                                        \
    _Pragma("unroll") for (int j = 0; j < TM; ++j)                                       \
        fx[j].load(sb + (NT + wm * TM + j) * FP8_BLOCK, lane, sx[j]);                    \
    _Pragma("unroll") for (int i = 0; i < TN; ++i)                                       \
        fw[i].load(sb + (wn * TN + i) * FP8_BLOCK, lane, sw[i]);                         \
    _Pragma("unroll") for (int i = 0; i < TN; ++i)                                       \
        _Pragma("unroll") for (int j = 0; j < TM; ++j)                                   \
            acc[i][j] = multiply(fw[i], fx[j], acc[i][j]);                               \
  }
    KO_STEP(0)
    KO_STEP(1)
    KO_STEP(2)
    KO_STEP(3)
#undef KO_STEP
  }
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int m = (m0 + wm * TM + j) * 16 + r;
    if constexpr (EPI == EPI_SWIGLU) {
      // two tiles' gate sums in one register, their up sums in the other
#pragma unroll
      for (int i = 0; i < TN; i += 2) {
        f32x4 gate, up;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][j][e]),
                                                          __float_as_uint(acc[i + 1][j][e]), false, false);
          gate[e] = __uint_as_float(p[0]);
          up[e] = __uint_as_float(p[1]);
        }
        store4<EPI>(a, m, (n0 + wn * TN + i + (g >> 1)) * 8 + 4 * (g & 1), gate, up, make_uint2(0, 0));
      }
    } else {
      uint2 hv[TN] = {};
      if constexpr (EPI == EPI_RESID) {
#pragma unroll
        for (int i = 0; i < TN; ++i) hv[i] = load4(a, m, (n0 + wn * TN + i) * 16 + 4 * g);
      }
#pragma unroll
      for (int i = 0; i < TN; ++i)
        store4<EPI>(a, m, (n0 + wn * TN + i) * 16 + 4 * g, acc[i][j], acc[i][j], hv[i]);
    }
  }
}

template <int EPI>
int launch(const LinearArgs& a, hipStream_t s) {
  const int nb = (a.wt + 7) / 8, mb = (a.xt + 7) / 8;
  if ((long long)nb * mb > 0x7fffffffll) return KO_ERANGE;
  hipLaunchKernelGGL((gemm_kernel<EPI, EPI == EPI_F32, 2, 2, 4, 4>), dim3(nb * mb), dim3(256), 0, s,
                     a, nb);
  return KO_LAUNCH_STATUS();
}

}  // namespace

extern "C" {

int ko_fp8_quantize(const void* x, int x_f32, long long stride, int rows, int K, int pair,
                    const void* nw, float eps, void* codes, void* scales, void* stream);

int ko_fp8_linear(const void* x, const void* nw, float eps, void* xc, void* xs, const void* wc,
                  const void* ws, void* y, const void* h, int M, int N, int K, int epi,
                  void* stream) {
  if (!xc || !xs || !wc || !ws || !y || M < 1 || N < 1 || K < 8 || (K & 7)) return KO_EINVAL;
  if (epi < EPI_F32 || epi > EPI_SWIGLU) return KO_ENOTSUP;
  if ((epi == EPI_RESID && !h) || (nw && !x)) return KO_EINVAL;
  const uintptr_t all = (uintptr_t)xc | (uintptr_t)xs | (uintptr_t)wc | (uintptr_t)ws | (uintptr_t)y |
                        (uintptr_t)x | (uintptr_t)nw;
  if ((all | (uintptr_t)h) & 15) return KO_EINVAL;
  if (N > 0x3fffffff) return KO_ERANGE;
  LinearArgs a;
  a.x = static_cast<const uint16_t*>(x);
  a.nw = static_cast<const uint16_t*>(nw);
  a.eps = eps;
  a.xc = static_cast<const uint8_t*>(xc);
  a.wc = static_cast<const uint8_t*>(wc);
  a.xs = static_cast<const uint32_t*>(xs);
  a.ws = static_cast<const uint32_t*>(ws);
  a.y = y;
  a.h = static_cast<const uint16_t*>(h);
  a.M = M, a.N = N, a.K = K;
  a.xt = (int)fp8_tiles(M, false);
  a.wt = (int)(epi == EPI_SWIGLU ? fp8_tiles(2 * N, true) : fp8_tiles(N, false));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool few = few_rows_served(a);
  if (x && !(few && few_rows_quantized(a))) {
    if (const int st = ko_fp8_quantize(x, 0, K, M, K, 0, nw, eps, xc, xs, stream)) return st;
    a.x = a.nw = nullptr;
  }
  if (few) return launch_few_rows(a, epi, s);
  if (mid_rows_served(a, epi)) return launch_mid_rows(a, epi, s);
  switch (epi) {
    case EPI_F32: return launch<EPI_F32>(a, s);
    case EPI_BF16: return launch<EPI_BF16>(a, s);
    case EPI_RESID: return launch<EPI_RESID>(a, s);
    default: return launch<EPI_SWIGLU>(a, s);
  }
}

}  // extern "C"
