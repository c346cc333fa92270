// y[M, N] = x W^T with both factors held in 8-bit floating point (layout: fp8_core.h).
//
// Tiled product: a workgroup stages the blocks of its x and W tiles for one step of 128 values in
// LDS by direct loads and multiplies the step before. W is the matrix instruction's first factor, so
// that a lane ends with 4 neighbouring columns of a row of y.
// 8192 rows of gate/up (19,456 x 2560) with the SwiGLU: 406 to 437 us by the box, 1.9 to 2.0 PFLOP/s (a
// plain library product of that size 378). The matrix cores are busy in 41 % of the cycles; a step's
// 192 KB read from LDS and 64 KB written take another 41 % at 128 bytes a clock, with no bank
// conflicts: the two go nearly one after the other, with a full wait between steps. 511 rows
// of qkv (6144 x 2560): 15.6 us, 20 steps that wait for one another.
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

__device__ __forceinline__ void widen(i32x8 c, uint32_t b, bf16x8 (&out)[4]) {
  const float s = __uint_as_float((b & 255u) << 23);
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = fp8_to_bf16((uint32_t)c[2 * i], (uint32_t)c[2 * i + 1], s);
}

// acc += the 16 x 16 products of a block of W and TM of x; byte I of the dwords are their scales.
// WIDE: through bf16 (fp8_core.h).
template <int I, bool WIDE, int TM>
__device__ __forceinline__ void multiply(i32x8 w, uint32_t sw, const i32x8 (&x)[TM],
                                         const uint32_t (&sx)[TM], f32x4 (&acc)[TM]) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int j = 0; j < TM; ++j)
      acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x[j], acc[j], 0, 0, I, (int)sw, I,
                                                                (int)sx[j]);
  } else {
    bf16x8 f[4], v[4];
    widen(w, sw >> (8 * I), f);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      widen(x[j], sx[j] >> (8 * I), v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[e], v[e], acc[j], 0, 0, 0);
    }
  }
}

// Waits until all but the N youngest loads of this wavefront (and its LDS reads) are done, then for
// the workgroup.
template <int N>
__device__ __forceinline__ void wait_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// WN x WM wavefronts of TN x TM tiles each; STAGES buffers of a step's blocks. With two, a step's loads
// have the products of the step before to arrive in, and the compiler may mix their issue with those;
// with more (small tiles, whose steps are shorter than a load) the waits are counted.
template <int EPI, bool WIDE, int WN, int WM, int TN, int TM, int STAGES>
__global__ __launch_bounds__(64 * WN * WM) void gemm_kernel(LinearArgs a, int nblocks) {
  constexpr int W = WN * WM, NT = WN * TN, MT = WM * TM, CH = 2 * (NT + MT) / W;
  static_assert(CH * W == 2 * (NT + MT), "every wavefront loads as much");
  static_assert(EPI != EPI_SWIGLU || TN % 2 == 0, "a wavefront's tiles in twos");
  __shared__ __attribute__((aligned(16))) uint8_t s_buf[STAGES][(NT + MT) * FP8_BLOCK];
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int wn = wv % WN, wm = wv / WN;
  const int KB = fp8_blocks(a.K), Q = fp8_quads(a.K);
  const int nb = blockIdx.x % nblocks, mb = blockIdx.x / nblocks;
  const int n0 = nb * NT, m0 = mb * MT;   // this workgroup's first tiles

  // Addresses are uniform but for the lane's place in a block. Tiles past the end: the last one,
  // their results unused.
  const uint8_t* src[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = wv * CH + i, t = c >> 1;
    const long long tile = t < NT ? min(n0 + t, a.wt - 1) : min(m0 + t - NT, a.xt - 1);
    src[i] = (t < NT ? a.wc : a.xc) + tile * KB * FP8_BLOCK + (c & 1) * 1024;
  }
  auto stage = [&](int kb, int buf) {   // past the end: the last step again, unused
    const int at = min(kb, KB - 1) * FP8_BLOCK;
#pragma unroll
    for (int i = 0; i < CH; ++i) load_lds(src[i] + at + 16 * lane, s_buf[buf] + (wv * CH + i) * 1024);
  };
  uint32_t sw[TN], sx[TM], next_w[TN], next_x[TM];   // a quad's scales, and the next one's
  auto load_scales = [&](int q) {
    q = min(q, Q - 1);   // past the end: unused
#pragma unroll
    for (int i = 0; i < TN; ++i)
      next_w[i] = (a.ws + ((long long)min(n0 + wn * TN + i, a.wt - 1) * Q + q) * 16)[r];
#pragma unroll
    for (int i = 0; i < TM; ++i)
      next_x[i] = (a.xs + ((long long)min(m0 + wm * TM + i, a.xt - 1) * Q + q) * 16)[r];
  };

  f32x4 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  if constexpr (STAGES > 2) load_scales(0);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) stage(i, i);
  int buf = 0;   // of the step
  for (int q = 0; q < Q; ++q) {
    if constexpr (STAGES == 2) load_scales(q);
#pragma unroll
    for (int i = 0; i < TN; ++i) sw[i] = next_w[i];
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[i] = next_x[i];
#define KO_STEP(I)                                                                       \
  if (4 * q + I < KB) {                                                                  \
    const int kb = 4 * q + I;                                                            \
    /* this step's blocks are there, and the last step's buffer is read out */           \
    if constexpr (STAGES == 2) {                                                         \
      __syncthreads();                                                                   \
      if (kb + 1 < KB) stage(kb + 1, (I + 1) & 1);                                       \
    } else {                                                                             \
      wait_barrier<CH * (STAGES - 2)>();                                                 \
      stage(kb + STAGES - 1, buf == 0 ? STAGES - 1 : buf - 1);                           \
      if constexpr (I == 0) load_scales(q + 1);                                          \
      __builtin_amdgcn_sched_barrier(0);                                                 \
    }                                                                                    \
    const uint8_t* sb = s_buf[STAGES == 2 ? I & 1 : buf];                                \
    i32x8 w[TN], x[TM];                                                                  \
    _Pragma("unroll") for (int j = 0; j < TM; ++j)                                       \
        x[j] = frag(sb + (NT + wm * TM + j) * FP8_BLOCK, lane);                          \
    _Pragma("unroll") for (int i = 0; i < TN; ++i)                                       \
        w[i] = frag(sb + (wn * TN + i) * FP8_BLOCK, lane);                               \
    _Pragma("unroll") for (int i = 0; i < TN; ++i)                                       \
        multiply<I, WIDE, TM>(w[i], sw[i], x, sx, acc[i]);                               \
    buf = buf == STAGES - 1 ? 0 : buf + 1;                                               \
  }
    KO_STEP(0)
    KO_STEP(1)
    KO_STEP(2)
    KO_STEP(3)
#undef KO_STEP
  }
  // no load into LDS outlives the workgroup: past the end there are some that nothing waited for
  if constexpr (STAGES > 2) __builtin_amdgcn_s_waitcnt(15 << 8 | 7 << 4);
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

template <int EPI, bool WIDE, int WN, int WM, int TN, int TM, int STAGES>
int launch_tiled(const LinearArgs& a, hipStream_t s) {
  constexpr int NT = WN * TN, MT = WM * TM;
  const int nb = (a.wt + NT - 1) / NT, mb = (a.xt + MT - 1) / MT;
  if (!fp8_launchable((long long)nb * mb, 64 * WN * WM)) return KO_ERANGE;
  hipLaunchKernelGGL((gemm_kernel<EPI, WIDE, WN, WM, TN, TM, STAGES>), dim3(nb * mb),
                     dim3(64 * WN * WM), 0, s, a, nb);
  return KO_LAUNCH_STATUS();
}

// Workgroups of tiles of 16 t x 16 t columns and rows.
long long groups(const LinearArgs& a, int t) {
  return ((a.wt + t - 1ll) / t) * ((a.xt + t - 1ll) / t);
}

// The tile by what its rounds of workgroups take, in us of K = 2560 (a round of 256, 512 and 768
// workgroups: one, two and three a CU):
//   256 x 256: 40 a round                        (8192 x 6144: 120 us against 135, 128 x 128)
//   128 x 128: 18 up to 256 workgroups, then 22.5 a round       (2048 x 19456: 114 against 123)
//   64 x 64:   10.4 up to 256, 11.7 up to 512, then 15.5 a round    (128 x 6144: 10.5 against 18)
// and through bf16, where rounds follow one another with less of a gap:
//   128 x 128: 26 up to 256 workgroups, 40 up to 409, then 40 for each 512    (1024 x 19456: 102 against 133)
//   64 x 64:   12.5, 17.7 and 24 up to 256, 512 and 712, then 20.5 for each 768   (128 x 6144: 13 against 25)
template <int EPI>
int launch(const LinearArgs& a, hipStream_t s) {
  const long long n8 = groups(a, 8), n4 = groups(a, 4);
  if constexpr (EPI == EPI_F32) {
    const double t8 = n8 <= 256 ? 26.0 : fmax(40.0, 8.0 + 40.0 / 512 * n8);
    const double t4 = n4 <= 256 ? 12.5 : n4 <= 512 ? 17.7 : fmax(24.0, 5.0 + 20.5 / 768 * n4);
    if (t4 < t8) return launch_tiled<EPI, true, 2, 2, 2, 2, 3>(a, s);
    return launch_tiled<EPI, true, 2, 2, 4, 4, 2>(a, s);
  } else {
    const long long n16 = groups(a, 16);
    const double t16 = 40.0 * ((n16 + 255) / 256);
    const double t8 = n8 <= 256 ? 18.0 : 22.5 * ((n8 + 511) / 512);
    const double t4 = n4 <= 256 ? 10.4 : n4 <= 512 ? 11.7 : 15.5 * ((n4 + 767) / 768);
    if (t4 < t8 && t4 < t16) return launch_tiled<EPI, false, 2, 2, 2, 2, 3>(a, s);
    if (t8 <= t16) return launch_tiled<EPI, false, 2, 2, 4, 4, 2>(a, s);
    return launch_tiled<EPI, false, 4, 2, 4, 8, 2>(a, s);
  }
}

}  // namespace

static void set_sizes(LinearArgs& a, int M, int N, int K, int epi) {
  a.M = M, a.N = N, a.K = K;
  a.xt = (int)fp8_tiles(M, false);
  a.wt = (int)(epi == EPI_SWIGLU ? fp8_tiles(2 * N, true) : fp8_tiles(N, false));
}

extern "C" {

long long ko_fp8_linear_scratch(int M, int N, int K, int epi) {
  if (M < 1 || N < 1 || N > 0x3fffffff || K < 8 || K > FP8_K_MAX || (K & 7)) return -1;
  if (epi < EPI_F32 || epi > EPI_SWIGLU) return -1;
  LinearArgs a;
  set_sizes(a, M, N, K, epi);
  return !few_rows_served(a) && mid_rows_served(a, epi) ? mid_rows_scratch(a) : 0;
}

int ko_fp8_quantize(const void* x, int x_f32, long long stride, int rows, int K, int pair,
                    const void* nw, float eps, void* codes, void* scales, void* stream);

int ko_fp8_linear(const void* x, const void* nw, float eps, void* xc, void* xs, const void* wc,
                  const void* ws, void* y, const void* h, void* scratch, long long scratch_bytes,
                  int M, int N, int K, int epi, void* stream) {
  if (!xc || !xs || !wc || !ws || !y || M < 1 || N < 1 || K < 8 || (K & 7)) return KO_EINVAL;
  if (epi < EPI_F32 || epi > EPI_SWIGLU) return KO_ENOTSUP;
  if ((epi == EPI_RESID && !h) || (nw && !x)) return KO_EINVAL;
  const uintptr_t all = (uintptr_t)xc | (uintptr_t)xs | (uintptr_t)wc | (uintptr_t)ws | (uintptr_t)y |
                        (uintptr_t)x | (uintptr_t)nw;
  if ((all | (uintptr_t)h | (uintptr_t)scratch) & 15) return KO_EINVAL;
  if (N > 0x3fffffff || K > FP8_K_MAX) return KO_ERANGE;
  const long long need = ko_fp8_linear_scratch(M, N, K, epi);
  if (need && (!scratch || scratch_bytes < need)) return KO_EINVAL;
  LinearArgs a;
  a.counters = static_cast<int*>(scratch);
  a.part = static_cast<float*>(scratch) + 1024;
  a.x = static_cast<const uint16_t*>(x);
  a.nw = static_cast<const uint16_t*>(nw);
  a.eps = eps;
  a.xc = static_cast<const uint8_t*>(xc);
  a.wc = static_cast<const uint8_t*>(wc);
  a.xs = static_cast<const uint32_t*>(xs);
  a.ws = static_cast<const uint32_t*>(ws);
  a.y = y;
  a.h = static_cast<const uint16_t*>(h);
  set_sizes(a, M, N, K, epi);
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
