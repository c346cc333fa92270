// y = x W^T with W in 8 bits for up to 16 rows of x: one weight pass at memory speed.
//
// The 16 rows are one tile of the matrix instruction. A workgroup's wavefronts share K: each holds
// its few blocks of x as bf16 in registers for the whole launch and streams the same blocks of one
// tile of W after another, two tiles' loads in flight at any time; a tile's partial sums meet in
// LDS, and one wavefront in turn adds and stores them (SWIGLU: a gate tile's and, in the next
// step, its up tile's). The codes go through bf16 to the matrix instruction (sums in fp32 throughout): 16
// conversions and 4 instructions of 16 cycles a block of 2 KB, a quarter of the time in which it comes from memory.
//
// bf16 rows are quantised by every workgroup itself, in the registers in which they are multiplied
// (layout of fp8_core.h), under the first weight loads: a launch less than quantising them first.
#include "fp8_linear.h"

namespace {

using namespace ko;

constexpr int GRID = 256;   // persistent workgroups, one a CU

template <int N>
struct Weights {   // N blocks of a tile
  uint4 c[N][2];
  uint32_t s[N];
};

// x's values 64 j + 16 g + 8 p .. + 7 of a block, packed bf16.
struct Raw {
  uint4 q[2][2];
  __device__ __forceinline__ void load(const uint16_t* row, int k, int K, bool ok) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int at = k + 64 * j + 8 * p;
        q[j][p] = ok && at < K ? ldg16(row + at) : make_uint4(0, 0, 0, 0);
      }
  }
  // bf16(gain * bf16(x * rstd)); gain: the block's, from 16 g on
  __device__ __forceinline__ void norm(const uint4* gain, float rstd) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint4 w = gain[8 * j + p];
        uint4& v = q[j][p];
        v = make_uint4(norm2(v.x, w.x, rstd), norm2(v.y, w.y, rstd), norm2(v.z, w.z, rstd),
                       norm2(v.w, w.w, rstd));
      }
  }
  static __device__ __forceinline__ uint32_t norm2(uint32_t x, uint32_t w, float rstd) {
    const uint32_t t = pack_bf16x2(bf16lo(x) * rstd, bf16hi(x) * rstd);
    return pack_bf16x2(bf16lo(w) * bf16lo(t), bf16hi(w) * bf16hi(t));
  }
  __device__ __forceinline__ void unpack(float (&v)[2][16]) const {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t w[4] = {q[j][p].x, q[j][p].y, q[j][p].z, q[j][p].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[j][8 * p + 2 * i] = bf16lo(w[i]);
          v[j][8 * p + 2 * i + 1] = bf16hi(w[i]);
        }
      }
  }
};

__device__ __forceinline__ void widen(const uint4 (&c)[2], uint32_t b, bf16x8 (&out)[4]) {
  const float s = __uint_as_float(b << 23);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    out[2 * j] = fp8_to_bf16(c[j].x, c[j].y, s);
    out[2 * j + 1] = fp8_to_bf16(c[j].z, c[j].w, s);
  }
}

// IN: 0 codes, 1 bf16, 2 bf16 behind a norm. BPW blocks a wavefront, at most WMAX wavefronts.
template <int EPI, int IN, int BPW, int WMAX>
__global__ __launch_bounds__(64 * WMAX) void few_kernel(LinearArgs a, int units) {
  constexpr int NT = EPI == EPI_SWIGLU ? 2 : 1;   // tiles of a unit
  __shared__ f32x4 s_part[2][WMAX][64];
  __shared__ float s_sq[IN == 2 ? WMAX * BPW : 1][16];
  __shared__ uint4 s_gain[IN == 2 ? WMAX * BPW * 16 : 1];
  const int W = blockDim.x >> 6;
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int KB = fp8_blocks(a.K), Q = fp8_quads(a.K);
  const int kb0 = wv * BPW;   // < KB

  // this workgroup's steps: tiles NT u .. of its units u
  const int steps = NT * ((units - 1 - (int)blockIdx.x) / GRID + 1);
  auto tile_of = [&](int st) { return (long long)(blockIdx.x + st / NT * GRID) * NT + st % NT; };
  const uint8_t* wl = a.wc + 16 * lane;
  auto load = [&](int st, Weights<BPW>& w) {
    if (st >= steps) return;
    const long long tile = tile_of(st);
    const uint8_t* c = wl + (tile * KB + kb0) * FP8_BLOCK;
    const uint32_t* sc = a.ws + tile * Q * 16 + r;
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      const int kb = min(i, KB - 1 - kb0);   // a block past the end: the last, not multiplied
#pragma unroll
      for (int j = 0; j < 2; ++j) w.c[i][j] = ldg16_stream(c + kb * FP8_BLOCK + 1024 * j);
      // BPW of 2 and 4: one dword has them all
      if (i == 0 || (BPW != 2 && BPW != 4)) w.s[i] = sc[((kb0 + kb) >> 2) * 16];
      else w.s[i] = w.s[0];
    }
  };

  bf16x8 x[BPW][4];
  Weights<BPW> wa, wb;
  auto load2 = [&]() {   // two tiles' loads under what follows
    load(0, wa);
    load(1, wb);
  };
  if constexpr (IN == 0) {
    uint4 c[BPW][2];
    uint32_t sx[BPW];
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      const int kb = min(kb0 + i, KB - 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) c[i][j] = ldg16(a.xc + kb * FP8_BLOCK + 1024 * j + 16 * lane);
      sx[i] = (a.xs[(kb >> 2) * 16 + r] >> (8 * (kb & 3))) & 255u;
    }
    load2();
#pragma unroll
    for (int i = 0; i < BPW; ++i) widen(c[i], sx[i], x[i]);
  } else {
    Raw raw[BPW];
    const uint16_t* row = a.x + (long long)(r < a.M ? r : 0) * a.K;
#pragma unroll
    for (int i = 0; i < BPW; ++i) raw[i].load(row, (kb0 + i) * 128 + 16 * g, a.K, r < a.M);
    constexpr int GL = (BPW * 16 + 63) / 64;   // a thread's loads of the gain
    uint4 gain[GL];
    if constexpr (IN == 2) {
#pragma unroll
      for (int i = 0; i < GL; ++i) {
        const int at = threadIdx.x + i * blockDim.x;
        gain[i] = 8 * at < a.K ? ldg16(a.nw + 8 * at) : make_uint4(0, 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);   // x ahead of the weights
    load2();
    __builtin_amdgcn_sched_barrier(0);
    float rstd = 0.f;
    if constexpr (IN == 2) {
#pragma unroll
      for (int i = 0; i < GL; ++i) {
        const int at = threadIdx.x + i * blockDim.x;
        if (at < WMAX * BPW * 16) s_gain[at] = gain[i];
      }
#pragma unroll
      for (int i = 0; i < BPW; ++i) {
        float v[2][16];
        raw[i].unpack(v);
        const float sq = fp8_square_sum(v);
        if (g == 0) s_sq[kb0 + i][r] = sq;
      }
      __syncthreads();
      float tot = 0.f;
      for (int kb = 0; kb < KB; ++kb) tot += s_sq[kb][r];
      rstd = r < a.M ? rsqrtf(tot / (float)a.K + a.eps) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      if constexpr (IN == 2) {
        if (r < a.M) raw[i].norm(s_gain + (kb0 + i) * 16 + 2 * g, rstd);
      }
      float v[2][16];
      raw[i].unpack(v);
      uint4 c[2];
      const uint32_t b = fp8_quantize_block(v, c);
      widen(c, b, x[i]);
    }
  }

  f32x4 gate = {0.f, 0.f, 0.f, 0.f};   // SWIGLU: the sums of the step before
  auto step = [&](int st, Weights<BPW>& w) {
    const bool mine = wv == st / NT % W;   // this wavefront adds the tile's sums
    const int n = (int)(blockIdx.x + st / NT * GRID) * 16 + 4 * g;
    uint2 hv = make_uint2(0, 0);
    if constexpr (EPI == EPI_RESID)
      if (mine) hv = load4(a, r, n);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      if (kb0 + i >= KB) break;
      bf16x8 f[4];
      widen(w.c[i], (w.s[i] >> (8 * ((kb0 + i) & 3))) & 255u, f);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[j], x[i][j], acc, 0, 0, 0);
    }
    s_part[st & 1][wv][lane] = acc;
    load(st + 2, w);
    __syncthreads();   // of the next step but one: every wavefront is past this step's sums
    if (mine) {
      f32x4 sum = s_part[st & 1][0][lane];
      for (int i = 1; i < W; ++i) sum += s_part[st & 1][i][lane];
      if (NT == 1 || st % NT) store4<EPI>(a, r, n, NT == 1 ? sum : gate, sum, hv);
      gate = sum;
    }
  };
  for (int st = 0; st < steps; st += 2) {
    step(st, wa);
    if (st + 1 < steps) step(st + 1, wb);
  }
}

// Longer rows: a workgroup takes one tile (pair), its wavefronts a run of blocks each, x loaded and
// quantised along the way. A group's GB blocks of W are all on their way at once (K = 9728: 16
// wavefronts x 5 blocks of 2 KB, the whole run), x two blocks ahead.
template <int EPI, int IN>
__global__ __launch_bounds__(1024) void deep_kernel(LinearArgs a) {
  constexpr int NT = EPI == EPI_SWIGLU ? 2 : 1, W = 16, GB = NT == 2 ? 3 : 5, AHEAD = 2;
  __shared__ f32x4 s_part[W][NT][64];
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int KB = fp8_blocks(a.K), Q = fp8_quads(a.K);
  const int begin = KB * wv / W, end = KB * (wv + 1) / W;
  const int unit = blockIdx.x, n = unit * 16 + 4 * g;
  const long long tile0 = (long long)unit * NT;
  const uint16_t* row = a.x + (long long)(r < a.M ? r : 0) * a.K + 16 * g;
  uint2 hv = make_uint2(0, 0);
  if constexpr (EPI == EPI_RESID)
    if (wv == 0) hv = load4(a, r, n);
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = begin; k0 < end; k0 += GB) {
    Raw raw[IN ? GB : 1];
    uint4 xc[IN ? 1 : GB][2];
    uint32_t xs[IN ? 1 : GB];
    auto load_x = [&](int i) {   // past the end: the last block, not multiplied
      const int kb = min(k0 + i, end - 1);
      if constexpr (IN) {
        raw[i].load(row, kb * 128, a.K - 16 * g, r < a.M);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) xc[i][j] = ldg16(a.xc + kb * FP8_BLOCK + 1024 * j + 16 * lane);
        xs[i] = (a.xs[(kb >> 2) * 16 + r] >> (8 * (kb & 3))) & 255u;
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load_x(i);
    __builtin_amdgcn_sched_barrier(0);   // x ahead of the weights
    uint4 wc[NT][GB][2];
    uint32_t ws[NT][GB];
#pragma unroll
    for (int i = 0; i < GB; ++i) {
      const int kb = min(k0 + i, end - 1);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          wc[t][i][j] = ldg16_stream(a.wc + ((tile0 + t) * KB + kb) * FP8_BLOCK + 1024 * j + 16 * lane);
        ws[t][i] = a.ws[((tile0 + t) * Q + (kb >> 2)) * 16 + r] >> (8 * (kb & 3));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < GB; ++i) {
      bf16x8 x[4], f[4];
      if constexpr (IN) {
        float v[2][16];
        raw[i].unpack(v);
        uint4 c[2];
        const uint32_t b = fp8_quantize_block(v, c);
        widen(c, b, x);
      } else {
        widen(xc[i], xs[i], x);
      }
      if (i + AHEAD < GB) load_x(i + AHEAD);
      if (k0 + i < end) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          widen(wc[t][i], ws[t][i] & 255u, f);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[j], x[j], acc[t], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) s_part[wv][t][lane] = acc[t];
  __syncthreads();
  if (wv) return;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    acc[t] = s_part[0][t][lane];
#pragma unroll
    for (int i = 1; i < W; ++i) acc[t] += s_part[i][t][lane];
  }
  store4<EPI>(a, r, n, acc[0], acc[NT - 1], hv);
}

// Blocks of K that x takes in registers: more would spill.
constexpr int HELD = 32, HELD_NORM = 20;

template <int EPI, int IN>
int launch(const LinearArgs& a, hipStream_t s) {
  const int KB = fp8_blocks(a.K), units = EPI == EPI_SWIGLU ? a.wt / 2 : a.wt;
  const dim3 grid(units < GRID ? units : GRID);
#define KO_FEW(B, WM)                                                                          \
  hipLaunchKernelGGL((few_kernel<EPI, IN, B, WM>), grid, dim3(64 * ((KB + B - 1) / B)), 0, s, a, \
                     units)
  if (KB <= 20) {
    KO_FEW(2, 10);
  } else if constexpr (IN < 2) {
    if (KB > HELD) hipLaunchKernelGGL((deep_kernel<EPI, IN>), dim3(units), dim3(1024), 0, s, a);
    else KO_FEW(2, 16);
  }
#undef KO_FEW
  return KO_LAUNCH_STATUS();
}

template <int EPI>
int launch_in(const LinearArgs& a, hipStream_t s) {
  if (a.nw) return launch<EPI, 2>(a, s);
  return a.x ? launch<EPI, 1>(a, s) : launch<EPI, 0>(a, s);
}

}  // namespace

namespace ko {

bool few_rows_quantized(const LinearArgs& a) { return !a.nw || fp8_blocks(a.K) <= HELD_NORM; }

int launch_few_rows(const LinearArgs& a, int epi, hipStream_t s) {
  switch (epi) {
    case EPI_F32: return launch_in<EPI_F32>(a, s);
    case EPI_BF16: return launch_in<EPI_BF16>(a, s);
    case EPI_RESID: return launch_in<EPI_RESID>(a, s);
    default: return launch_in<EPI_SWIGLU>(a, s);
  }
}

}  // namespace ko
