// y = x W^T with W in 8 bits for up to 16 rows of x: one weight pass at memory speed.
//
// The 16 rows are one tile of the matrix instruction. A workgroup's wavefronts share K: each streams
// its few blocks of one tile of W after another, two or three tiles' loads in flight at any time; a tile's
// partial sums meet in LDS, and one wavefront in turn adds and stores them. The codes go through bf16
// to the matrix instruction (sums in fp32 throughout): 16 conversions and 4 instructions of 16 cycles
// a block of 2 KB, a quarter of the time in which it comes from memory.
//
// Memory bounds it: the LM head (151,936 x 2560) takes 64 us for 4 rows, 6.2 TB/s of the 6.5 that
// reads reach, gate/up (19,456 x 2560) of 16 rows 12.0, 4.2 TB/s with its beginning and end. One row
// of the attention output (2560 x 4096) takes 4.7, most of it a launch's and a load's latency.
//
// Up to 4 bf16 rows are quantised by every workgroup itself under its first weight loads, a launch
// less than quantising them first: thread by thread 8 values of a row at a time, codes and scales to
// LDS. (Each wavefront quantising the blocks it multiplies, in the lanes that hold them for the
// instruction, needs no LDS but has 15 of 16 lanes at work on nothing when there is one row: 3 us of a
// projection of 10.5.) More rows cost every workgroup more than the launch.
#include "fp8_linear.h"

namespace {

using namespace ko;

constexpr int GRID = 256;   // persistent workgroups, one a CU
constexpr int OWN = 4;      // rows that a workgroup quantises itself

template <int N>
struct Weights {   // N blocks of a tile
  uint4 c[N][2];
  uint32_t s[N];
};

__device__ __forceinline__ void widen(const uint4 (&c)[2], uint32_t b, bf16x8 (&out)[4]) {
  const float s = __uint_as_float(b << 23);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    out[2 * j] = fp8_to_bf16(c[j].x, c[j].y, s);
    out[2 * j + 1] = fp8_to_bf16(c[j].z, c[j].w, s);
  }
}

// IN: 0 codes, 1 bf16, 2 bf16 behind a norm. BPW blocks a wavefront, at most WMAX wavefronts; SETS
// tiles in flight.
template <int EPI, int IN, int BPW, int WMAX, int SETS>
__global__ __launch_bounds__(64 * WMAX) void few_kernel(LinearArgs a) {
  constexpr bool HOLD = BPW <= 2;                 // x as bf16 in registers for the whole launch
  __shared__ f32x4 s_part[2][WMAX][64];
  __shared__ float s_sq[IN == 2 ? WMAX * BPW * OWN : 1], s_rstd[OWN];
  __shared__ uint4 s_gain[IN == 2 ? WMAX * BPW * 16 : 1];
  // x: codes [KB][2][4][M][16] and scale bytes [KB][M]
  __shared__ __attribute__((aligned(16))) uint8_t s_x[IN ? WMAX * BPW * 128 * OWN : 16];
  __shared__ uint8_t s_xs[IN ? WMAX * BPW * OWN : 1];
  const int W = blockDim.x >> 6, T = blockDim.x;
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int KB = fp8_blocks(a.K), Q = fp8_quads(a.K), M = a.M;
  const int kb0 = wv * BPW;   // < KB

  // this workgroup's steps: its tiles of W
  const int steps = (a.wt - 1 - (int)blockIdx.x) / GRID + 1;
  const uint8_t* wl = a.wc + 16 * lane;
  Weights<BPW> ws[SETS];
  auto load = [&](int st, int set) {
    Weights<BPW>& w = ws[set];
    const long long tile = (int)blockIdx.x + st * GRID;
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
  auto load_first = [&]() {   // a workgroup with fewer steps: its last one again
#pragma unroll
    for (int i = 0; i < SETS; ++i) load(min(i, steps - 1), i);
  };

  // x's codes as the lane multiplies them: rows past M are zeros. Codes in memory that are not held
  // are loaded two blocks ahead.
  constexpr int AHEAD = 2;
  uint4 xc[IN ? 1 : BPW][2];
  uint32_t xs[IN ? 1 : BPW];
  auto load_x = [&](int i) {
    if constexpr (IN == 0) {
      const int kb = min(kb0 + i, KB - 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) xc[i][j] = ldg16(a.xc + kb * FP8_BLOCK + 1024 * j + 16 * lane);
      xs[i] = (a.xs[(kb >> 2) * 16 + r] >> (8 * (kb & 3))) & 255u;
    }
  };
  auto operand = [&](int i, bf16x8 (&out)[4]) {
    if constexpr (IN == 0) {
      widen(xc[i], xs[i], out);
    } else {
      const int kb = min(kb0 + i, KB - 1);
      uint4 c[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      uint32_t b = 0;
      if (r < M) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          c[j] = *reinterpret_cast<const uint4*>(s_x + (((kb * 2 + j) * 4 + g) * M + r) * 16);
        b = s_xs[kb * M + r];
      }
      widen(c, b, out);
    }
  };

  if constexpr (IN == 0) {
#pragma unroll
    for (int i = 0; i < AHEAD && i < BPW; ++i) load_x(i);
    __builtin_amdgcn_sched_barrier(0);   // x ahead of the weights
    load_first();
  } else {
    // an eighth e of x: 8 values of row e / (16 KB); 16 neighbouring lanes have a block's row
    const int per = KB * 16, all = M * per;
    const float inv = 1.0f / (float)per;
    auto row_of = [&](int e) { return (int)(((float)e + 0.5f) * inv); };   // e < 2^13: exact
    constexpr int HELD = BPW;   // OWN * per <= BPW * T
    uint4 q[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int e = i * T + (int)threadIdx.x, m = row_of(e), k = 8 * (e - m * per);
      q[i] = e < all && k < a.K ? ldg16(a.x + (long long)m * a.K + k) : make_uint4(0, 0, 0, 0);
    }
    uint4 gain = make_uint4(0, 0, 0, 0);
    if constexpr (IN == 2)   // per <= 16 * BPW * W <= T (BPW <= 4)
      if (8 * (int)threadIdx.x < a.K) gain = ldg16(a.nw + 8 * threadIdx.x);
    __builtin_amdgcn_sched_barrier(0);   // x ahead of the weights
    load_first();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (IN == 2) {
      if ((int)threadIdx.x < per) s_gain[threadIdx.x] = gain;
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        const int e = i * T + (int)threadIdx.x;
        if (e >= all) break;
        const float v[8] = {bf16lo(q[i].x), bf16hi(q[i].x), bf16lo(q[i].y), bf16hi(q[i].y),
                            bf16lo(q[i].z), bf16hi(q[i].z), bf16lo(q[i].w), bf16hi(q[i].w)};
        const float sq = row_sum16(fp8_squares(v));
        if ((lane & 15) == 0) s_sq[e >> 4] = sq;
      }
      __syncthreads();
      if ((int)threadIdx.x < M) {
        double tot = 0.0;
        for (int kb = 0; kb < KB; ++kb) tot += s_sq[threadIdx.x * KB + kb];
        s_rstd[threadIdx.x] = fp8_rstd(tot, a.K, a.eps);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int e = i * T + (int)threadIdx.x;
      if (e >= all) break;
      const int m = row_of(e), at = e - m * per, kb = at >> 4;
      if constexpr (IN == 2) {
        const float rstd = s_rstd[m];
        const uint4 w = s_gain[at];
        q[i] = make_uint4(fp8_norm2(q[i].x, w.x, rstd), fp8_norm2(q[i].y, w.y, rstd),
                          fp8_norm2(q[i].z, w.z, rstd), fp8_norm2(q[i].w, w.w, rstd));
      }
      uint2 c;
      const uint32_t b = fp8_quantize8(q[i], c);
      // the eighth at of the row: 64 j + 16 g + 8 p
      *reinterpret_cast<uint2*>(s_x + ((at >> 1) * M + m) * 16 + 8 * (at & 1)) = c;
      if ((lane & 15) == 0) s_xs[kb * M + m] = (uint8_t)b;
    }
    __syncthreads();
  }
  bf16x8 x[HOLD ? BPW : 1][4];
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < BPW; ++i) operand(i, x[i]);
  }

  auto step = [&](int st, int set, auto load_next) {
    const Weights<BPW>& w = ws[set];
    const bool mine = wv == st % W;   // this wavefront adds the tile's sums
    const int tile = (int)blockIdx.x + st * GRID;
    uint2 hv = make_uint2(0, 0);
    if constexpr (EPI == EPI_RESID) hv = load4(a, r, tile * 16 + 4 * g);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      if (kb0 + i >= KB) break;
      bf16x8 f[4];
      if constexpr (!HOLD) {
        operand(i, x[0]);
        if (i + AHEAD < BPW) load_x(i + AHEAD);
      }
      widen(w.c[i], (w.s[i] >> (8 * ((kb0 + i) & 3))) & 255u, f);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[j], x[HOLD ? i : 0][j], acc, 0, 0, 0);
    }
    s_part[st & 1][wv][lane] = acc;
    if constexpr (IN == 0 && !HOLD) {
      load_x(0);
      load_x(1);
    }
    load_next();
    __syncthreads();   // of the next step but one: every wavefront is past this step's sums
    if (mine) {
      const f32x4 sum = add_parts(s_part[st & 1], 1, W, lane);
      if constexpr (EPI == EPI_SWIGLU) {
        f32x4 up;   // 32 lanes on
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = __float_as_uint(sum[i]);
          up[i] = __uint_as_float(__builtin_amdgcn_permlane32_swap(u, u, false, false)[1]);
        }
        if (g < 2) store4<EPI>(a, r, tile * 8 + 4 * g, sum, up, hv);
      } else {
        store4<EPI>(a, r, tile * 16 + 4 * g, sum, sum, hv);
      }
    }
  };
  pipeline<SETS>(steps, load, step);
}

template <int EPI, int IN>
int launch(const LinearArgs& a, hipStream_t s) {
  const int KB = fp8_blocks(a.K);
  const dim3 grid(a.wt < GRID ? a.wt : GRID);
#define KO_FEW(B, WM, S) \
  hipLaunchKernelGGL((few_kernel<EPI, IN, B, WM, S>), grid, dim3(64 * ((KB + B - 1) / B)), 0, s, a)
  const bool one = a.wt <= GRID;   // a step for every workgroup
  if (KB <= 20) {
    if (one) KO_FEW(2, 10, 1);
    else KO_FEW(2, 10, 2);
  } else if (KB <= 32) {
    if (one) KO_FEW(2, 16, 1);
    else KO_FEW(2, 16, 2);
  } else if constexpr (IN < 2) {
    if (KB <= 48) KO_FEW(3, 16, 1);
    else KO_FEW(5, 16, 1);
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

bool few_rows_served(const LinearArgs& a) { return a.M <= 16 && fp8_blocks(a.K) <= 80; }

bool few_rows_quantized(const LinearArgs& a) {
  const int KB = fp8_blocks(a.K);
  return a.M <= OWN && (!a.nw || KB <= 32);
}

int launch_few_rows(const LinearArgs& a, int epi, hipStream_t s) {
  switch (epi) {
    case EPI_F32: return launch_in<EPI_F32>(a, s);
    case EPI_BF16: return launch_in<EPI_BF16>(a, s);
    case EPI_RESID: return launch_in<EPI_RESID>(a, s);
    default: return launch_in<EPI_SWIGLU>(a, s);
  }
}

}  // namespace ko
