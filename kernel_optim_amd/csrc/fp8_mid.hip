// y = x W^T with W in 8 bits for 17 to 64 rows of x (2 or 4 tiles), held in 8 bits: one weight pass.
//
// As for fewer rows a workgroup's 8 wavefronts share K and stream tiles of W, but every block of W
// now meets 2 or 4 blocks of x: a wavefront holds the codes of its blocks of x in registers for the
// whole launch (K = 2560, 64 rows: 96 of its 256), where loads of x between those of W would make
// each wait for the weights ahead of it. Longer rows do not fit: they take x with W, block by
// block, several blocks ahead. 2 tiles go through bf16 (fp8_core.h); 4 would spill the registers so
// (64 rows of gate/up 36 us) and go to the matrix instruction as codes (19 us).
#include "fp8_linear.h"

namespace {

using namespace ko;

constexpr int GRID = 256, WMAX = 8;

struct Block {
  uint4 c[2];
  uint32_t s;   // the scale's byte is the lowest
  // block kb of tile t
  __device__ __forceinline__ void load_x(const LinearArgs& a, int t, int kb, int KB, int Q, int lane) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      c[j] = ldg16(a.xc + ((long long)t * KB + kb) * FP8_BLOCK + 1024 * j + 16 * lane);
    s = a.xs[((long long)t * Q + (kb >> 2)) * 16 + (lane & 15)] >> (8 * (kb & 3));
  }
  __device__ __forceinline__ void load_w(const LinearArgs& a, long long t, int kb, int KB, int Q,
                                         int lane) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      c[j] = ldg16_stream(a.wc + (t * KB + kb) * FP8_BLOCK + 1024 * j + 16 * lane);
    s = a.ws[(t * Q + (kb >> 2)) * 16 + (lane & 15)] >> (8 * (kb & 3));
  }
  __device__ __forceinline__ void widen(bf16x8 (&out)[4]) const {
    const float sc = __uint_as_float((s & 255u) << 23);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      out[2 * j] = fp8_to_bf16(c[j].x, c[j].y, sc);
      out[2 * j + 1] = fp8_to_bf16(c[j].z, c[j].w, sc);
    }
  }
};

__device__ __forceinline__ i32x8 codes(const Block& b) {
  return (i32x8){(int)b.c[0].x, (int)b.c[0].y, (int)b.c[0].z, (int)b.c[0].w,
                 (int)b.c[1].x, (int)b.c[1].y, (int)b.c[1].z, (int)b.c[1].w};
}

template <int MT>
__device__ __forceinline__ void multiply(const Block& w, const Block (&x)[MT], f32x4 (&acc)[MT]) {
  if constexpr (MT == 4) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
      acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes(w), codes(x[t]), acc[t], 0, 0, 0,
                                                                (int)w.s, 0, (int)x[t].s);
    return;
  }
  bf16x8 f[4], v[4];
  w.widen(f);
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    x[t].widen(v);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[j], v[j], acc[t], 0, 0, 0);
  }
}

// The sums of W wavefronts for tile t of x and a tile of W, stored.
template <int EPI>
__device__ __forceinline__ void finish(const LinearArgs& a, const f32x4 (*part)[64], int stride, int W,
                                       int tile, int t, int lane, uint2 hv) {
  const int r = lane & 15, g = lane >> 4, m = 16 * t + r;
  const f32x4 sum = add_parts(part, stride, W, lane);
  if constexpr (EPI == EPI_SWIGLU) {
    f32x4 up;   // 32 lanes on
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = __float_as_uint(sum[i]);
      up[i] = __uint_as_float(__builtin_amdgcn_permlane32_swap(u, u, false, false)[1]);
    }
    if (g < 2) store4<EPI>(a, m, tile * 8 + 4 * g, sum, up, hv);
  } else {
    store4<EPI>(a, m, tile * 16 + 4 * g, sum, sum, hv);
  }
}

// SETS tiles of W in flight.
template <int EPI, int MT, int BPW, int SETS>
__global__ __launch_bounds__(64 * WMAX) void mid_kernel(LinearArgs a) {
  __shared__ f32x4 s_part[2][WMAX][MT][64];
  const int W = blockDim.x >> 6;
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int KB = fp8_blocks(a.K), Q = fp8_quads(a.K);
  const int kb0 = wv * BPW;   // < KB
  const int steps = (a.wt - 1 - (int)blockIdx.x) / GRID + 1;
  Block x[BPW][MT], ws[SETS][BPW];
  auto load = [&](int st, int set) {
#pragma unroll
    for (int i = 0; i < BPW; ++i)   // a block past the end: the last, not multiplied
      ws[set][i].load_w(a, (int)blockIdx.x + st * GRID, min(kb0 + i, KB - 1), KB, Q, lane);
  };
#pragma unroll
  for (int i = 0; i < BPW; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t)
      x[i][t].load_x(a, min(t, a.xt - 1), min(kb0 + i, KB - 1), KB, Q, lane);
  __builtin_amdgcn_sched_barrier(0);   // x ahead of the weights
#pragma unroll
  for (int i = 0; i < SETS; ++i) load(min(i, steps - 1), i);   // fewer steps: the last one again
  auto step = [&](int st, int set, auto load_next) {
    const int tile = (int)blockIdx.x + st * GRID;
    const int mine = (wv + W - st % W) % W;   // the tile of x whose sums this wavefront adds
    uint2 hv = make_uint2(0, 0);
    if constexpr (EPI == EPI_RESID) hv = load4(a, 16 * mine + r, tile * 16 + 4 * g);
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
      if constexpr (MT == 2 && (BPW == 4 || EPI == EPI_RESID)) {
        // widened anew in every step: the bf16 of all its blocks would not fit the registers
#pragma unroll
        for (int t = 0; t < MT; ++t) asm volatile("" : "+v"(x[i][t].s));
      }
      if (kb0 + i < KB) multiply<MT>(ws[set][i], x[i], acc);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) s_part[st & 1][wv][t][lane] = acc[t];
    load_next();
    __syncthreads();   // of the next step but one: every wavefront is past this step's sums
    for (int t = mine; t < MT; t += W)
      finish<EPI>(a, &s_part[st & 1][0][t], MT, W, tile, t, lane,
                  EPI == EPI_RESID && t != mine ? load4(a, 16 * t + r, tile * 16 + 4 * g) : hv);
  };
  pipeline<SETS>(steps, load, step);
}

// Any K: a workgroup takes one tile of W, its wavefronts a run of blocks each, D of them ahead.
template <int EPI, int MT>
__global__ __launch_bounds__(64 * WMAX) void mid_deep_kernel(LinearArgs a) {
  constexpr int W = WMAX, D = 4;
  __shared__ f32x4 s_part[W][MT][64];
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int KB = fp8_blocks(a.K), Q = fp8_quads(a.K);
  const int begin = KB * wv / W, end = KB * (wv + 1) / W, tile = blockIdx.x;
  Block x[D][MT], w[D];
  auto load = [&](int kb, int i) {
    if (kb >= end) return;
    w[i].load_w(a, tile, kb, KB, Q, lane);
#pragma unroll
    for (int t = 0; t < MT; ++t) x[i][t].load_x(a, min(t, a.xt - 1), kb, KB, Q, lane);
  };
#pragma unroll
  for (int i = 0; i < D; ++i) load(begin + i, i);
  uint2 hv = make_uint2(0, 0);
  if constexpr (EPI == EPI_RESID)
    if (wv < MT) hv = load4(a, 16 * wv + r, tile * 16 + 4 * g);
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = begin; k0 < end; k0 += D) {
#pragma unroll
    for (int i = 0; i < D; ++i) {
      if (k0 + i >= end) break;
      multiply<MT>(w[i], x[i], acc);
      load(k0 + i + D, i);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) s_part[wv][t][lane] = acc[t];
  __syncthreads();
  if (wv < MT) finish<EPI>(a, &s_part[0][wv], MT, W, tile, wv, lane, hv);
}

template <int EPI, int MT>
int launch(const LinearArgs& a, hipStream_t s) {
  const int KB = fp8_blocks(a.K);
  const dim3 grid(a.wt < GRID ? a.wt : GRID);
#define KO_MID(B, S) \
  hipLaunchKernelGGL((mid_kernel<EPI, MT, B, S>), grid, dim3(64 * ((KB + B - 1) / B)), 0, s, a)
  const bool one = a.wt <= GRID;   // a step for every workgroup
  if (KB <= 8) KO_MID(1, 2);
  else if (KB <= 24) {
    if (one) KO_MID(3, 1);
    else KO_MID(3, 2);
  } else if (KB <= 32) {
    if (one || MT == 4) KO_MID(4, 1);   // 64 rows: a second set would spill
    else KO_MID(4, MT == 4 ? 1 : 2);
  } else hipLaunchKernelGGL((mid_deep_kernel<EPI, MT>), dim3(a.wt), dim3(64 * WMAX), 0, s, a);
#undef KO_MID
  return KO_LAUNCH_STATUS();
}

}  // namespace

namespace ko {

bool mid_rows_served(const LinearArgs& a, int epi) { return a.xt <= (epi == EPI_F32 ? 2 : 4); }

int launch_mid_rows(const LinearArgs& a, int epi, hipStream_t s) {
#define KO_EPI(E) return a.xt <= 2 ? launch<E, 2>(a, s) : launch<E, 4>(a, s)
  switch (epi) {
    case EPI_F32: return launch<EPI_F32, 2>(a, s);
    case EPI_BF16: KO_EPI(EPI_BF16);
    case EPI_RESID: KO_EPI(EPI_RESID);
    default: KO_EPI(EPI_SWIGLU);
  }
#undef KO_EPI
}

}  // namespace ko
