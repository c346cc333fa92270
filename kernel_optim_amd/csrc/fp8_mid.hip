// y = x W^T with W in 8 bits for 17 to 64 rows of x (2 or 4 tiles), held in 8 bits: one weight pass.
//
// As for fewer rows a workgroup's 8 wavefronts share K and stream tiles of W, but every block of W
// now meets 2 or 4 blocks of x: a wavefront holds the codes of its blocks of x in registers for the
// whole launch (K = 2560, 64 rows: 96 of its 256), where loads of x between those of W would make
// each wait for the weights ahead of it. Longer rows do not fit: they are split. 2 tiles go through
// bf16 (fp8_core.h); 4 would spill the registers so (64 rows of gate/up, 19,456 x 2560, 36 us) and go
// to the matrix instruction as codes (19 us with x's own launch, 2.6 TB/s of W).
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

// The sums of tile t of x and a tile of W, stored.
template <int EPI>
__device__ __forceinline__ void finish(const LinearArgs& a, f32x4 sum, int tile, int t, int lane,
                                       uint2 hv) {
  const int r = lane & 15, g = lane >> 4, m = 16 * t + r;
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
      finish<EPI>(a, add_parts(&s_part[st & 1][0][t], MT, W, lane), tile, t, lane,
                  EPI == EPI_RESID && t != mine ? load4(a, 16 * t + r, tile * 16 + 4 * g) : hv);
  };
  pipeline<SETS>(steps, load, step);
}

// Longer rows: a workgroup takes two tiles of W and one of S runs of K's blocks, its wavefronts a part
// of the run each, D blocks of x and W ahead. With all of K, 80 workgroups (2560 columns) would read
// 622 KB of x each and leave most CUs idle (160 with one tile each: 20 us for 9728 values by 64 rows);
// a CU takes in what others read too at 70 (256 KB) to 120 bytes a ns (4 MB), from L2, and its
// share of what nobody else reads at 25 with all 256 at it. The S partial sums of
// a pair of tiles meet in memory, where the last of its workgroups adds them in order. 9728 values by
// 64 rows, 2560 columns: 13.4 us, in which a workgroup reads 208 KB of x and 104 KB of W, about 3 and 4 us
// at those rates; the rest is latency and the meeting (wavefronts wait in 65 % of their cycles).
template <int EPI, int MT>
__global__ __launch_bounds__(64 * WMAX) void split_kernel(LinearArgs a, int S) {
  constexpr int W = WMAX, NT = 2, D = MT == 4 ? 2 : 4, PARTS = MT * NT;
  __shared__ f32x4 s_part[W][PARTS][64];
  __shared__ int s_arrived;
  const int lane = threadIdx.x & 63, wv = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int KB = fp8_blocks(a.K), Q = fp8_quads(a.K);
  const int pair = blockIdx.x / S, run = blockIdx.x - pair * S;
  const int r0 = KB * run / S, r1 = KB * (run + 1) / S;
  const int begin = r0 + (r1 - r0) * wv / W, end = r0 + (r1 - r0) * (wv + 1) / W;
  const int tile0 = pair * NT;
  Block x[D][MT], w[D][NT];
  auto load = [&](int kb, int i) {
    if (kb >= end) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) w[i][t].load_w(a, min(tile0 + t, a.wt - 1), kb, KB, Q, lane);
#pragma unroll
    for (int t = 0; t < MT; ++t) x[i][t].load_x(a, min(t, a.xt - 1), kb, KB, Q, lane);
  };
#pragma unroll
  for (int i = 0; i < D; ++i) load(begin + i, i);
  // wavefront wv < PARTS ends with the sums of tile wv / MT of W and wv % MT of x
  const int tile = tile0 + wv / MT, xt = wv % MT;
  uint2 hv = make_uint2(0, 0);
  if constexpr (EPI == EPI_RESID) hv = load4(a, 16 * xt + r, tile * 16 + 4 * g);
  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[n][t] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = begin; k0 < end; k0 += D) {
#pragma unroll
    for (int i = 0; i < D; ++i) {
      if (k0 + i >= end) break;
#pragma unroll
      for (int n = 0; n < NT; ++n) multiply<MT>(w[i][n], x[i], acc[n]);
      load(k0 + i + D, i);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < MT; ++t) s_part[wv][n * MT + t][lane] = acc[n][t];
  __syncthreads();
  const bool adds = wv < PARTS;   // uniform per wavefront
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (adds) sum = add_parts(&s_part[0][wv], PARTS, W, lane);
  if (S > 1) {
    typedef unsigned long long u64;
    u64* slots = reinterpret_cast<u64*>(a.part) + (long long)pair * S * PARTS * 128;
    if (adds) {
      u64* mine = slots + ((long long)run * PARTS + wv) * 128 + 2 * lane;
      const u64* v = reinterpret_cast<const u64*>(&sum);
      __hip_atomic_store(mine, v[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(mine + 1, v[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __builtin_amdgcn_s_waitcnt(0);   // this thread's slot stores are performed
    __syncthreads();
    if (threadIdx.x == 0)
      s_arrived = __hip_atomic_fetch_add(a.counters + pair, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_arrived != S - 1) return;
    if (threadIdx.x == 0)   // for the next call
      __hip_atomic_store(a.counters + pair, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (adds) {
      sum = {0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < S; ++i) {
        const uint4 v = ldg16_coherent(slots + ((long long)i * PARTS + wv) * 128 + 2 * lane);
        sum += (f32x4){__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
      }
    }
  }
  if (adds && tile < a.wt) finish<EPI>(a, sum, tile, xt, lane, hv);
}

int split_pairs(const LinearArgs& a) { return (a.wt + 1) / 2; }
int split_runs(const LinearArgs& a) {
  const int s = 256 / split_pairs(a), most = fp8_blocks(a.K) / WMAX;   // a block for every wavefront
  return s < 1 ? 1 : s < most ? s : most;
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
  } else {
    const int S = split_runs(a);
    hipLaunchKernelGGL((split_kernel<EPI, MT>), dim3(split_pairs(a) * S), dim3(64 * WMAX), 0, s, a, S);
  }
#undef KO_MID
  return KO_LAUNCH_STATUS();
}

}  // namespace

namespace ko {

long long mid_rows_scratch(const LinearArgs& a) {
  const int S = split_runs(a);
  // the counters first: their place does not depend on the number of rows
  return fp8_blocks(a.K) <= 32 || S == 1 ? 0 : 4096 + (long long)split_pairs(a) * S * 8192;
}

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
