// Rows to 8-bit floating point and back (layout: fp8_core.h).
//
// A wavefront takes a block of 16 rows and 128 values: lane l holds 2 x 16 values of row l % 16,
// the maximum over the row's 128 takes two lane swaps, and the codes leave in two stores of 1 KB.
// HBM bounds both ways: 4099 x 9736 bf16 values are quantised in 28 us (120 MB, 4.3 TB/s) and read
// back in 24.6 (4.9 TB/s, a large copy's rate), 8192 x 2560 behind a norm in 19.1 (3.3 TB/s, as the
// rows wait for their sum of squares between reading and writing).
#include "fp8_core.h"

namespace {

using namespace ko;

// A lane's 2 x 16 values of a block's row (k: the first), packed as they come; values from K on are
// zero. K is a multiple of 8 and rows are 16-byte aligned. No load is under a condition (what lies
// past the end reads the row's beginning), so that many are on their way at once.
template <bool F32IN>
struct Raw {
  static constexpr int L = F32IN ? 2 : 1;   // loads of 8 values
  uint4 q[2][2][L];
  __device__ __forceinline__ void load(const void* x, long long at, int k, int K) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int e = k + 64 * j + 8 * p;
        const long long o = at + (e < K ? e : 0);
#pragma unroll
        for (int l = 0; l < L; ++l)
          q[j][p][l] = F32IN ? ldg16(static_cast<const float*>(x) + o + 4 * l)
                             : ldg16(static_cast<const uint16_t*>(x) + o);
      }
  }
  __device__ __forceinline__ void clear(int k, int K, bool ok) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p)
        if (!ok || k + 64 * j + 8 * p >= K) {
#pragma unroll
          for (int l = 0; l < L; ++l) q[j][p][l] = make_uint4(0, 0, 0, 0);
        }
  }
  __device__ __forceinline__ void unpack(float (&v)[2][16]) const {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int l = 0; l < L; ++l) {
          const uint4 t = q[j][p][l];
          const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (F32IN) {
              v[j][8 * p + 4 * l + i] = __uint_as_float(w[i]);
            } else {
              v[j][8 * p + 2 * i] = bf16lo(w[i]);
              v[j][8 * p + 2 * i + 1] = bf16hi(w[i]);
            }
          }
        }
  }
};

// One block's codes into the matrix; returns the row's scale byte.
__device__ __forceinline__ uint32_t store_block(const float (&v)[2][16], uint8_t* block, int lane) {
  uint4 c[2];
  const uint32_t b = fp8_quantize_block(v, c);
#pragma unroll
  for (int j = 0; j < 2; ++j) *reinterpret_cast<uint4*>(block + 1024 * j + 16 * lane) = c[j];
  return b;
}

// A wavefront for each quad of blocks of a tile.
template <bool F32IN>
__global__ __launch_bounds__(256) void quantize_kernel(const void* __restrict__ x, long long stride,
                                                       int rows, int K, int pair,
                                                       uint8_t* __restrict__ codes,
                                                       uint32_t* __restrict__ scales,
                                                       long long units) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int Q = fp8_quads(K), KB = fp8_blocks(K);
  const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (u >= units) return;
  const long long t = u / Q;
  const int q = (int)(u - t * Q);
  const int row = fp8_row(t, r, rows, pair);
  const long long at = (long long)max(row, 0) * stride;
  uint32_t sc = 0;
  Raw<F32IN> raw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[i].load(x, at, (4 * q + i) * 128 + 16 * g, K);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int kb = 4 * q + i;
    if (kb < KB) {
      float v[2][16];
      raw[i].clear(kb * 128 + 16 * g, K, row >= 0);
      raw[i].unpack(v);
      sc |= store_block(v, codes + (t * KB + kb) * FP8_BLOCK, lane) << (8 * i);
    }
  }
  if (g == 0) scales[(t * Q + q) * 16 + r] = sc;
}

constexpr int NORM_BLOCKS = 1024;   // K up to 131,072

// RMSNorm in front (bf16 rows): a workgroup takes a tile, sums the squares of its 16 rows (a block's
// in fp32, blocks in 64 bits), and its wavefronts quantise bf16(nw * bf16(x * rstd)). R blocks a
// wavefront stay in registers between the two; R = 0 (long rows) reads them again.
template <int R>
__global__ __launch_bounds__(1024) void quantize_norm_kernel(
    const uint16_t* __restrict__ x, long long stride, int rows, int K,
    const uint16_t* __restrict__ nw, float eps, uint8_t* __restrict__ codes,
    uint32_t* __restrict__ scales) {
  extern __shared__ float s_sq[];   // [blocks][16]
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, W = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int Q = fp8_quads(K), KB = fp8_blocks(K);
  const long long t = blockIdx.x;
  const int row = fp8_row(t, r, rows, false);
  const long long at = (long long)max(row, 0) * stride;
  Raw<false> raw[R ? R : 1];
  auto fetch = [&](int i, int kb) {
    raw[i].load(x, at, min(kb, KB - 1) * 128 + 16 * g, K);
  };
  auto squares = [&](int i, int kb) {
    if (kb >= KB) return;
    float v[2][16];
    raw[i].clear(kb * 128 + 16 * g, K, row >= 0);
    raw[i].unpack(v);
    const float sq = fp8_square_sum(v);
    if (g == 0) s_sq[kb * 16 + r] = sq;
  };
  if constexpr (R) {
#pragma unroll
    for (int i = 0; i < R; ++i) fetch(i, wv + i * W);
#pragma unroll
    for (int i = 0; i < R; ++i) squares(i, wv + i * W);
  } else {
    for (int kb = wv; kb < KB; kb += W) fetch(0, kb), squares(0, kb);
  }
  __syncthreads();
  double tot = 0.0;
  for (int kb = 0; kb < KB; ++kb) tot += s_sq[kb * 16 + r];
  const float rstd = row >= 0 ? fp8_rstd(tot, K, eps) : 0.f;   // eps may be 0
  uint8_t* sc = reinterpret_cast<uint8_t*>(scales);
  auto quantize = [&](int i, int kb) {
    uint32_t b = 0;
    if (kb < KB) {
      float v[2][16];
      Raw<false> gain;
      gain.load(nw, 0, kb * 128 + 16 * g, K);
      gain.clear(kb * 128 + 16 * g, K, row >= 0);   // padding rows stay zeros, with no sign
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint4& q = raw[i].q[j][p][0];
          const uint4 w = gain.q[j][p][0];
          q = make_uint4(fp8_norm2(q.x, w.x, rstd), fp8_norm2(q.y, w.y, rstd),
                         fp8_norm2(q.z, w.z, rstd), fp8_norm2(q.w, w.w, rstd));
        }
      raw[i].unpack(v);
      b = store_block(v, codes + (t * KB + kb) * FP8_BLOCK, lane);
    }
    if (g == 0 && kb < 4 * Q) sc[((t * Q + (kb >> 2)) * 16 + r) * 4 + (kb & 3)] = (uint8_t)b;
  };
  if constexpr (R) {
#pragma unroll
    for (int i = 0; i < R; ++i) quantize(i, wv + i * W);
    if (wv == 0)   // the last quad's padding
      for (int kb = R * W; kb < 4 * Q; ++kb) quantize(0, kb);
  } else {
    for (int kb = wv; kb < 4 * Q; kb += W) {
      if (kb < KB) {
        fetch(0, kb);
        raw[0].clear(kb * 128 + 16 * g, K, row >= 0);
      }
      quantize(0, kb);
    }
  }
}

// Few bf16 rows: a workgroup for each row of a tile (padding rows among them), 8 values a thread, so
// that a decode step's rows are spread over the GPU. It stores 8 bytes at a time, which many rows
// feel: behind a norm 512 x 2560 take 4.7 us against 9.1 with a workgroup a tile, 1024 6.1 against 9.3,
// 2048 11.0 against 10.5; of 9728 values 256 rows 5.2 against 6.5, 512 8.9 against 7.7.
constexpr long long FEW = 3ll << 20;   // values
constexpr int ROW_LOADS = 8;   // K up to 8 * 1024 * ROW_LOADS

template <bool NORM>
__global__ __launch_bounds__(1024) void quantize_row_kernel(const uint16_t* __restrict__ x,
                                                            long long stride, int rows, int K,
                                                            int pair,
                                                            const uint16_t* __restrict__ nw,
                                                            float eps, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales) {
  extern __shared__ float s_sq[];   // NORM: [blocks]
  const int KB = fp8_blocks(K), Q = fp8_quads(K), T = blockDim.x, all = 16 * KB;
  const long long t = blockIdx.x >> 4;
  const int r = blockIdx.x & 15, row = fp8_row(t, r, rows, pair);
  const uint16_t* src = x + (long long)max(row, 0) * stride;
  uint4 q[ROW_LOADS], w[NORM ? ROW_LOADS : 1];
#pragma unroll
  for (int i = 0; i < ROW_LOADS; ++i) {
    const int e = i * T + (int)threadIdx.x;
    if (e >= all) break;
    const bool in = row >= 0 && 8 * e < K;
    q[i] = in ? ldg16(src + 8 * e) : make_uint4(0, 0, 0, 0);
    if constexpr (NORM) w[i] = in ? ldg16(nw + 8 * e) : make_uint4(0, 0, 0, 0);
  }
  float rstd = 0.f;
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < ROW_LOADS; ++i) {
      const int e = i * T + (int)threadIdx.x;
      if (e >= all) break;
      const float v[8] = {bf16lo(q[i].x), bf16hi(q[i].x), bf16lo(q[i].y), bf16hi(q[i].y),
                          bf16lo(q[i].z), bf16hi(q[i].z), bf16lo(q[i].w), bf16hi(q[i].w)};
      const float sq = row_sum16(fp8_squares(v));
      if ((e & 15) == 0) s_sq[e >> 4] = sq;
    }
    __syncthreads();
    double tot = 0.0;
    for (int kb = 0; kb < KB; ++kb) tot += s_sq[kb];
    rstd = row >= 0 ? fp8_rstd(tot, K, eps) : 0.f;   // eps may be 0
  }
#pragma unroll
  for (int i = 0; i < ROW_LOADS; ++i) {
    const int e = i * T + (int)threadIdx.x;
    if (e >= all) break;
    if constexpr (NORM)
      q[i] = make_uint4(fp8_norm2(q[i].x, w[i].x, rstd), fp8_norm2(q[i].y, w[i].y, rstd),
                        fp8_norm2(q[i].z, w[i].z, rstd), fp8_norm2(q[i].w, w[i].w, rstd));
    uint2 c;
    const uint32_t b = fp8_quantize8(q[i], c);
    const int kb = e >> 4;
    *reinterpret_cast<uint2*>(codes + (t * KB + kb) * FP8_BLOCK + ((e >> 1) & 7) * 256 + r * 16 +
                              8 * (e & 1)) = c;
    if ((e & 15) == 0) scales[((t * Q + (kb >> 2)) * 16 + r) * 4 + (kb & 3)] = (uint8_t)b;
  }
  if ((int)threadIdx.x < 4 * Q - KB)   // the last quad's padding
    scales[((t * Q + Q - 1) * 16 + r) * 4 + 3 - (int)threadIdx.x] = 0;
}

// The values back: a wavefront for each block, rows written in pieces of 16 values.
template <bool F32OUT>
__global__ __launch_bounds__(256) void read_kernel(const uint8_t* __restrict__ codes,
                                                   const uint32_t* __restrict__ scales, int rows,
                                                   int K, int pair, void* __restrict__ out,
                                                   long long stride, long long units) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int Q = fp8_quads(K), KB = fp8_blocks(K);
  const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (u >= units) return;
  const long long t = u / KB;
  const int kb = (int)(u - t * KB);
  const int row = fp8_row(t, r, rows, pair);
  if (row < 0) return;
  const uint32_t b = (scales[(t * Q + (kb >> 2)) * 16 + r] >> (8 * (kb & 3))) & 255u;
  const float s = fp8_scale(b);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint4 c = ldg16(codes + u * FP8_BLOCK + 1024 * j + 16 * lane);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    const int k = kb * 128 + 64 * j + 16 * g;
    float v[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
      v[4 * i] = lo[0] * s;
      v[4 * i + 1] = lo[1] * s;
      v[4 * i + 2] = hi[0] * s;
      v[4 * i + 3] = hi[1] * s;
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (k + 8 * p >= K) break;
      const float* e = v + 8 * p;
      if constexpr (F32OUT) {
        float* o = static_cast<float*>(out) + row * stride + k + 8 * p;
        *reinterpret_cast<float4*>(o) = make_float4(e[0], e[1], e[2], e[3]);
        *reinterpret_cast<float4*>(o + 4) = make_float4(e[4], e[5], e[6], e[7]);
      } else {
        uint16_t* o = static_cast<uint16_t*>(out) + row * stride + k + 8 * p;
        *reinterpret_cast<uint4*>(o) =
            make_uint4(pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3]), pack_bf16x2(e[4], e[5]),
                       pack_bf16x2(e[6], e[7]));
      }
    }
  }
}

// Sizes whose units fit one launch and whose byte offsets fit 63 bits.
int check(int rows, int K, int pair, long long stride) {
  if (rows < 1 || K < 8 || (K & 7) || stride < 0 || (stride & 7) || (pair && (rows & 1)))
    return KO_EINVAL;
  if (K > FP8_K_MAX || fp8_tiles(rows, pair) * fp8_blocks(K) > 0x7fffffffll) return KO_ERANGE;
  return KO_OK;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

extern "C" {

int ko_fp8_quantize(const void* x, int x_f32, long long stride, int rows, int K, int pair,
                    const void* nw, float eps, void* codes, void* scales, void* stream) {
  if (!x || !codes || !scales) return KO_EINVAL;
  if (const int st = check(rows, K, pair, stride)) return st;
  if (!al16(x) || !al16(codes) || !al16(scales) || (nw && !al16(nw))) return KO_EINVAL;
  if (nw && (x_f32 || pair)) return KO_ENOTSUP;
  if (nw && fp8_blocks(K) > NORM_BLOCKS) return KO_ERANGE;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const long long tiles = fp8_tiles(rows, pair);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint32_t* sc = static_cast<uint32_t*>(scales);
  const int all = 16 * fp8_blocks(K);
  if (!x_f32 && (long long)rows * K <= FEW && all <= 1024 * ROW_LOADS) {
    const int per = (all + ROW_LOADS - 1) / ROW_LOADS;
    const int threads = all <= 1024 ? (all + 63) / 64 * 64 : per <= 640 ? 640 : 1024;
    const dim3 grid((unsigned)(16 * tiles));
    if (nw)
      hipLaunchKernelGGL(quantize_row_kernel<true>, grid, dim3(threads), 4 * fp8_blocks(K), s,
                         static_cast<const uint16_t*>(x), stride, rows, K, pair,
                         static_cast<const uint16_t*>(nw), eps, c, static_cast<uint8_t*>(scales));
    else
      hipLaunchKernelGGL(quantize_row_kernel<false>, grid, dim3(threads), 0, s,
                         static_cast<const uint16_t*>(x), stride, rows, K, pair, nullptr, 0.f, c,
                         static_cast<uint8_t*>(scales));
    return KO_LAUNCH_STATUS();
  }
  if (nw) {
    const int KB = fp8_blocks(K);
    const uint16_t *xb = static_cast<const uint16_t*>(x), *wb = static_cast<const uint16_t*>(nw);
    if (!fp8_launchable(tiles, 64 * (KB <= 32 ? (KB + 1) / 2 : 16))) return KO_ERANGE;
#define KO_NORM(R, WAVES)                                                                      \
  hipLaunchKernelGGL(quantize_norm_kernel<R>, dim3((unsigned)tiles), dim3(64 * (WAVES)), 64 * KB, s, \
                     xb, stride, rows, K, wb, eps, c, sc)
    if (KB <= 32) KO_NORM(2, (KB + 1) / 2);
    else if (KB <= 64) KO_NORM(4, (KB + 3) / 4);
    else KO_NORM(0, 16);
#undef KO_NORM
    return KO_LAUNCH_STATUS();
  }
  const long long units = tiles * fp8_quads(K);
  if (!fp8_launchable((units + 3) / 4, 256)) return KO_ERANGE;
  const dim3 grid((unsigned)((units + 3) / 4));
  if (x_f32)
    hipLaunchKernelGGL(quantize_kernel<true>, grid, dim3(256), 0, s, x, stride, rows, K, pair, c,
                       sc, units);
  else
    hipLaunchKernelGGL(quantize_kernel<false>, grid, dim3(256), 0, s, x, stride, rows, K, pair, c,
                       sc, units);
  return KO_LAUNCH_STATUS();
}

int ko_fp8_read(const void* codes, const void* scales, int rows, int K, int pair, void* out,
                int out_f32, long long stride, void* stream) {
  if (!codes || !scales || !out) return KO_EINVAL;
  if (const int st = check(rows, K, pair, stride)) return st;
  if (!al16(codes) || !al16(scales) || !al16(out)) return KO_EINVAL;
  const long long units = fp8_tiles(rows, pair) * fp8_blocks(K);
  if (!fp8_launchable((units + 3) / 4, 256)) return KO_ERANGE;
  const dim3 grid((unsigned)((units + 3) / 4));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (out_f32)
    hipLaunchKernelGGL(read_kernel<true>, grid, dim3(256), 0, s,
                       static_cast<const uint8_t*>(codes), static_cast<const uint32_t*>(scales),
                       rows, K, pair, out, stride, units);
  else
    hipLaunchKernelGGL(read_kernel<false>, grid, dim3(256), 0, s,
                       static_cast<const uint8_t*>(codes), static_cast<const uint32_t*>(scales),
                       rows, K, pair, out, stride, units);
  return KO_LAUNCH_STATUS();
}

}  // extern "C"
