// Writers and the reader of the 4-bit KV cache (kv4_core.h), for gfx950.
//
//   ko_kv4_write   bf16 K/V rows of a prompt into the cache
//   ko_kv4_read    cached keys back as bf16
//   ko_kv4_append  the decode and verify steps' q/k RMSNorm + RoPE with the quantised append,
//                  beside ko_qk_norm_rope (engine/kernels/fused.py:54-106)
//
// All three are bound by the bytes they move.
#include "kv4_core.h"

using namespace ko;

namespace {

constexpr int NT = 256;
constexpr long long KV4_MAX_WAVES = (1LL << 26) - 4;

struct Kv4Rows {
  const uint16_t* k;  // [B, nkv, S, D], strides in elements
  const uint16_t* v;
  long long kb, kh, ks, vb, vh, vs;
  uint8_t* cache;
  long long cb, ch;  // bytes
  const int* start;
  const int* lengths;
  int B, S, nkv, cap, nb;
};

// A block to write or read: which (sequence, head, block), the first slot's row and the number
// of rows. False where the block holds no row.
__device__ __forceinline__ bool locate(const Kv4Rows& a, long long item, int& b, int& h, int& blk,
                                       int& row0, int& rows) {
  if (item >= (long long)a.B * a.nkv * a.nb) return false;
  const int pair = (int)(item / a.nb), ib = (int)(item - (long long)pair * a.nb);
  b = pair / a.nkv;
  h = pair - b * a.nkv;
  const int start = a.start ? a.start[b] : 0;
  // rows of this sequence: at most S, none behind the cache's last slot
  const long long room = (long long)a.cap - start;
  rows = a.lengths ? min(a.lengths[b], a.S) : a.S;
  if (room < rows) rows = (int)(room < 0 ? 0 : room);
  const long long bl = (long long)(start >> 5) + ib;  // floor, for negative starts too
  const long long r0 = bl * KV4_KEYS - start;         // row of the block's first slot
  if (bl < 0 || bl * KV4_KEYS >= a.cap || r0 >= rows || rows <= 0) return false;
  blk = (int)bl;
  row0 = (int)r0;
  return true;
}

// Writing and reading a block take two wavefronts, one for K and one for V, with all of a
// block's loads in flight at once.
//
// A writing lane holds 32 consecutive values of a key, so a group's smallest and largest come from
// its registers (and its 1 or 3 neighbours') and its scale is computed once. (With V in the layout
// it is stored in, 16 lanes a key, every lane computed the scales of 32 groups: 57 against 36
// us for 32768 tokens of 8 heads of 128 in groups of 32, 4.9 TB/s, a copy's rate.) K's codes leave
// as they are, V's through LDS, which holds the block as the cache does.
template <int D, int NG, bool V>
__device__ __forceinline__ void write_block(const uint16_t* src, long long stride, uint8_t* dst,
                                            int row0, int rows, int lane, uint8_t* lds) {
  constexpr int I = D / 32, HP = D / 64, IPG = I / NG, KP = 64 / I, PASSES = 32 / KP;
  const int i = lane % I, kk = lane / I;
  uint32_t* scales = reinterpret_cast<uint32_t*>(dst + 32 * D) + (V ? 32 * NG : 0);
  uint4 x[PASSES][4];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int row = min(max(row0 + p * KP + kk, 0), rows - 1);  // others are not stored
#pragma unroll
    for (int e = 0; e < 4; ++e) x[p][e] = ldg16(src + row * stride + 32 * i + 8 * e);
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int key = p * KP + kk, row = row0 + key;
    const bool live = row >= 0 && row < rows;
    uint32_t u[16];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      u[4 * e] = x[p][e].x, u[4 * e + 1] = x[p][e].y, u[4 * e + 2] = x[p][e].z, u[4 * e + 3] = x[p][e].w;
    float mn = bf16lo(u[0]), mx = mn;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      mn = kv4_min(kv4_min(mn, bf16lo(u[e])), bf16hi(u[e]));
      mx = kv4_max(kv4_max(mx, bf16lo(u[e])), bf16hi(u[e]));
    }
    if (IPG >= 2) mn = kv4_min(mn, dpp_f<0xB1>(mn)), mx = kv4_max(mx, dpp_f<0xB1>(mx));  // lane ^ 1
    if (IPG >= 4) mn = kv4_min(mn, dpp_f<0x4E>(mn)), mx = kv4_max(mx, dpp_f<0x4E>(mx));  // lane ^ 2
    Kv4Group gr;
    gr.from(mn, mx);
    if (live && i % IPG == 0) scales[i / IPG * 32 + key] = gr.sc;
    if constexpr (V) {  // the byte of columns 32 i + 2 n, + 1
      uint8_t* d = lds + (key / 8 * HP + i / 2) * 256 + key % 8 * 2 + (i & 1);
#pragma unroll
      for (int n = 0; n < 16; ++n)
        d[16 * n] = (uint8_t)(gr.raw(bf16lo(u[n])) | gr.raw(bf16hi(u[n])) << 4);
    } else if (live) {
#pragma unroll
      for (int kg = 0; kg < 4; ++kg) {  // the dword of values 32 i + 8 kg .. + 7
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int e = 3; e >= 0; --e) {
          lo = lo << 4 | gr.raw(bf16lo(u[4 * kg + e]));
          hi = hi << 4 | gr.raw(bf16hi(u[4 * kg + e]));
        }
        reinterpret_cast<uint32_t*>(dst + key * (D / 2) + kg * (D / 8))[i] = (lo & 0xffffu) | hi << 16;
      }
    }
  }
  if constexpr (V) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < HP; ++p) {
      const int at = 64 * p + lane;  // 16 bytes: 8 keys in pairs
      const int row8 = row0 + at / (16 * HP) * 8;
      const uint4 w = reinterpret_cast<const uint4*>(lds)[at];
      uint8_t* d = dst + 16 * D + 16 * at;
      if (row8 >= 0 && row8 + 8 <= rows) {
        *reinterpret_cast<uint4*>(d) = w;
      } else {  // a part of the 8 keys: two bytes of each
        const uint32_t y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (row8 + e >= 0 && row8 + e < rows)
            *reinterpret_cast<uint16_t*>(d + 2 * e) = (uint16_t)(y[e / 2] >> (16 * (e & 1)));
      }
    }
  }
}

template <int D, int NG>
__global__ __launch_bounds__(NT) void kv4_write_kernel(Kv4Rows a) {
  __shared__ __align__(16) uint8_t lds[NT / 64][16 * D];
  const int wave = uniform(threadIdx.x >> 6);
  const long long item = (long long)blockIdx.x * (NT / 64) + wave;
  int b, h, blk, row0, rows;
  if (!locate(a, item >> 1, b, h, blk, row0, rows)) return;
  uint8_t* dst = a.cache + b * a.cb + h * a.ch + (long long)blk * kv4_block_bytes(D, NG);
  if (item & 1)
    write_block<D, NG, true>(a.v + b * a.vb + h * a.vh, a.vs, dst, row0, rows, threadIdx.x & 63,
                             lds[wave]);
  else
    write_block<D, NG, false>(a.k + b * a.kb + h * a.kh, a.ks, dst, row0, rows, threadIdx.x & 63,
                              lds[wave]);
}

// c + s (n - 8): the product is exact in fp32 (8 by 4 bits), the sum rounds once. Past bf16's largest
// value it is that value: lim is, and NaN where s or c is (v_med3_f32 of three NaN is one; with
// two numbers beside a NaN it would be a number). 32768 tokens of 8 heads of 128: 39.1 us, 38.5 without
// the clamp (groups of 128: 38.8, 37.1). A smaller s cannot take its place: where (max - c) / 7 is far
// above (c - min) / 8, codes that are used stay past the end.
__device__ __forceinline__ float kv4_lim(uint32_t sc) {
  return fmaf(bf16lo(sc), 0.f, fmaf(bf16hi(sc), 0.f, 0x1.fep127f));
}
__device__ __forceinline__ float kv4_value(uint32_t n, uint32_t sc, float lim) {
  const float x = fmaf(bf16lo(sc), (float)(int)(n & 15u) - 8.0f, bf16hi(sc));
  return __builtin_amdgcn_fmed3f(x, -lim, lim);
}

template <int D, int NG>
__device__ __forceinline__ void read_k(const uint8_t* src, uint16_t* kp, long long ks, int row0,
                                       int rows, int lane) {
  constexpr int I = D / 32, IPG = I / NG;
  const int r = lane & 15, q = lane >> 4;
  const uint32_t* ksc = reinterpret_cast<const uint32_t*>(src + 32 * D);
  uint32_t w[2][I], sc[2][NG];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int key = 16 * half + r;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(src + key * (D / 2) + q * (D / 8));
#pragma unroll
    for (int i = 0; i < I; ++i) w[half][i] = p[i];
#pragma unroll
    for (int g = 0; g < NG; ++g) sc[half][g] = ksc[g * 32 + key];
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + 16 * half + r;
    const bool live = row >= 0 && row < rows;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t x = w[half][i], c = sc[half][i / IPG];
      const float lim = kv4_lim(c);
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[e] = pack_bf16x2(kv4_value(x >> (4 * e), c, lim), kv4_value(x >> (4 * e + 16), c, lim));
      if (live)
        *reinterpret_cast<uint4*>(kp + row * ks + 32 * i + 8 * q) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// o[i] of lane l of a quad becomes o[l] of lane i: two exchanges of halves.
__device__ __forceinline__ uint32_t dpp_u(uint32_t v, bool by2) {
  return (uint32_t)(by2 ? __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false)
                        : __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
}
__device__ __forceinline__ void quad_transpose(uint32_t (&o)[4], int l) {
#pragma unroll
  for (int s = 1; s <= 2; s *= 2) {
    const bool up = l & s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & s) continue;
      // the lane without bit s gives o[i + s] and takes the other's o[i]
      const uint32_t give = up ? o[i] : o[i + s];
      const uint32_t got = dpp_u(give, s == 2);
      o[i] = up ? got : o[i];
      o[i + s] = up ? o[i + s] : got;
    }
  }
}

template <int D, int NG>
__device__ __forceinline__ void read_v(const uint8_t* src, uint16_t* vp, long long vs, int row0,
                                       int rows, int lane) {
  constexpr int I = D / 32, HP = D / 64, IPG = I / NG;
  const int r = lane & 15, q = lane >> 4;
  const uint32_t* vsc = reinterpret_cast<const uint32_t*>(src + 32 * D) + 32 * NG;
  uint32_t w[HP][4], sc[NG][8];
#pragma unroll
  for (int p = 0; p < HP; ++p) {
    const uint4 x = ldg16(src + 16 * D + ((q * HP + p) * 16 + r) * 16);
    w[p][0] = x.x, w[p][1] = x.y, w[p][2] = x.z, w[p][3] = x.w;
  }
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const uint4 x = ldg16(vsc + g * 32 + 8 * q + e);
      sc[g][e] = x.x, sc[g][e + 1] = x.y, sc[g][e + 2] = x.z, sc[g][e + 3] = x.w;
    }
  const int row8 = row0 + 8 * q;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool live = row8 + e >= 0 && row8 + e < rows;
    uint32_t o[I];
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint32_t n = w[i / 2][e / 2] >> (16 * (e & 1) + 8 * (i & 1));
      const uint32_t c = sc[i / IPG][e];
      const float lim = kv4_lim(c);
      o[i] = pack_bf16x2(kv4_value(n, c, lim), kv4_value(n >> 4, c, lim));
    }
    // 4 lanes hold 8 neighbouring columns of each step i. They exchange, so that lane n stores 16
    // bytes of step n % 4 (d = 64: 8 bytes of step n % 2), and a key's row leaves in one
    // instruction (4-byte stores: 42.6 against 38.5 us for 32768 tokens of 8 heads of 128).
    if constexpr (I == 4) {
      quad_transpose(o, r & 3);
      if (live)
        *reinterpret_cast<uint4*>(vp + (row8 + e) * vs + 32 * (r & 3) + 8 * (r >> 2)) =
            make_uint4(o[0], o[1], o[2], o[3]);
    } else {
      const bool odd = r & 1;
      const uint32_t got = dpp_u(odd ? o[0] : o[1], false);
      if (live)
        *reinterpret_cast<uint2*>(vp + (row8 + e) * vs + 32 * (r & 1) + 2 * (r & 14)) =
            odd ? make_uint2(got, o[1]) : make_uint2(o[0], got);
    }
  }
}

template <int D, int NG>
__global__ __launch_bounds__(NT) void kv4_read_kernel(Kv4Rows a) {
  const int wave = uniform(threadIdx.x >> 6);
  const long long item = (long long)blockIdx.x * (NT / 64) + wave;
  int b, h, blk, row0, rows;
  if (!locate(a, item >> 1, b, h, blk, row0, rows)) return;
  const uint8_t* src = a.cache + b * a.cb + h * a.ch + (long long)blk * kv4_block_bytes(D, NG);
  if (item & 1)
    read_v<D, NG>(src, const_cast<uint16_t*>(a.v) + b * a.vb + h * a.vh, a.vs, row0, rows,
                  threadIdx.x & 63);
  else
    read_k<D, NG>(src, const_cast<uint16_t*>(a.k) + b * a.kb + h * a.kh, a.ks, row0, rows,
                  threadIdx.x & 63);
}

// ---- q/k RMSNorm + RoPE + quantised append: one wavefront per (row, head) ----
// Lane l holds the pair of elements 2 l, 2 l + 1 (d = 64: both halves of the wavefront hold
// the head). Norm and RoPE run in fp32 throughout and q rounds once at the end, to the bf16 that the
// attention's matrix products take; k is quantised from fp32, so no rounding to bf16 moves a value
// over a code's border. 2.8-3.4 us for 1 to 32 rows of 48 heads of 128: a launch's latency.
template <int D, int NG>
__global__ __launch_bounds__(NT) void kv4_append_kernel(
    const uint16_t* __restrict__ qkv, const uint16_t* __restrict__ qw,
    const uint16_t* __restrict__ kw, const uint16_t* __restrict__ cosb,
    const uint16_t* __restrict__ sinb, const int* __restrict__ pos, uint16_t* __restrict__ q_out,
    uint8_t* __restrict__ cache, int M, int T, long long cb, long long ch, float eps, int nq,
    int nkv, int max_pos, const uint16_t* __restrict__ rope) {
  constexpr int HP = D / 64, IPG = D / 32 / NG;
  const int lane = threadIdx.x & 63, l = lane & (D / 2 - 1);
  const int nh = nq + 2 * nkv;
  const long long item = (long long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  if (item >= (long long)M * nh) return;
  const int m = (int)(item / nh), hd = (int)(item - (long long)m * nh);
  const int b = m / T;
  const long long p = (long long)pos[b] + (m - b * T);
  if (p < 0 || p >= max_pos) return;
  const uint32_t x = reinterpret_cast<const uint32_t*>(qkv)[item * (D / 2) + l];
  float x0 = bf16lo(x), x1 = bf16hi(x);
  const bool is_v = hd >= nq + nkv;
  if (!is_v) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(hd < nq ? qw : kw)[l];
    const uint32_t cw = reinterpret_cast<const uint32_t*>(rope ? rope + 2LL * b * D : cosb + p * D)[l];
    const uint32_t sw =
        reinterpret_cast<const uint32_t*>(rope ? rope + (2LL * b + 1) * D : sinb + p * D)[l];
    // 64 lanes add the squares of a head once (d = 128) or twice (d = 64)
    const float rstd = rsqrtf(wave_sum(x0 * x0 + x1 * x1) * (1.0f / 128.0f) + eps);
    const float n0 = x0 * rstd * bf16lo(w), n1 = x1 * rstd * bf16hi(w);
    const float sign = l < D / 4 ? -1.f : 1.f;  // rotate_half: the first half takes -x[d + D/2]
    const float r0 = sign * __shfl_xor(n0, D / 4, 64), r1 = sign * __shfl_xor(n1, D / 4, 64);
    x0 = n0 * bf16lo(cw) + r0 * bf16lo(sw);
    x1 = n1 * bf16hi(cw) + r1 * bf16hi(sw);
    if (hd < nq) {
      if (lane < D / 2)
        reinterpret_cast<uint32_t*>(q_out)[((long long)m * nq + hd) * (D / 2) + l] =
            pack_bf16x2(x0, x1);
      return;
    }
  }
  // 32 values are the 16 lanes of a row, larger groups 2 or 4 rows
  float mn = kv4_min_row16(kv4_min(x0, x1)), mx = kv4_max_row16(kv4_max(x0, x1));
  if (IPG >= 2) kv4_minmax_xor16(mn, mx);
  if (IPG >= 4) kv4_minmax_xor32(mn, mx);
  Kv4Group gr;
  gr.from(mn, mx);
  const uint32_t n0 = gr.code(x0), n1 = gr.code(x1);
  if (lane >= D / 2) return;
  const int i = l >> 4, n = l & 15, key = (int)(p & 31);
  uint8_t* dst = cache + b * cb + (hd - nq - (is_v ? nkv : 0)) * ch +
                 (p >> 5) * kv4_block_bytes(D, NG);
  uint32_t* sc = reinterpret_cast<uint32_t*>(dst + 32 * D) + (is_v ? 32 * NG : 0);
  if (n == 0 && i % IPG == 0) sc[i / IPG * 32 + key] = gr.sc;
  if (is_v) {  // columns 32 i + 2 n, + 1: one byte
    dst[16 * D + ((key / 8 * HP + i / 2) * 16 + n) * 16 + key % 8 * 2 + (i & 1)] =
        (uint8_t)(n0 | n1 << 4);
  } else {  // values e = 2 (n % 4), + 1 of the dword of lane group n / 4: four lanes make it
    uint32_t w = n0 << (4 * (n & 3)) | n1 << (4 * (n & 3) + 16);
    w |= __shfl_xor(w, 1, 64);
    w |= __shfl_xor(w, 2, 64);
    if ((n & 3) == 0) *reinterpret_cast<uint32_t*>(dst + key * (D / 2) + n / 4 * (D / 8) + 4 * i) = w;
  }
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int rows_args(Kv4Rows& a, const void* k, long long kb, long long kh, long long ks, const void* v,
              long long vb, long long vh, long long vs, const void* cache, long long cb,
              long long ch, const int* start, const int* lengths, int B, int S, int nkv, int cap,
              int d, int group) {
  if (!k || !v || !cache || B < 1 || S < 1 || nkv < 1 || cap < 1) return KO_EINVAL;
  if (!kv4_served(d, group)) return KO_ENOTSUP;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(cache, 16) || (cb & 15) || (ch & 15))
    return KO_EINVAL;
  if ((kb & 7) || (kh & 7) || (ks & 7) || (vb & 7) || (vh & 7) || (vs & 7)) return KO_EINVAL;
  // blocks that S rows can touch from any first slot; a launch has less than 2^32 threads
  const long long nb = ((long long)S + 31) / 32 + (start ? 1 : 0);
  if ((long long)B * nkv > KV4_MAX_WAVES / 2 / nb) return KO_ERANGE;
  a = {static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), kb, kh, ks, vb, vh, vs,
       static_cast<uint8_t*>(const_cast<void*>(cache)), cb, ch, start, lengths, B, S, nkv, cap,
       (int)nb};
  return KO_OK;
}

}  // namespace

extern "C" {

int ko_kv4_write(const void* k, long long k_b_stride, long long k_h_stride, long long k_s_stride,
                 const void* v, long long v_b_stride, long long v_h_stride, long long v_s_stride,
                 void* cache, long long cache_b_stride, long long cache_h_stride, const int* start,
                 const int* lengths, int B, int S, int nkv, int cap, int d, int group,
                 void* stream) {
  Kv4Rows a;
  const int st = rows_args(a, k, k_b_stride, k_h_stride, k_s_stride, v, v_b_stride, v_h_stride,
                           v_s_stride, cache, cache_b_stride, cache_h_stride, start, lengths, B, S,
                           nkv, cap, d, group);
  if (st) return st;
  const dim3 grid((unsigned)((2LL * B * nkv * a.nb + 3) / 4)), block(NT);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define CALL(D_, NG_) hipLaunchKernelGGL((kv4_write_kernel<D_, NG_>), grid, block, 0, s, a);
  KV4_PICK(d, group, CALL)
#undef CALL
  return KO_LAUNCH_STATUS();
}

int ko_kv4_read(const void* cache, long long cache_b_stride, long long cache_h_stride, void* k,
                long long k_b_stride, long long k_h_stride, long long k_s_stride, void* v,
                long long v_b_stride, long long v_h_stride, long long v_s_stride, const int* start,
                const int* lengths, int B, int S, int nkv, int cap, int d, int group,
                void* stream) {
  Kv4Rows a;
  const int st = rows_args(a, k, k_b_stride, k_h_stride, k_s_stride, v, v_b_stride, v_h_stride,
                           v_s_stride, cache, cache_b_stride, cache_h_stride, start, lengths, B, S,
                           nkv, cap, d, group);
  if (st) return st;
  const dim3 grid((unsigned)((2LL * B * nkv * a.nb + 3) / 4)), block(NT);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define CALL(D_, NG_) hipLaunchKernelGGL((kv4_read_kernel<D_, NG_>), grid, block, 0, s, a);
  KV4_PICK(d, group, CALL)
#undef CALL
  return KO_LAUNCH_STATUS();
}

int ko_kv4_append(const void* qkv, const void* q_w, const void* k_w, const void* cos,
                  const void* sin, const int* pos, void* q_out, void* cache, int M, int T,
                  long long cache_b_stride, long long cache_h_stride, float eps, int nq, int nkv,
                  int d, int group, int max_pos, const void* rope, void* stream) {
  if (!qkv || !q_w || !k_w || !cos || !sin || !pos || !q_out || !cache) return KO_EINVAL;
  if (M < 1 || T < 1 || M % T || nq < 1 || nkv < 1 || max_pos < 1) return KO_EINVAL;
  if (rope && (T != 1 || !aligned(rope, 16))) return KO_EINVAL;
  if (!kv4_served(d, group)) return KO_ENOTSUP;
  if (!aligned(qkv, 16) || !aligned(q_w, 16) || !aligned(k_w, 16) || !aligned(cos, 16) ||
      !aligned(sin, 16) || !aligned(q_out, 16) || !aligned(cache, 16) || (cache_b_stride & 15) ||
      (cache_h_stride & 15))
    return KO_EINVAL;
  const long long items = (long long)M * (nq + 2LL * nkv);
  if (items > KV4_MAX_WAVES) return KO_ERANGE;
  const dim3 grid((unsigned)((items + 3) / 4)), block(NT);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define CALL(D_, NG_)                                                                          \
  hipLaunchKernelGGL((kv4_append_kernel<D_, NG_>), grid, block, 0, s,                          \
                     static_cast<const uint16_t*>(qkv), static_cast<const uint16_t*>(q_w),     \
                     static_cast<const uint16_t*>(k_w), static_cast<const uint16_t*>(cos),     \
                     static_cast<const uint16_t*>(sin), pos, static_cast<uint16_t*>(q_out),    \
                     static_cast<uint8_t*>(cache), M, T, cache_b_stride, cache_h_stride, eps,  \
                     nq, nkv, max_pos, static_cast<const uint16_t*>(rope));
  KV4_PICK(d, group, CALL)
#undef CALL
  return KO_LAUNCH_STATUS();
}

}  // extern "C"
