// Decode attention over the 4-bit KV cache (kv4_core.h), for gfx950.
//
// Query row (t, h) of sequence b and KV head j, t of T tokens, sees the keys below len - T + t + 1:
//   score_k = scale sum_g (s_kg sum_{d in g} q_d (n_kd - 8) + c_kg sum_{d in g} q_d)
//   out_d   = sum_k p_k (c_kg + s_kg (n_kd - 8)) / sum_k p_k,  p_k = exp(score_k - max)
// A row that sees no key is zero. Bound by the bytes of the cache, as long as no more than about
// three VALU operations fall on a value; so no value is dequantised:
//
// - The codes go to the matrix cores as bf16 128 + n: four bits and a constant, one shift and one
//   bit operation for two values. 16x16x32 products run over d for the scores and over the
//   keys for the output, 32 keys (one block of the cache) a step.
// - Scores: A is K (rows = keys), B is q (columns). A group's scale applies to its part of the
//   sum, so a column is a (query row, group) pair: q with zeros outside the group. GPT groups
//   share a 16-column tile, 16 / GPT query rows each; one tile holds the 4 heads x 4 groups of
//   a decode step, and with 16 rows every tile has a group to itself and runs over its d
//   alone. The tile starts from -136 sum q, so it ends as sum q (n - 8); the lane then adds s
//   times that and c sum q, and sums over the GPT neighbouring lanes of a row.
// - The result leaves each lane with 8 consecutive keys of one column, which is the A operand
//   of the product over keys: p s goes from registers into the matrix cores, no exchange. p s is
//   rounded to bf16, the type that the matrix cores take (up to 2^-8 of each term; the terms add
//   up, their roundings do not: 0.0023 of the output in 2-norm against 0.0017 for its own rounding
//   alone), as P is over the bf16 cache; p and sum p c stay fp32.
// - Output: B is V, a tile of 16 columns of one group. The offset leaves with the constant -136
//   in a product of its own, before the codes' product: what accumulates is sum p s (n - 8), as
//   small as the result, and not 136 sum p s, whose roundings would grow with the length.
//
// Work: the steps of all (sequence, KV head) pairs are dealt out from the lengths, on the device, to
// two workgroups of 4 wavefronts on a CU or one of 8: each pair cut into parts of equal runs where
// the workgroups suffice, else one list of all steps, cut into equal runs. The wavefronts take the
// steps of a run in turn, each with two blocks in flight. A pair within one run writes its output;
// else the workgroup that finishes the pair last merges the partial sums (fp32, in run order:
// the result does not depend on who is last).
//
// Measured, 32 query and 8 KV heads of 128 in groups of 32: 16 x 8192 keys (168 MB) 31.5-33.2 us, 16 x
// 32768 108-111 us (6.0-6.2 TB/s; the bf16 cache's attention reads at 6.6), 512 keys 7.1-7.4 us. Per
// step and wavefront 297 VALU instructions with up to 4 query rows, 381 with 16, of about 4
// cycles: two wavefronts on a SIMD keep ahead of the HBM with one query token, not with 4 and more
// (16 x 8192 keys, 5 tokens: 59-62 us). With groups of 32 of 128 and more than 8 query rows 8 to 11
// registers spill, stored ahead of the loop over pairs and read outside that over steps.
#include "kv4_core.h"

#include <limits.h>

#include <type_traits>

using namespace ko;

extern "C" int ko_kv4_append(const void* qkv, const void* q_w, const void* k_w, const void* cos,
                             const void* sin, const int* pos, void* q_out, void* cache, int M, int T,
                             long long cache_b_stride, long long cache_h_stride, float eps, int nq,
                             int nkv, int d, int group, int max_pos, const void* rope,
                             void* stream);

namespace {

constexpr float TAU = 8.0f;            // a running maximum is raised by more than 2^8 only
constexpr float NEG_BIG = -1.0e30f;    // a key whose q k lies below counts for nothing
// Up to SOLO steps a pair is not cut: its 5 steps a wavefront take less than the partial sums'
// way through memory (one sequence of 512 keys 6.7 against 8.0 us in two parts; 1000 keys 9.8
// against 8.6 us in four).
constexpr int SOLO = 20;
// What a pair costs beside its steps, about 3 us, in steps of a workgroup of 4 or 8 wavefronts.
__host__ __device__ constexpr int pair_steps(int waves) { return 3 * waves; }

struct Kv4AttnArgs {
  const uint16_t* q;  // [B*T, nq*D]
  const uint8_t* cache;
  long long cb, ch;  // bytes
  const int* lens;
  int len_off, cap, B, T, nkv, G, min_run;
  float inv_nkv;
  float scale_log2;
  float* part;    // [2 * grid][rows][D], then [2 * grid][rows][2]
  int* counters;  // [grid], zero; left zero
  uint16_t* out;
  long long most;  // a sequence of more keys has none
};

// A sequence's length. One that passes the cache's end still says where its query tokens are, as
// far as cap + T - 1, where all of them see every key.
__device__ __forceinline__ int seq_len(const Kv4AttnArgs& a, int b) {
  const long long n = (long long)a.lens[b] + a.len_off, last = a.cap + a.T - 1;
  return (int)(n < 0 || n > a.most ? 0 : n < last ? n : last);
}
__device__ __forceinline__ int steps_of(const Kv4AttnArgs& a, int len) {
  return len > 0 ? (min(len, a.cap) + 31) >> 5 : 1;
}

// The lane's thread index, opaque: what follows from it is computed where it is used, not
// ahead of the loop over the pairs, where it would take registers from the steps.
__device__ __forceinline__ int fresh_tid() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// a / b for 0 <= a < 2^24, 0 < b, with 1 / b as fp32 has it: two estimates and one correction,
// a third of the instructions of a 32-bit division; in front of a wavefront's first load.
__device__ __forceinline__ int quot(int a, int b, float inv) {
  int q = (int)((float)a * inv);
  int rem = a - q * b;
  const int more = (int)((float)rem * inv);
  q += more;
  rem -= more * b;
  return q + (rem >= b ? 1 : 0) - (rem < 0 ? 1 : 0);
}

// Sum over the n neighbouring lanes (1, 2, 4) that hold a row's groups.
template <int N>
__device__ __forceinline__ float sum_lanes(float v) {
  if (N >= 2) v += dpp_f<0xB1>(v);  // quad_perm [1, 0, 3, 2]
  if (N >= 4) v += dpp_f<0x4E>(v);  // quad_perm [2, 3, 0, 1]
  return v;
}

// Two codes from the 4 bits at k of each half of w: bf16 128 + n each. mask and bias are 0x000f000f
// and 0x43004300 in registers whose values the compiler does not know: one v_and_or_b32, where
// two literals would make it two instructions.
struct Codes {
  uint32_t mask = 0x000f000fu, bias = 0x43004300u;
  __device__ __forceinline__ Codes() { asm("" : "+s"(mask), "+v"(bias)); }
  __device__ __forceinline__ uint32_t operator()(uint32_t w, int k) const {
    return ((w >> k) & mask) | bias;
  }
};

__device__ __forceinline__ f32x4 mfma(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, make_uint4(a[0], a[1], a[2], a[3])),
      __builtin_bit_cast(bf16x8, make_uint4(b[0], b[1], b[2], b[3])), c, 0, 0, 0);
}

__device__ __forceinline__ void store2_coherent(float* p, float x, float y) {
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p),
                     __builtin_bit_cast(unsigned long long, make_float2(x, y)), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load2_coherent(const float* p) {
  return __builtin_bit_cast(
      float2, __hip_atomic_load(reinterpret_cast<unsigned long long*>(const_cast<float*>(p)),
                                __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

__device__ __forceinline__ uint2 ldg8(const void* p) {
  typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 v = __builtin_nontemporal_load((const __attribute__((address_space(1))) u32x2*)p);
  return make_uint2(v.x, v.y);
}

// A block's bytes as one lane holds them.
template <int D, int NG>
struct Block {
  uint32_t k[2][D / 32];   // K: keys 8 (r / 4) + r % 4 (+ 4), D / 8 bytes from lane group kg
  uint32_t v[D / 64][4];   // V: planes, keys 8 kg .. + 7 in pairs
  uint32_t sc[NG];         // NG of the 64 NG scale dwords
  __device__ __forceinline__ void load_k(const uint8_t* p, int r, int kg, int lane) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint8_t* kp = p + (8 * (r >> 2) + (r & 3) + 4 * c) * (D / 2) + kg * (D / 8);
      if constexpr (D == 128) {
        const uint4 x = ldg16_stream(kp);
        k[c][0] = x.x, k[c][1] = x.y, k[c][2] = x.z, k[c][3] = x.w;
      } else {
        const uint2 x = ldg8(kp);
        k[c][0] = x.x, k[c][1] = x.y;
      }
    }
    const uint8_t* s = p + 32 * D + 4 * NG * lane;
    if constexpr (NG == 4) {
      const uint4 x = ldg16_stream(s);
      sc[0] = x.x, sc[1] = x.y, sc[2] = x.z, sc[3] = x.w;
    } else if constexpr (NG == 2) {
      const uint2 x = ldg8(s);
      sc[0] = x.x, sc[1] = x.y;
    } else {
      sc[0] = *reinterpret_cast<const uint32_t*>(s);
    }
  }
  __device__ __forceinline__ void load_v(const uint8_t* p, int r, int kg) {
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      const uint4 x = ldg16_stream(p + 16 * D + ((kg * (D / 64) + h) * 16 + r) * 16);
      v[h][0] = x.x, v[h][1] = x.y, v[h][2] = x.z, v[h][3] = x.w;
    }
  }
  // The scales to LDS as fp32: s and c of K, then of V, [2][2][NG][32]. Every lane that serves a
  // group reads them there; unpacked once here, not in each of up to 16 lanes (16 sequences of 8192
  // keys, 7 tokens each 68.3 -> 63.4 us, with one token as before).
  __device__ __forceinline__ void scales_to(float* lds, int lane) const {
    const int at = lane * NG, kv = at / (32 * NG), rest = at % (32 * NG);
    float* s = lds + 2 * kv * 32 * NG + rest;
    float* c = s + 32 * NG;
    if constexpr (NG == 4) {
      *reinterpret_cast<float4*>(s) =
          make_float4(bf16lo(sc[0]), bf16lo(sc[1]), bf16lo(sc[2]), bf16lo(sc[3]));
      *reinterpret_cast<float4*>(c) =
          make_float4(bf16hi(sc[0]), bf16hi(sc[1]), bf16hi(sc[2]), bf16hi(sc[3]));
    } else if constexpr (NG == 2) {
      *reinterpret_cast<float2*>(s) = make_float2(bf16lo(sc[0]), bf16lo(sc[1]));
      *reinterpret_cast<float2*>(c) = make_float2(bf16hi(sc[0]), bf16hi(sc[1]));
    } else {
      *s = bf16lo(sc[0]);
      *c = bf16hi(sc[0]);
    }
  }
};

// RB: blocks of 16 query rows (above 1 with GPT = 1): wavefront w serves rows 16 (w % RB) ..,
// and the steps w / RB, w / RB + 4 / RB, ... of a run.
template <int D, int NG, int GPT, int RB, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void kv4_attn_kernel(Kv4AttnArgs a) {
  constexpr int I = D / 32, IPG = I / NG, NT = NG / GPT, RP = 16 / GPT, J = D / 16;
  constexpr int NWP = WAVES / RB, ROWS = RB * RP;
  static_assert(GPT == 1 || RB == 1, "more than 16 rows have a tile a group");
  __shared__ __align__(16) float lds_sc[WAVES][128 * NG];
  __shared__ __align__(16) float lds_o[WAVES][RP][D];
  __shared__ float lds_ml[WAVES][RP][2];
  __shared__ int lds_prev;

  const int wave = uniform(threadIdx.x >> 6), lane0 = threadIdx.x & 63;
  const int rb = wave % RB, wp = wave / RB;
  const int R = a.T * a.G;
  const Codes codes;
  const int grid = gridDim.x, wg = blockIdx.x;

  // ---- which steps this workgroup takes ----
  // Lane b holds the length, steps and places of sequence b of the first 64.
  int my_len = 0, all = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int len = b0 + lane0 < a.B ? seq_len(a, b0 + lane0) : 0;
    if (b0 == 0) my_len = len;
    all += readlane(wave_incl_scan(b0 + lane0 < a.B ? steps_of(a, len) : 0), 63);
  }
  auto up = [](int n) { return (n + NWP - 1) / NWP * NWP; };
  const int share =
      max(a.min_run, quot(all * a.nkv + grid - 1, grid, __builtin_amdgcn_rcpf((float)grid)));
  // (1) Every pair cut into parts of `run` steps, a workgroup for each: with the least run for
  // which the workgroups suffice, if that is at most a half longer than an equal share. One
  // workgroup on each CU goes before two, which take half as long again as one (4 x 2049 keys, 288
  // workgroups of 8 steps 11.0 us, 192 of 12 9.4).
  int run = up(share), my_places = 0, my_incl = 0, total = 0;
  auto parts_of = [&](int r) {
    const int n = steps_of(a, my_len);
    const int parts = n <= SOLO ? 1 : quot(n + r - 1, r, __builtin_amdgcn_rcpf((float)r));
    my_places = lane0 < a.B ? parts : 0;
    my_incl = wave_incl_scan(my_places);
    return (long long)readlane(my_incl, 63) * a.nkv;
  };
  auto least = [&](int lo, int hi, int most) {  // the least run of lo .. hi that needs at most most
    while (lo < hi) {
      const int mid = lo + (hi - lo) / (2 * NWP) * NWP;
      if (parts_of(mid) <= most)
        hi = mid;
      else
        lo = mid + NWP;
    }
    return hi;
  };
  bool whole = false;
  if (a.B <= 64) {
    const int one = WAVES == 4 ? (grid + 1) / 2 : grid;  // workgroups at one on each CU
    const int longer = run + run / 2 / NWP * NWP;
    const long long need = parts_of(run);
    whole = need <= one;
    if (!whole && parts_of(longer) <= one) {
      run = least(run + NWP, longer, one);
      parts_of(run);
      whole = true;
    } else if (!whole && (need <= grid || parts_of(longer) <= grid)) {
      run = need <= grid ? run : least(run + NWP, longer, grid);
      parts_of(run);
      whole = true;
    }
  }
  // (2) Else one list of all pairs' steps, cut into equal runs that cross from pair to pair.
  // Beginning and ending a pair costs as much as pair_steps steps, and takes so many places more
  // (with none: a ragged 64 of up to 16384 keys 136 us; 12 for the pairs shorter than a run 107, for
  // all 105.5; two thirds or twice of it 106 both, a ragged 24 of up to 4600 21.6 and 23.3 for 21.8).
  auto places = [&](int len) { return steps_of(a, len) + pair_steps(WAVES); };
  if (!whole) {
    total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int len = b0 == 0 ? my_len : b0 + lane0 < a.B ? seq_len(a, b0 + lane0) : 0;
      const int st = b0 + lane0 < a.B ? places(len) : 0;
      const int in = wave_incl_scan(st);
      total += readlane(in, 63);
      if (b0 == 0) my_places = st, my_incl = in;
    }
    total *= a.nkv;
    run = up(max(a.min_run, (total + grid - 1) / grid));
  }

  // The part of a pair that a workgroup takes: sequence b of len keys and n steps, KV head, the
  // steps st0 .. st1 - 1; the workgroups w0 .. w1 hold the pair.
  struct Segment {
    int b, len, n, kvh, st0, st1, w0, w1;
  };
  const long long first = whole ? 0 : (long long)wg * run;
  int s = (int)min(first, (long long)total);
  const int end = (int)min(first + run, (long long)total);
  auto find = [&](Segment& g) {  // the next of this workgroup's segments
    while (s < end) {
      const int pair_step = uniform(quot(s, a.nkv, a.inv_nkv));
      g.b = g.len = 0;
      int n = 0, at = 0;
      if (a.B <= 64) {
        g.b = uniform(__popcll(__ballot(my_incl <= pair_step && lane0 < a.B)));
        g.len = readlane(my_len, g.b);
        n = readlane(my_places, g.b);
        at = (readlane(my_incl, g.b) - n) * a.nkv;
      } else {
        int below = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
          const int l = b0 + lane0 < a.B ? seq_len(a, b0 + lane0) : 0;
          const int st = b0 + lane0 < a.B ? places(l) : 0;
          const int incl = wave_incl_scan(st) + below;
          const int k = uniform(__popcll(__ballot(incl <= pair_step && b0 + lane0 < a.B)));
          if (k < min(64, a.B - b0)) {
            g.b = b0 + k;
            g.len = readlane(l, k);
            n = readlane(st, k);
            at = (readlane(incl, k) - n) * a.nkv;
            break;
          }
          below = readlane(incl, 63);
        }
      }
      g.kvh = (s - at) / n;
      at += g.kvh * n;
      g.st0 = s - at;
      s = min(at + n, end);
      g.n = steps_of(a, g.len);  // the places behind them are empty
      g.st1 = min(g.n, s - at);
      g.w0 = at / run;
      g.w1 = (at + g.n - 1) / run;
      if (g.st0 < g.st1) return true;
    }
    return false;
  };
  Segment g;
  if (whole) {
    const int pair_part = quot(wg, a.nkv, a.inv_nkv);
    if (pair_part >= readlane(my_incl, 63)) return;
    g.b = uniform(__popcll(__ballot(my_incl <= pair_part && lane0 < a.B)));
    g.len = readlane(my_len, g.b);
    g.n = steps_of(a, g.len);
    const int parts = readlane(my_places, g.b);
    const int at = wg - (readlane(my_incl, g.b) - parts) * a.nkv;
    g.kvh = uniform(quot(at, parts, __builtin_amdgcn_rcpf((float)parts)));
    const int part = at - g.kvh * parts;
    g.st0 = part * run;
    g.st1 = parts == 1 ? g.n : min(g.n, g.st0 + run);
    g.w0 = wg - part;
    g.w1 = g.w0 + parts - 1;
  } else if (!find(g)) {
    return;
  }
  auto base_of = [&](const Segment& g) { return a.cache + g.b * a.cb + g.kvh * a.ch; };
  auto block_of = [&](const Segment& g, int st) {
    return base_of(g) + (long long)st * kv4_block_bytes(D, NG);
  };
  // The wavefront's steps of a segment: st0 + wp, and every NWP-th from there.
  auto steps_here = [&](const Segment& g) { return (g.st1 - g.st0 - wp + NWP - 1) / NWP; };
  // Its next two blocks. They change places from step to step; an odd step goes first, in x1, so
  // that the rest are pairs (x0, x1) and no register moves. Where there are less than two, the
  // segment's last block is read in their place.
  Block<D, NG> x0, x1;
  auto load_first = [&](const Segment& g) {
    const int l = fresh_tid() & 63, r = l & 15, kg = l >> 4;
    const int odd = steps_here(g) & 1, st = g.st0 + wp;
    const uint8_t* p0 = block_of(g, min(st + odd * NWP, g.st1 - 1));
    const uint8_t* p1 = block_of(g, min(st + (1 - odd) * NWP, g.st1 - 1));
    x0.load_k(p0, r, kg, l);
    x0.load_v(p0, r, kg);
    x1.load_k(p1, r, kg, l);
    x1.load_v(p1, r, kg);
  };

  // Output row rw of a pair.
  auto out_row = [&](int b, int kvh, int rw) {
    const int t = a.T == 1 ? 0 : rw / a.G;
    const long long row = (((long long)b * a.T + t) * a.nkv + kvh) * a.G + (rw - t * a.G);
    return reinterpret_cast<uint32_t*>(a.out + row * D);
  };

  load_first(g);
  for (;;) {
    const int b = g.b, len = g.len, n = g.n, kvh = g.kvh, st0 = g.st0, st1 = g.st1;
    const int lane = fresh_tid() & 63, r = lane & 15, kg = lane >> 4;
    const int hh = r / GPT, gg = r % GPT;
    const int row = min(rb * RP + hh, R - 1);  // rows past R repeat the last; they are not stored
    const int t = a.T == 1 ? 0 : row / a.G, h = row - t * a.G;
    // q: column (row, group): zeros outside the group
    uint32_t q[I][4];
    const uint16_t* qp = a.q + (((long long)b * a.T + t) * a.nkv * a.G + kvh * a.G + h) * D;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const uint4 x = ldg16(qp + 32 * i + 8 * kg);
      const bool mine = i / IPG % GPT == gg;
      q[i][0] = mine ? x.x : 0u, q[i][1] = mine ? x.y : 0u;
      q[i][2] = mine ? x.z : 0u, q[i][3] = mine ? x.w : 0u;
    }
    float cq[NT];  // sum of q over the group of this lane's column in tile u
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      f32x4 c = {0.f, 0.f, 0.f, 0.f};
      const uint32_t one[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
      for (int i = 0; i < I; ++i)
        if (i / IPG / GPT == u) c = mfma(one, q[i], c);
      cq[u] = c[0];
    }
    const float tau = TAU / a.scale_log2;
    const int lim = min(len - a.T + t + 1, a.cap);  // keys that this lane's row sees

    f32x4 acc[J];
#pragma unroll
    for (int j = 0; j < J; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m = NEG_BIG, l = 0.f, pc[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) pc[u] = 0.f;

    // The running maximum m is kept in units of the unscaled scores.
    auto step = [&](Block<D, NG>& x, int st, auto masked_, auto ahead_) {
      constexpr bool masked = decltype(masked_)::value, ahead = decltype(ahead_)::value;
      float* lsc = lds_sc[wave];
      x.scales_to(lsc, lane);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      // ---- scores of keys 8 kg .. + 7 for this lane's row ----
      float sc[8];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        f32x4 raw[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const float z = -136.f * cq[u];
          raw[u] = (f32x4){z, z, z, z};
        }
#pragma unroll
        for (int i = 0; i < I; ++i) {
          uint32_t kx[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) kx[e] = codes(x.k[c][i], 4 * e);
          raw[i / IPG / GPT] = mfma(kx, q[i], raw[i / IPG / GPT]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v;
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            const float* w = lsc + (u * GPT + gg) * 32 + 8 * kg + 4 * c + e;
            v = fmaf(w[32 * NG], cq[u], u == 0 ? 0.f : v);
            v = fmaf(w[0], raw[u][e], v);
          }
          sc[4 * c + e] = sum_lanes<GPT>(v);
        }
      }
      [[maybe_unused]] const uint8_t* next = block_of(g, st + 2 * NWP);
      if constexpr (ahead) x.load_k(next, r, kg, lane);
      const int k0 = st * KV4_KEYS + 8 * kg;
      if constexpr (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[e] = k0 + e < lim ? sc[e] : -INFINITY;
      }
      float mx = sc[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sc[e]);
      if (__ballot(mx > m + tau)) {
        const float mn = fmaxf(m, max_xor32(max_xor16(mx)));
        const float al = __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
        m = mn;
        l *= al;
#pragma unroll
        for (int u = 0; u < NT; ++u) pc[u] *= al;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float ar = __shfl(al, 4 * kg + e, 64);  // accumulator row 4 kg + e
#pragma unroll
          for (int j = 0; j < J; ++j) acc[j][e] *= ar;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // the difference first: in fma(sc, scale, -m scale) the rounding of m scale stays, and
        // passes exp2's range for scores of 2^31 (the fma is at most 1 % faster: 512 keys 7.24 for
        // 7.32 us, 16 x 32768 109.6 for 110.1)
        sc[e] = __builtin_amdgcn_exp2f((sc[e] - m) * a.scale_log2);
        l += sc[e];
      }
      // ---- p s, and sum p c ----
      uint32_t ps[NT][4];
      int seen = lim - k0;
      if constexpr (masked) asm("" : "+v"(seen));  // compared again, not held from the scores on
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const float* w = lsc + 64 * NG + (u * GPT + gg) * 32 + 8 * kg + 2 * e;
          float s0 = w[0], s1 = w[1], c0 = w[32 * NG], c1 = w[32 * NG + 1];
          if constexpr (masked) {  // an unwritten slot's scales may be NaN
            s0 = 2 * e < seen ? s0 : 0.f, c0 = 2 * e < seen ? c0 : 0.f;
            s1 = 2 * e + 1 < seen ? s1 : 0.f, c1 = 2 * e + 1 < seen ? c1 : 0.f;
          }
          pc[u] = fmaf(sc[2 * e], c0, pc[u]);
          pc[u] = fmaf(sc[2 * e + 1], c1, pc[u]);
          ps[u][e] = pack_bf16x2(sc[2 * e] * s0, sc[2 * e + 1] * s1);
        }
      // ---- output ----
      const uint32_t off[4] = {0xc308c308u, 0xc308c308u, 0xc308c308u, 0xc308c308u};  // -136
#pragma unroll
      for (int j = 0; j < J; ++j) acc[j] = mfma(ps[j / 2 / IPG / GPT], off, acc[j]);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t vx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) vx[e] = codes(x.v[j / 4][e], 4 * (j % 4));
        acc[j] = mfma(ps[j / 2 / IPG / GPT], vx, acc[j]);
      }
      if constexpr (ahead) x.load_v(next, r, kg);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };

    // A wavefront's last two steps may be masked: rows that see different numbers of keys, at
    // most 64 apart, and the end of the sequence.
    using Yes = std::true_type;
    using No = std::false_type;
    int st = st0 + wp, left = steps_here(g);
    if (left == 1) {
      step(x1, st, Yes{}, No{});
    } else if (left > 1) {
      if (left & 1) {
        step(x1, st, No{}, Yes{});
        st += NWP;
        --left;
      }
      for (; left > 2; left -= 2, st += 2 * NWP) {
        step(x0, st, No{}, Yes{});
        step(x1, st + NWP, No{}, Yes{});
      }
      step(x0, st, Yes{}, No{});
      step(x1, st + NWP, Yes{}, No{});
    }

    // the next pair's first blocks come while this one's sums are put together
    Segment nx;
    const bool more = find(nx);   // none with (1)
    if (more) load_first(nx);

    // ---- this wavefront's sums to LDS: accumulator row 4 kg + e is column (hh, gg) ----
    const int tid = fresh_tid(), el = tid & 63, er = el & 15, ek = el >> 4;
    l = sum_xor32(sum_xor16(l));
    if (el < 16 && er % GPT == 0) {
      lds_ml[wave][er / GPT][0] = m;
      lds_ml[wave][er / GPT][1] = l;
    }
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const float c = sum_xor32(sum_xor16(pc[u]));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float ce = __shfl(c, 4 * ek + e, 64);
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (j / 2 / IPG / GPT == u) acc[j][e] += ce;
      }
    }
#pragma unroll
    for (int j = 0; j < J; j += 2)
#pragma unroll
      for (int x = 0; x < 4 / GPT; ++x) {
        const int e = x * GPT + j / 2 / IPG % GPT;
        *reinterpret_cast<float2*>(&lds_o[wave][ek * (4 / GPT) + x][16 * j + 2 * er]) =
            make_float2(acc[j][e], acc[j + 1][e]);
      }
    __syncthreads();

    // ---- merge the wavefronts; a whole pair is done, a part goes to the workspace ----
    const int w0 = g.w0, w1 = g.w1;
    const int mine = wg == w0 ? 1 : 0;                     // of this run's two slots
    float* po = a.part + (2LL * wg + mine) * ROWS * D;
    float* pm = a.part + 2LL * grid * ROWS * D + (2LL * wg + mine) * ROWS * 2;
    for (int x = tid; x < R * (D / 2); x += 64 * WAVES) {
      const int rw = x / (D / 2), c2 = x - rw * (D / 2);
      float M = NEG_BIG, L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
      for (int k = 0; k < NWP; ++k) M = fmaxf(M, lds_ml[rw / RP + RB * k][rw % RP][0]);
#pragma unroll
      for (int k = 0; k < NWP; ++k) {
        const int w = rw / RP + RB * k;
        const float f = __builtin_amdgcn_exp2f((lds_ml[w][rw % RP][0] - M) * a.scale_log2);
        const float2 o = *reinterpret_cast<const float2*>(&lds_o[w][rw % RP][2 * c2]);
        L = fmaf(f, lds_ml[w][rw % RP][1], L);
        o0 = fmaf(f, o.x, o0);
        o1 = fmaf(f, o.y, o1);
      }
      if (w0 == w1) {
        out_row(b, kvh, rw)[c2] = L == 0.f ? 0u : pack_bf16x2(o0 / L, o1 / L);
      } else {
        store2_coherent(po + rw * D + 2 * c2, o0, o1);
        if (c2 == 0) store2_coherent(pm + rw * 2, M, L);
      }
    }
    if (w0 != w1) {
      // the stores are performed at the device's coherence point before the run is counted
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      if (tid == 0)
        lds_prev = __hip_atomic_fetch_add(a.counters + w0, 1, __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (lds_prev == w1 - w0) {  // the last of the pair's runs to be counted merges them
        if (tid == 0)
          __hip_atomic_store(a.counters + w0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int parts = w1 - w0 + 1, c2 = el & (D / 2 - 1);
        // slots of the pair's parts: the first run's second, then every run's first
        auto slot_of = [&](int k) { return k == 0 ? 2 * w0 + 1 : 2 * (w0 + k); };
        const float* ml = a.part + 2LL * grid * ROWS * D;
        // A wavefront takes KR rows and a batch of parts at a time, their loads in flight together,
        // the first with those of (m, l). All of a batch's loads are made, and coherent loads cost, so
        // it is not much larger than the parts there are: with one row 4 to 32 (32 always: 4 x 2049
        // keys, 8 parts, 9.9 against 9.2 us, 16 x 8192 33.7 and 32.3); with 2 and 4 rows 8 kB,
        // of one size (16 kB: 4 x 7 tokens 18.7 against 17.8, 4 x 2048 keys with 2 9.8 and 9.2; in
        // three sizes 18.5, and a kernel of 20 heads of 64 5 % slower).
        constexpr int KR = ROWS >= 16 ? 4 : ROWS / 4;
        for (int rw0 = wave; rw0 < R; rw0 += WAVES * KR) {
          float M[KR], L[KR], o0[KR], o1[KR], f[KR];
          int rw[KR];
#pragma unroll
          for (int k = 0; k < KR; ++k) {
            rw[k] = min(rw0 + WAVES * k, R - 1);
            M[k] = NEG_BIG, L[k] = o0[k] = o1[k] = 0.f;
          }
          for (int p0 = 0; p0 < parts; p0 += 64) {
            const int np = min(64, parts - p0);
            float2 x[KR];
#pragma unroll
            for (int k = 0; k < KR; ++k)
              x[k] = el < np ? load2_coherent(ml + ((long long)slot_of(p0 + el) * ROWS + rw[k]) * 2)
                             : make_float2(NEG_BIG, 0.f);
            auto batch = [&](int q0, auto size) __attribute__((always_inline)) {
              constexpr int PB = decltype(size)::value;
              float2 o[KR][PB];
#pragma unroll
              for (int q = 0; q < PB; ++q) {
                // past the last part its loads are repeated: no branch between the loads,
                // which would make each wait for the one before
                const int part = min(p0 + q0 + q, parts - 1);
                const float* src = a.part + (long long)slot_of(part) * ROWS * D + 2 * c2;
#pragma unroll
                for (int k = 0; k < KR; ++k) o[k][q] = load2_coherent(src + rw[k] * D);
              }
              if (q0 == 0) {
#pragma unroll
                for (int k = 0; k < KR; ++k) {
                  const float Mn = fmaxf(M[k], wave_max(x[k].x));
                  const float old = __builtin_amdgcn_exp2f((M[k] - Mn) * a.scale_log2);
                  f[k] = __builtin_amdgcn_exp2f((x[k].x - Mn) * a.scale_log2);
                  L[k] = fmaf(L[k], old, wave_sum(f[k] * x[k].y));
                  o0[k] *= old;
                  o1[k] *= old;
                  M[k] = Mn;
                }
              }
#pragma unroll
              for (int q = 0; q < PB; ++q)
                if (q0 + q < np) {
#pragma unroll
                  for (int k = 0; k < KR; ++k) {
                    const float fq = readlane(f[k], q0 + q);
                    o0[k] = fmaf(fq, o[k][q].x, o0[k]);
                    o1[k] = fmaf(fq, o[k][q].y, o1[k]);
                  }
                }
              return q0 + PB;
            };
            for (int q0 = 0; q0 < np;) {
              [[maybe_unused]] const int left = np - q0;
              if constexpr (KR == 1)
                q0 = left > 16  ? batch(q0, std::integral_constant<int, 32>{})
                     : left > 8 ? batch(q0, std::integral_constant<int, 16>{})
                     : left > 4 ? batch(q0, std::integral_constant<int, 8>{})
                                : batch(q0, std::integral_constant<int, 4>{});
              else
                q0 = batch(q0, std::integral_constant<int, 2048 / D / KR>{});
            }
          }
#pragma unroll
          for (int k = 0; k < KR; ++k)
            if (el < D / 2 && rw0 + WAVES * k < R)
              out_row(b, kvh, rw[k])[c2] =
                  L[k] == 0.f ? 0u : pack_bf16x2(o0[k] / L[k], o1[k] / L[k]);
        }
      }
    }
    if (!more) break;
    __syncthreads();  // the next pair's sums reuse the LDS
    g = nx;
  }
}

// Query rows a workgroup holds: groups that share a tile (GPT) and blocks of 16 rows (RB).
int tile_groups(int rows, int ng) {
  return rows <= 4 && ng == 4 ? 4 : rows <= 8 && ng >= 2 ? 2 : 1;
}
int row_blocks(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Wavefronts of a workgroup (two of 4 or one of 8 fill a CU's registers): 8 where blocks of 16
// query rows share each step (4 x 7 tokens of ragged sequences 24.0 -> 18.7 us), and where there
// is a workgroup of 8 for each pair, as 129 to 256 pairs have it: pairs of one length then need
// no merge (32 x 2048 keys 20.9 -> 17.5 us; a ragged 32 23.7 -> 25.0). Fewer pairs are cut either
// way (16 x 8192 33.3 and 32.4 us, 4 x 2048 9.0 and 9.2), more take a CU's two workgroups
// (ragged 64 109 and 119 us).
int waves_for(int rb, long long pairs) { return rb > 1 || (pairs > 128 && pairs <= 256) ? 8 : 4; }

template <int D, int NG>
int launch(const Kv4AttnArgs& a, int grid, hipStream_t s) {
  const int rows = a.T * a.G;
  const int gpt = tile_groups(rows, NG), rb = row_blocks(rows);
  const int waves = waves_for(rb, (long long)a.B * a.nkv);
  const dim3 g(waves == 8 ? (grid + 1) / 2 : grid), blk(64 * waves);
#define KV4_LAUNCH(GPT_, RB_, WAVES_)                                                       \
  {                                                                                         \
    hipLaunchKernelGGL((kv4_attn_kernel<D, NG, GPT_, RB_, WAVES_>), g, blk, 0, s, a);       \
    return KO_LAUNCH_STATUS();                                                              \
  }
  if constexpr (NG == 4)
    if (gpt == 4) {
      if (waves == 8) KV4_LAUNCH(4, 1, 8)
      KV4_LAUNCH(4, 1, 4)
    }
  if constexpr (NG >= 2)
    if (gpt == 2) {
      if (waves == 8) KV4_LAUNCH(2, 1, 8)
      KV4_LAUNCH(2, 1, 4)
    }
  if (rb == 2) KV4_LAUNCH(1, 2, 8)
  if (rb == 4) KV4_LAUNCH(1, 4, 8)
  if (waves == 8) KV4_LAUNCH(1, 1, 8)
  KV4_LAUNCH(1, 1, 4)
#undef KV4_LAUNCH
}

long long scratch_floats(int rows, int d, int group, int grid) {
  if (rows < 1 || rows > 64 || !kv4_served(d, group) || grid < 1) return -1;
  const int held = row_blocks(rows) * 16 / tile_groups(rows, d / group);
  return 2LL * grid * held * (d + 2);
}

// What the two entry points check alike.
int check(const void* q, const void* cache, long long cb, long long ch, const int* lens, int cap,
          int B, int T, int nq, int nkv, int d, int group, float scale, const float* part,
          long long part_len, const int* counters, int grid, int min_run, const void* out) {
  if (!q || !cache || !lens || !out || !part || !counters || B < 1 || T < 1 || nkv < 1 || nq < 1 ||
      cap < 1 || grid < 1 || min_run < 1)
    return KO_EINVAL;
  if (!(scale > 0.f && scale < 1.0e4f)) return KO_EINVAL;
  if (!kv4_served(d, group) || nq % nkv || T > 64 || T * (long long)(nq / nkv) > 64)
    return KO_ENOTSUP;
  if (!aligned16(q) || !aligned16(cache) || !aligned16(out) || (cb & 15) || (ch & 15) ||
      (reinterpret_cast<uintptr_t>(part) & 7))
    return KO_EINVAL;
  if (part_len < scratch_floats(T * (nq / nkv), d, group, grid)) return KO_ERANGE;
  // the places of the list, and what is divided, stay below 2^24 (quot)
  const long long blocks = ((long long)cap + 31) / 32;
  if (grid > (1 << 20) || min_run > (1 << 20) ||
      (long long)B * nkv > ((1LL << 24) - grid - min_run) / (blocks + pair_steps(8)))
    return KO_ERANGE;
  return KO_OK;
}

int attention(const void* q, const void* cache, long long cb, long long ch, const int* lens,
              int len_off, int cap, long long most, int B, int T, int nq, int nkv, int d, int group,
              float scale, float* part, long long part_len, int* counters, int grid, int min_run,
              void* out, void* stream) {
  const int st = check(q, cache, cb, ch, lens, cap, B, T, nq, nkv, d, group, scale, part, part_len,
                       counters, grid, min_run, out);
  if (st) return st;
  const Kv4AttnArgs a = {static_cast<const uint16_t*>(q), static_cast<const uint8_t*>(cache), cb, ch,
                         lens, len_off, cap, B, T, nkv, nq / nkv, min_run, 1.0f / nkv,
                         scale * 1.4426950408889634f, part, counters, static_cast<uint16_t*>(out),
                         most};
  hipStream_t s = static_cast<hipStream_t>(stream);
#define CALL(D_, NG_) return launch<D_, NG_>(a, grid, s);
  KV4_PICK(d, group, CALL)
#undef CALL
  return KO_ENOTSUP;
}

}  // namespace

extern "C" {

long long ko_kv4_attn_scratch(int rows, int d, int group, int grid) {
  return scratch_floats(rows, d, group, grid);
}

int ko_kv4_attn(const void* q, const void* cache, long long cache_b_stride,
                long long cache_h_stride, const int* kv_lens, int len_offset, int cap, int B,
                int T, int nq, int nkv, int d, int group, float scale, float* part,
                long long part_len, int* counters, int grid, int min_run, void* out,
                void* stream) {
  return attention(q, cache, cache_b_stride, cache_h_stride, kv_lens, len_offset, cap, LLONG_MAX, B,
                   T, nq, nkv, d, group, scale, part, part_len, counters, grid, min_run, out, stream);
}

int ko_kv4_attn_qkv(const void* qkv, const void* q_w, const void* k_w, const void* cos,
                    const void* sin, int max_pos, const int* pos, void* cache,
                    long long cache_b_stride, long long cache_h_stride, int cap, int B, int nq,
                    int nkv, int d, int group, float eps, float scale, void* q, float* part,
                    long long part_len, int* counters, int grid, int min_run, void* out,
                    const void* rope, void* stream) {
  const int st = check(q, cache, cache_b_stride, cache_h_stride, pos, cap, B, 1, nq, nkv, d, group,
                       scale, part, part_len, counters, grid, min_run, out);
  if (st) return st;
  const int limit = cap < max_pos ? cap : max_pos;
  const int ap = ko_kv4_append(qkv, q_w, k_w, cos, sin, pos, q, cache, B, 1, cache_b_stride,
                               cache_h_stride, eps, nq, nkv, d, group, limit, rope, stream);
  if (ap) return ap;
  return attention(q, cache, cache_b_stride, cache_h_stride, pos, 1, cap, limit, B, 1, nq, nkv, d,
                   group, scale, part, part_len, counters, grid, min_run, out, stream);
}

}  // extern "C"
