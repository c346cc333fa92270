// One token for each row of logits by temperature, top-k, top-p and min-p from given random numbers.
//
// With the row's tokens in order of falling logit (ties: the lowest index first), every filter
// keeps a beginning of the order, and the drawn token is where the running mass passes u times
// the kept mass: all four are places in one order, found by count or by mass, and no sort of the row
// is needed. Masses are whole numbers, W = rint(2^42 exp((x - max) / T)) from an exp in 64
// bits: sums of up to 2^20 of them are exact in 64 bits in any order, so atomics and splits of a row do
// not show in the result. A token of probability below 2^-43 of the largest has mass 0.
//
// Three launches, the first two of which cut a row into chunks, as does the third:
// - maxima: the largest logit of each chunk of a row and its first index (greedy rows end here).
// - bins: tokens by z = (max - x) log2(e) / T in 2048 bins over 44 octaves, masses (a row with a small
//   top-k counts only: no exp for its whole vocabulary) in LDS, then added to the row's in memory. A
//   row's last workgroup forms running sums over the bins, which give the bins in which the cuts and
//   the drawn token can lie: a cut moves the places behind it by no more than its bin's mass.
// - draw: the tokens of these bins, of all chunks, meet in one list, in which a row's last workgroup
//   narrows the exact places down, 8 bits of (logit, index) at a time. Where the list is too long for
//   LDS, more than 2048 tokens, it does the same over the whole row, alone: thousands of equal
//   logits, or flat distributions. A bin is 0.015 T wide, so normal logits of deviation s over 151,936
//   tokens come to it from T = 2.3 s on, earlier with several filters. One row then takes 0.40 to
//   0.47 ms, with top-p 0.65 to 0.84, with top-k past 1024 besides 0.80 to 1.03 (64 rows: 0.62 to
//   0.77, 1.0 to 1.3, 1.1 to 1.5), where it takes 0.026 (0.057) else.
// A row that is one chunk does all of it in one workgroup and one launch.
//
// 64 rows of 151,936 bf16 logits, mixed settings: maxima 6.3 us (3.1 TB/s), bins 30.6 (an exponential
// of 64 bits and an LDS atomic a token, half of whose LDS cycles are conflicts, not the 19 MB; the
// wavefronts wait in 56 % of their cycles), draw 20.6 (the places' passes, one after the other). One
// row, top-k 50: 2.6, 10.1 and 10.7, in chunks of 4096: latency of the trips to memory on which the next
// step depends.
#include "ko_common.h"

namespace {

using namespace ko;

typedef unsigned long long u64;

constexpr int NT = 512, NW = NT / 64;
constexpr int BINS = 2048, CAP = 2048;
constexpr int SHIFT = 42;             // a mass of 1 is 2^42: 2^20 tokens sum below 2^63
constexpr float ZMAX = SHIFT + 2;     // octaves: masses from here on are 0
constexpr float PER_OCTAVE = BINS / ZMAX;
constexpr int K_COUNTED = 1024;       // top-k up to here: counts alone find the kept tokens
constexpr int SPANS = 3;
constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;

// What a row's places need of its bins, as picked from the running sums.
struct Picked {
  u64 best;                   // the row's, as in maxima
  u64 before[SPANS], upto[SPANS];   // the mass before each span of bins, and with it
  u64 all, minp;              // the mass of all tokens, and of those that min_p keeps (not of counted rows)
  uint32_t count[SPANS];      // the count before each
  float hi[SPANS], lo[SPANS];    // the spans' logits, falling; lo > hi: no span
  uint32_t total;             // tokens in the bins
  uint32_t slow;              // counted rows whose k-th token's bin reaches past the list
};

struct Rows {
  const void* x;
  long long stride;
  int V, chunks;
  const float *u, *temperature, *top_p, *min_p;   // a row's settings, or the value beside it
  const int* top_k;
  float temperature1, top_p1, min_p1;
  int top_k1;
  long long* ids;
  float* logp;
  // scratch, [B] each
  u64* best;         // [chunks]: ordered logit << 32 | ~index
  u64* mass;         // [BINS + 1]: the last is min-p's
  u64* list;         // [chunks][CAP]
  Picked* picked;
  uint32_t* count;   // [BINS + 4]: the last are two arrival counters
  uint32_t* found;   // [chunks]: the tokens that a chunk found for the list
};

// Larger floats have larger patterns; -0 is 0. NaN does not come here.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

template <bool F32>
struct Row {
  static constexpr int VE = F32 ? 4 : 8;   // elements of 16 bytes
  const uint8_t* base;                     // the row's first element
  int V, skew, vectors;                    // elements between the 16-byte border below and base

  __device__ Row(const Rows& r, long long b) {
    base = static_cast<const uint8_t*>(r.x) + b * r.stride * (F32 ? 4 : 2);
    V = r.V;
    skew = (int)((reinterpret_cast<uintptr_t>(base) & 15) / (F32 ? 4 : 2));
    vectors = (V + skew + VE - 1) / VE;
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (F32) return reinterpret_cast<const float*>(base)[i];
    else return bf16_to_f32(reinterpret_cast<const uint16_t*>(base)[i]);
  }
  // The vector v, elements v * VE - skew ..; elements outside the row are NaN.
  __device__ __forceinline__ uint4 load(int v) const {
    const int e = v * VE - skew;
    if (e >= 0 && e + VE <= V) return ldg16(base + (long long)e * (F32 ? 4 : 2));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (F32) {
        w[i] = e + i >= 0 && e + i < V ? __float_as_uint(at(e + i)) : 0x7fc00000u;
      } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base);
        const int lo = e + 2 * i, hi = lo + 1;
        w[i] = (lo >= 0 && lo < V ? p[lo] : 0x7fc0u) | (hi >= 0 && hi < V ? p[hi] : 0x7fc0u) << 16;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // f(index, logit) for the elements of the vectors [v0, v1), U loads of a thread at a time; elements
  // outside the row are NaN.
  template <int U, class F>
  __device__ __forceinline__ void each(int v0, int v1, F f) const {
    for (int v = v0 + threadIdx.x; v < v1; v += U * NT) {
      uint4 q[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (v + i * NT < v1) q[i] = load(v + i * NT);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (v + i * NT >= v1) break;
        const int e = (v + i * NT) * VE - skew;
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (F32) {
            f(e + j, __uint_as_float(w[j]));
          } else {
            f(e + 2 * j, bf16lo(w[j]));
            f(e + 2 * j + 1, bf16hi(w[j]));
          }
        }
      }
    }
  }
};

struct Settings {
  float t, p, mp, u;
  int k;
  __device__ Settings(const Rows& r, long long b) {
    t = r.temperature ? r.temperature[b] : r.temperature1;
    k = r.top_k ? r.top_k[b] : r.top_k1;
    p = r.top_p ? r.top_p[b] : r.top_p1;
    mp = r.min_p ? r.min_p[b] : r.min_p1;
    u = r.u[b];
    if (!(mp > 0.f)) mp = 0.f;
    if (!(p < 1.f)) p = 1.f;
    if (k <= 0 || k >= r.V) k = 0;
  }
  // One token is kept whatever the others are (a temperature that is no number: greedy too).
  __device__ bool first() const { return !(t > 0.f) || k == 1 || p <= 0.f; }
  __device__ bool counted() const { return k > 0 && k <= K_COUNTED; }
};

// z of a logit and its mass, from the row's largest.
struct Scale {
  float top, inv;   // inv: of twice the half differences, which cannot overflow
  double invd;
  __device__ Scale(float top_, float t) : top(top_) {
    invd = LOG2E / (double)t;
    inv = fminf((float)(2 * invd), 3.0e38f);
  }
  // Never falls as x falls; -1: a token of mass 0 (a logit of -infinity or NaN among them).
  __device__ __forceinline__ int bin(float x) const {
    if (top == __builtin_huge_valf()) return x == top ? 0 : -1;
    const float z = fmaf(x, -0.5f, 0.5f * top) * inv;   // falls with x, roundings and all
    return z < ZMAX ? min((int)(z * PER_OCTAVE), BINS - 1) : -1;
  }
  __device__ __forceinline__ double octaves(float x) const {
    return x == top ? 0.0 : ((double)top - (double)x) * invd;
  }
  // 2^SHIFT exp((x - top) / T) within 2^-46 of itself: 2^-z = 2^-n exp(-(z - n) ln 2), |z - n| <= 1/2, by
  // the exponential's series (the first term left out, 0.347^12 / 12!, is 2^-47).
  __device__ __forceinline__ double scaled(float x) const {
    const double z = fmin(octaves(x), 2.0 * ZMAX), n = __builtin_rint(z), y = (n - z) * LN2;
    double p = 1.0 / 39916800;
    p = fma(p, y, 1.0 / 3628800);
    p = fma(p, y, 1.0 / 362880);
    p = fma(p, y, 1.0 / 40320);
    p = fma(p, y, 1.0 / 5040);
    p = fma(p, y, 1.0 / 720);
    p = fma(p, y, 1.0 / 120);
    p = fma(p, y, 1.0 / 24);
    p = fma(p, y, 1.0 / 6);
    p = fma(p, y, 0.5);
    p = fma(p, y, 1.0);
    p = fma(p, y, 1.0);
    return __builtin_ldexp(p, SHIFT - (int)n);
  }
  // The nearest whole number of one below 2^52: the last bits of its sum with 2^52.
  static __device__ __forceinline__ u64 whole(double v) {
    return (u64)__double_as_longlong(v + 4503599627370496.0) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 mass(float x) const { return whole(scaled(x)); }
};

struct Shared {
  uint32_t count[BINS];   // of each bin, then running
  u64 mass[BINS];
  u64 part[NW];
  u64 minp;
  int at[2];
  u64 digit_count[256], digit_mass[256], found, found_mass;   // narrow's
};
struct List {
  u64 key[CAP], w[CAP];   // tokens by (falling logit, index), in any order, and their masses
  u64 digit_mass[256];
  uint32_t digit_count[256];
  u64 part[NW];
  u64 found, found_mass;
  uint32_t found_count, found_n, n;
  int at;
};
// Used one after the other.
union Both {
  Shared s;
  List l;
  __device__ Both() {}
};
__device__ __forceinline__ u64 shfl_xor(u64 v, int d) {
  return ((u64)(uint32_t)__shfl_xor((int)(v >> 32), d) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)v, d);
}
// v of the lane n places below in the 16-lane row, 0 where there is none (CTRL: 0x110 + n).
template <int CTRL>
__device__ __forceinline__ u64 row_below(u64 v) {
  return ((u64)(uint32_t)dpp_i<CTRL>((int)(v >> 32)) << 32) | (uint32_t)dpp_i<CTRL>((int)(uint32_t)v);
}
__device__ __forceinline__ u64 readlane64(u64 v, int l) {
  return ((u64)(uint32_t)readlane((int)(v >> 32), l) << 32) | (uint32_t)readlane((int)(uint32_t)v, l);
}
// The sum of v over the wavefront's lanes up to and with this one (all lanes active).
__device__ __forceinline__ u64 wave_running(u64 v) {
  v += row_below<0x111>(v);
  v += row_below<0x112>(v);
  v += row_below<0x114>(v);
  v += row_below<0x118>(v);
  const u64 t0 = readlane64(v, 15), t1 = readlane64(v, 31), t2 = readlane64(v, 47);
  const int row = lane_id() >> 4;
  return v + (row >= 1 ? t0 : 0) + (row >= 2 ? t1 : 0) + (row >= 3 ? t2 : 0);
}

// The sum of v over the threads up to and with this one.
__device__ u64 running(u64 v, u64* part) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  v = wave_running(v);
  __syncthreads();
  if (lane == 63) part[wv] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW - 1; ++i) v += i < wv ? part[i] : 0;
  return v;
}

__device__ u64 block_max(u64 v, u64* part) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = shfl_xor(v, d);
    v = o > v ? o : v;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
  for (int i = 1; i < NW; ++i) v = part[i] > v ? part[i] : v;
  return v;
}

template <bool F32>
__device__ u64 best_of(const Row<F32>& row, int v0, int v1, u64* part) {
  float best = -__builtin_huge_valf();
  int at = -1;   // nothing: no logit is a number above -infinity
  row.template each<4>(v0, v1, [&](int i, float x) {   // a thread's indexes rise
    if (x > best) best = x, at = i;
  });
  return block_max(at < 0 ? 0 : (u64)ordered(best) << 32 | (uint32_t)~at, part);
}

// Counts and masses of the vectors' tokens by bin, into s.
template <bool F32>
__device__ void histogram(const Row<F32>& row, int v0, int v1, const Scale& sc, bool counts,
                          bool masses, float mp, Shared& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) s.count[i] = 0, s.mass[i] = 0;
  if (threadIdx.x == 0) s.minp = 0;
  __syncthreads();
  u64 kept = 0;
  const double least = (double)mp * (double)(1ull << SHIFT);
  row.template each<2>(v0, v1, [&](int, float x) {
    const int b = sc.bin(x);
    if (b < 0) return;
    if (counts) atomicAdd(&s.count[b], 1u);
    if (masses) {
      const double w = sc.scaled(x);
      const u64 m = Scale::whole(w);
      atomicAdd(&s.mass[b], m);
      if (w >= least) kept += m;
    }
  });
  if (masses && mp > 0.f) atomicAdd(&s.minp, kept);
  __syncthreads();
}

// Bins to running sums.
__device__ void accumulate(Shared& s) {
  constexpr int EACH = BINS / NT;
  const int t = threadIdx.x * EACH;
  u64 c = 0, m = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) c += s.count[t + i], m += s.mass[t + i];
  u64 rc = running(c, s.part) - c, rm = running(m, s.part) - m;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    rc += s.count[t + i], rm += s.mass[t + i];
    s.count[t + i] = (uint32_t)rc, s.mass[t + i] = rm;
  }
  __syncthreads();
}

// The first bins at which the running count or mass reaches either target (some bin does).
__device__ int2 bins_of(bool by_count, u64 target0, u64 target1, Shared& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) {
    const u64 here = by_count ? s.count[i] : s.mass[i];
    const u64 before = i ? (by_count ? s.count[i - 1] : s.mass[i - 1]) : 0;
    if (here >= target0 && before < target0) s.at[0] = i;
    if (here >= target1 && before < target1) s.at[1] = i;
  }
  __syncthreads();
  return make_int2(s.at[0], s.at[1]);
}
__device__ int bin_of(bool by_count, u64 target, Shared& s) {
  return bins_of(by_count, target, target, s).x;
}

// u's place in a kept mass, and top-p's in one: 1 and more, at most the mass. Neither falls as the
// mass rises.
__device__ __forceinline__ u64 draw(float u, u64 kept) {
  const double t = (double)u * (double)kept;
  const u64 target = t > 0.0 ? (u64)fmin(t, (double)kept) + 1 : 1;   // u that is no number: 0
  return target < kept ? target : kept;
}
__device__ __forceinline__ u64 nucleus(float p, u64 mass) {
  const double t = ceil((double)p * (double)mass);
  const u64 target = t > 1.0 ? (u64)t : 1;
  return target < mass ? target : mass;
}
__device__ __forceinline__ u64 least_kept(u64 minp) {   // nothing reaches a min_p above 1: the first token
  return minp ? minp : 1ull << SHIFT;
}

// The least (low) or the largest logit of bins [b0, b1]: of all numbers in order, by cutting what is
// left in 65 with a wavefront's 64 lanes.
__device__ float span_end(const Scale& sc, int b0, int b1, bool low) {
  if (!low && b0 == 0) return sc.top;
  // the largest is next to the least of the bins before
  const int limit = low ? b1 : b0 - 1;
  uint32_t lo = ordered(-__builtin_huge_valf()), hi = ordered(sc.top);   // bin(lo) < 0 <= bin(hi) <= limit
  while (hi - lo > 1) {
    const uint32_t step = max((hi - lo) / 65, 1u);
    const uint32_t mid = min(lo + step * (uint32_t)(lane_id() + 1), hi - 1);
    const int b = sc.bin(unordered(mid));
    const u64 in = __ballot(b >= 0 && b <= limit);   // from some lane on
    const int first = in ? __builtin_ctzll(in) : 64;
    const uint32_t below = first ? (uint32_t)readlane((int)mid, first - 1) : lo;
    hi = first < 64 ? (uint32_t)readlane((int)mid, first) : hi;
    lo = below;
  }
  return unordered(low ? hi : hi - 1);
}

// Which bins a row's places can lie in, from running sums in s (counts only if counted).
__device__ void pick(const Settings& st, const Scale& sc, Shared& s, Picked* out) {
  const uint32_t total = s.count[BINS - 1];
  // spans of bins [f, l] for the places of top-k, top-p and the draw, in falling order of bins; l < f: none
  int kf = 1, kl = 0, pf = 1, pl = 0, uf = 1, ul = 0;
  uint32_t slow = 0;
  if (st.counted()) {
    kf = 0, kl = bin_of(true, min((uint32_t)st.k, total), s);
    slow = s.count[kl] > CAP;
  } else {
    u64 lo = s.mass[BINS - 1], hi = lo;   // what the kept mass lies between
    auto within = [&](int f, int l) {
      hi = s.mass[l];
      lo = (f ? s.mass[f - 1] : 0) + 1;
      lo = lo < hi ? lo : hi;
    };
    if (st.k && (uint32_t)st.k < total) {
      kf = kl = bin_of(true, (u64)st.k, s);
      within(kf, kl);
    }
    if (st.p < 1.f) {
      const int2 p = bins_of(false, nucleus(st.p, lo), nucleus(st.p, hi), s);
      pf = p.x, pl = p.y;
      within(pf, pl);
    }
    if (st.mp > 0.f) {
      const u64 m = least_kept(s.minp);
      lo = lo < m ? lo : m, hi = hi < m ? hi : m;
    }
    const int2 u = bins_of(false, draw(st.u, lo), draw(st.u, hi), s);
    uf = u.x, ul = u.y;
    // spans that meet become one: a token is gathered once
    if (pf <= pl && ul >= pf) pf = min(pf, uf), uf = 1, ul = 0;
    if (kf <= kl && pf <= pl && pl >= kf) kf = min(kf, pf), pf = 1, pl = 0;
    if (kf <= kl && uf <= ul && ul >= kf) kf = min(kf, uf), uf = 1, ul = 0;
  }
  const int wv = uniform(threadIdx.x >> 6), j = wv >> 1;   // a wavefront for each end of a span
  if (j < SPANS) {
    const int f = j == 0 ? kf : j == 1 ? pf : uf, l = j == 0 ? kl : j == 1 ? pl : ul;
    const bool low = wv & 1;
    const float end = f <= l ? span_end(sc, f, l, low) : low ? 1.f : 0.f;
    if ((threadIdx.x & 63) == 0) {
      if (low) {
        out->lo[j] = end;
      } else {
        out->hi[j] = end;
        out->before[j] = f <= l && f ? s.mass[f - 1] : 0;
        out->upto[j] = f <= l ? s.mass[l] : 0;
        out->count[j] = f <= l && f ? s.count[f - 1] : 0;
      }
    }
  }
  if (threadIdx.x == 0) out->all = s.mass[BINS - 1], out->minp = s.minp, out->total = total, out->slow = slow;
}

// The row's tokens of the spans among the vectors, into the list of this workgroup.
template <bool F32>
__device__ void gather(const Row<F32>& row, int v0, int v1, const Picked& p, List& l) {
  __syncthreads();
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
  const float h0 = p.hi[0], h1 = p.hi[1], h2 = p.hi[2], l0 = p.lo[0], l1 = p.lo[1], l2 = p.lo[2];
  row.template each<4>(v0, v1, [&](int i, float x) {
    if ((x >= l0 && x <= h0) || (x >= l1 && x <= h1) || (x >= l2 && x <= h2)) {
      const uint32_t at = atomicAdd(&l.n, 1u);
      if (at < CAP) l.key[at] = (u64)~ordered(x) << 32 | (uint32_t)i;
    }
  });
  __syncthreads();
}

__device__ __forceinline__ float logit_of(u64 key) { return unordered(~(uint32_t)(key >> 32)); }

__device__ void result(const Rows& r, long long b, const Scale& sc, u64 key, u64 kept) {
  if (threadIdx.x) return;
  r.ids[b] = (uint32_t)key;
  if (r.logp) {
    const double octaves = sc.octaves(logit_of(key));
    r.logp[b] = (float)(-octaves * LN2 - log((double)kept) + SHIFT * LN2);
  }
}

// The row's token from the list of all the spans' tokens: a place lies in one span, and there 8 bits of
// the key at a time narrow it down, until one token is left. The keys are the lists' without the
// bits that are always the same, and a place begins below those that its span's keys share: atomics on
// one digit that all tokens have would come one after the other.
template <bool F32>
__device__ void finish(const Rows& r, long long b, const Settings& st, const Scale& sc,
                       const Picked& p, List& l, int n) {
  const int ibits = 32 - __builtin_clz((uint32_t)r.V);   // of an index
  auto narrow_key = [&](uint32_t logit_key, uint32_t index) {   // logit_key: ~ordered
    return (u64)(F32 ? logit_key : logit_key >> 16) << ibits | index;
  };
  constexpr int EACH = CAP / NT;
  u64 key[EACH], nkey[EACH], w[EACH], kept_minp = 0;
  int span[EACH];
  const double least = (double)st.mp * (double)(1ull << SHIFT);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = threadIdx.x + i * NT;
    key[i] = at < n ? l.key[at] : ~0ull;
    nkey[i] = narrow_key((uint32_t)(key[i] >> 32), (uint32_t)key[i]);
    const float x = logit_of(key[i]);
    span[i] = at >= n ? -1 : x >= p.lo[0] && x <= p.hi[0] ? 0 : x >= p.lo[1] && x <= p.hi[1] ? 1 : 2;
    const double m = at < n ? sc.scaled(x) : 0.0;
    w[i] = Scale::whole(m);
    if (m >= least) kept_minp += w[i];
  }
  u64 minp = p.minp;
  if (st.counted() && st.mp > 0.f) {   // the list has all that min_p may keep
    const u64 sum = running(kept_minp, l.part);
    if (threadIdx.x == NT - 1) l.found_mass = sum;
    __syncthreads();
    minp = l.found_mass;
    __syncthreads();
  }
  // the token at which the count or the mass reaches target: l.found, l.found_mass
  auto place = [&](bool by_count, u64 target) {
    // its span: the lists of rows that are counted have one
    int j = 0;
    if (!st.counted())
      j = by_count ? 0   // top-k's own span, or the one that it met
          : target > p.before[2] && target <= p.upto[2] ? 2
          : target > p.before[1] && target <= p.upto[1] ? 1 : 0;
    const u64 first = narrow_key(~ordered(p.hi[j]), 0);
    const u64 last = narrow_key(~ordered(p.lo[j]), (1u << ibits) - 1);
    int left = first == last ? 0 : 64 - __builtin_clzll(first ^ last);   // bits not known
    u64 prefix = first >> left, mass = p.before[j];
    uint32_t count = p.count[j];
    while (left > 0) {
      const int shift = max(left - 8, 0);
      __syncthreads();
      if (threadIdx.x < 256) l.digit_mass[threadIdx.x] = 0, l.digit_count[threadIdx.x] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (span[i] == j && nkey[i] >> left == prefix) {
          const int digit = (int)(nkey[i] >> shift) & ((1 << (left - shift)) - 1);
          atomicAdd(&l.digit_count[digit], 1u);
          atomicAdd(&l.digit_mass[digit], w[i]);
        }
      __syncthreads();
      if (threadIdx.x < 64) {   // 4 digits a lane
        u64 m[4], sm = 0;
        uint32_t c[4], sn = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m[i] = l.digit_mass[4 * threadIdx.x + i], c[i] = l.digit_count[4 * threadIdx.x + i];
          sm += m[i], sn += c[i];
        }
        u64 rm = mass + wave_running(sm) - sm;
        uint32_t rc = count + (uint32_t)wave_incl_scan((int)sn) - sn;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u64 before = by_count ? rc : rm, here = before + (by_count ? c[i] : m[i]);
          if (here >= target && before < target)
            l.at = 4 * threadIdx.x + i, l.found_mass = rm, l.found_count = rc, l.found_n = c[i];
          rm += m[i], rc += c[i];
        }
      }
      __syncthreads();
      prefix = prefix << (left - shift) | (u64)l.at;
      left = shift;
      mass = l.found_mass, count = l.found_count;
      if (l.found_n == 1) break;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (span[i] == j && nkey[i] >> left == prefix) l.found = key[i], l.found_mass = mass + w[i];
    __syncthreads();
  };
  u64 kept = p.all;
  if (st.k && ((uint32_t)st.k < p.total || st.counted())) {
    place(true, min((uint32_t)st.k, p.total));
    kept = l.found_mass;
  }
  if (st.p < 1.f) {
    place(false, nucleus(st.p, kept));
    kept = l.found_mass;
  }
  if (st.mp > 0.f) {
    const u64 m = least_kept(minp);
    kept = m < kept ? m : kept;
  }
  place(false, draw(st.u, kept));
  result(r, b, sc, l.found, kept);
}

struct Place {
  u64 key, mass;   // the token, and the mass up to and with it
};

// The first token of the order at which the count or the mass reaches target, over the whole row: its
// bin from the running sums in s, then 8 bits of its key at a time.
template <bool F32>
__device__ Place narrow(const Row<F32>& row, const Scale& sc, bool by_count, u64 target, Shared& s) {
  const int b = bin_of(by_count, target, s);
  u64 prefix = 0, known = 0, count = b ? s.count[b - 1] : 0, mass = b ? s.mass[b - 1] : 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    if (!F32 && (shift == 32 || shift == 40)) {
      // a bf16 logit's lower half is zeros: in the key ones, of a negative logit zeros
      if (!(prefix >> 63)) prefix |= 0xffull << shift;
      known |= 0xffull << shift;
      continue;
    }
    const bool in = threadIdx.x < 256;
    __syncthreads();
    if (in) s.digit_count[threadIdx.x] = s.digit_mass[threadIdx.x] = 0;
    __syncthreads();
    row.template each<2>(0, row.vectors, [&](int i, float x) {
      if (sc.bin(x) != b) return;
      const u64 key = (u64)~ordered(x) << 32 | (uint32_t)i;
      if ((key & known) != prefix) return;
      const int digit = (int)(key >> shift) & 255;
      atomicAdd(&s.digit_count[digit], 1ull);
      atomicAdd(&s.digit_mass[digit], sc.mass(x));
    });
    __syncthreads();
    const u64 c = in ? s.digit_count[threadIdx.x] : 0, m = in ? s.digit_mass[threadIdx.x] : 0;
    const u64 rc = count + running(c, s.part), rm = mass + running(m, s.part);
    const u64 here = by_count ? rc : rm, before = by_count ? rc - c : rm - m;
    if (in && here >= target && before < target)
      s.at[0] = threadIdx.x, s.found = rc - c, s.found_mass = rm - m;
    __syncthreads();
    prefix |= (u64)s.at[0] << shift, known |= 0xffull << shift;
    count = s.found, mass = s.found_mass;
  }
  return {prefix, mass + sc.mass(logit_of(prefix))};
}

// The row's token without a list, by one workgroup.
template <bool F32>
__device__ void finish_slowly(const Rows& r, long long b, const Row<F32>& row, const Settings& st,
                              const Scale& sc, Shared& s) {
  histogram(row, 0, row.vectors, sc, true, true, st.mp, s);
  accumulate(s);
  u64 kept = s.mass[BINS - 1];
  if (st.k && (uint32_t)st.k < s.count[BINS - 1]) kept = narrow(row, sc, true, (u64)st.k, s).mass;
  if (st.p < 1.f) kept = narrow(row, sc, false, nucleus(st.p, kept), s).mass;
  if (st.mp > 0.f) {
    const u64 m = least_kept(s.minp);
    kept = m < kept ? m : kept;
  }
  const Place at = narrow(row, sc, false, draw(st.u, kept), s);
  result(r, b, sc, at.key, kept);
}

// What needs no more than the row's best; true if that was all.
__device__ bool decided(const Rows& r, long long b, const Settings& st, u64 best, bool write) {
  if (best && !st.first()) return false;
  if (write && threadIdx.x == 0) {
    r.ids[b] = best ? (long long)(uint32_t)~(uint32_t)best : -1;
    if (r.logp) r.logp[b] = best ? 0.f : -__builtin_huge_valf();
  }
  return true;
}

template <bool F32>
__global__ __launch_bounds__(NT) void sample_kernel(Rows r) {
  __shared__ Both both;
  __shared__ Picked p;
  Shared& s = both.s;
  List& l = both.l;
  const long long b = blockIdx.x;
  const Row<F32> row(r, b);
  const Settings st(r, b);
  const u64 best = best_of(row, 0, row.vectors, s.part);
  if (decided(r, b, st, best, true)) return;
  const Scale sc(unordered((uint32_t)(best >> 32)), st.t);
  histogram(row, 0, row.vectors, sc, st.k > 0, !st.counted(), st.mp, s);
  accumulate(s);
  pick(st, sc, s, &p);
  __syncthreads();
  if (!p.slow) {
    gather(row, 0, row.vectors, p, l);
    const int n = (int)l.n;
    if (n <= CAP) {
      finish<F32>(r, b, st, sc, p, l, n);
      return;
    }
  }
  finish_slowly(r, b, row, st, sc, s);
}

// The chunk of vectors that workgroup c of a row takes.
template <bool F32>
struct Chunk {
  int v0, v1;
  __device__ Chunk(const Rows& r, const Row<F32>& row) {
    const int per = (row.vectors + r.chunks - 1) / r.chunks, c = blockIdx.x;
    v0 = min(c * per, row.vectors), v1 = min((c + 1) * per, row.vectors);
  }
};

template <bool F32>
__global__ __launch_bounds__(NT) void maxima_kernel(Rows r) {
  __shared__ u64 part[NW];
  const long long b = blockIdx.y;
  const Row<F32> row(r, b);
  const Chunk<F32> c(r, row);
  // the row's bins and counters, for the launches that follow
  for (int i = blockIdx.x * NT + threadIdx.x; i < BINS + 4; i += r.chunks * NT) {
    r.count[b * (BINS + 4) + i] = 0;
    if (i <= BINS) r.mass[b * (BINS + 1) + i] = 0;
  }
  const u64 best = best_of(row, c.v0, c.v1, part);
  if (threadIdx.x == 0) r.best[b * r.chunks + blockIdx.x] = best;
}

// The best of the row's chunks.
__device__ u64 best_of_chunks(const Rows& r, long long b) {
  u64 best = 0;
  for (int i = threadIdx.x & 63; i < r.chunks; i += 64) {
    const u64 o = r.best[b * r.chunks + i];
    best = o > best ? o : best;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = shfl_xor(best, d);
    best = o > best ? o : best;
  }
  return best;
}

// Counts this workgroup in (everything it stored before is performed); true in the row's last.
__device__ bool last_of(uint32_t* counter, int chunks, int* at) {
  __builtin_amdgcn_s_waitcnt(0);   // this thread's stores and atomics
  __syncthreads();
  if (threadIdx.x == 0)
    *at = (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return *at == chunks - 1;
}

// The row's sums of all chunks, into s.
__device__ void load_bins(const Rows& r, long long b, bool counts, bool masses, Shared& s) {
  const u64* mass = r.mass + b * (BINS + 1);
  const uint32_t* count = r.count + b * (BINS + 4);
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) {
    s.count[i] = counts ? __hip_atomic_load(count + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    s.mass[i] = masses ? __hip_atomic_load(mass + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
  }
  if (threadIdx.x == 0) s.minp = __hip_atomic_load(mass + BINS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
}

template <bool F32>
__global__ __launch_bounds__(NT) void bins_kernel(Rows r) {
  __shared__ Shared s;
  const long long b = blockIdx.y;
  const Row<F32> row(r, b);
  const Settings st(r, b);
  const u64 best = best_of_chunks(r, b);
  if (blockIdx.x == 0 && threadIdx.x == 0) r.picked[b].best = best;
  if (decided(r, b, st, best, blockIdx.x == 0)) return;
  const Scale sc(unordered((uint32_t)(best >> 32)), st.t);
  const Chunk<F32> c(r, row);
  const bool counts = st.k > 0, masses = !st.counted();
  histogram(row, c.v0, c.v1, sc, counts, masses, st.mp, s);
  u64* mass = r.mass + b * (BINS + 1);
  uint32_t* count = r.count + b * (BINS + 4);
  for (int i = threadIdx.x; i < BINS; i += NT) {
    if (counts && s.count[i])
      __hip_atomic_fetch_add(count + i, s.count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (masses && s.mass[i])
      __hip_atomic_fetch_add(mass + i, s.mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (threadIdx.x == 0 && s.minp)
    __hip_atomic_fetch_add(mass + BINS, s.minp, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!last_of(count + BINS, r.chunks, s.at)) return;
  load_bins(r, b, counts, masses, s);
  accumulate(s);
  pick(st, sc, s, r.picked + b);
}

template <bool F32>
__global__ __launch_bounds__(NT) void draw_kernel(Rows r) {
  __shared__ Both both;
  __shared__ Picked p;
  __shared__ int s_arrived;
  Shared& s = both.s;
  List& l = both.l;
  const long long b = blockIdx.y;
  const Row<F32> row(r, b);
  const Settings st(r, b);
  if (threadIdx.x < sizeof(Picked) / 4)
    reinterpret_cast<uint32_t*>(&p)[threadIdx.x] = reinterpret_cast<const uint32_t*>(r.picked + b)[threadIdx.x];
  __syncthreads();
  if (decided(r, b, st, p.best, false)) return;
  const Scale sc(unordered((uint32_t)(p.best >> 32)), st.t);
  uint32_t* found = r.found + b * r.chunks;
  u64* list = r.list + b * r.chunks * CAP;
  if (!p.slow) {
    const Chunk<F32> c(r, row);
    gather(row, c.v0, c.v1, p, l);
    u64* mine = list + (long long)blockIdx.x * CAP;
    for (int i = threadIdx.x; i < min((int)l.n, CAP); i += NT)
      __hip_atomic_store(mine + i, l.key[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (threadIdx.x == 0)
      __hip_atomic_store(found + blockIdx.x, l.n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (!last_of(r.count + b * (BINS + 4) + BINS + 1, r.chunks, &s_arrived)) return;
  // the chunks' tokens, one chunk behind the other
  int n = 0;
  if (!p.slow)
    for (int c = 0; c < r.chunks && n <= CAP; c += 64) {
      const int at = c + (int)(threadIdx.x & 63);
      const int m = at < r.chunks ? (int)__hip_atomic_load(found + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
      const int end = n + wave_incl_scan(min(m, CAP + 1)), first = end - min(m, CAP + 1);
      // a wavefront for each chunk in turn
      for (int i = uniform(threadIdx.x >> 6); i < 64 && c + i < r.chunks; i += NW) {
        const int f = readlane(first, i), e = readlane(end, i);
        for (int j = f + (int)(threadIdx.x & 63); j < min(e, CAP); j += 64)
          l.key[j] = __hip_atomic_load(list + (long long)(c + i) * CAP + (j - f), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
      }
      n = readlane(end, 63);
    }
  if (p.slow || n > CAP) {
    finish_slowly(r, b, row, st, sc, s);
    return;
  }
  finish<F32>(r, b, st, sc, p, l, n);
}

}  // namespace

extern "C" {

long long ko_sample_scratch(int B, int chunks) {
  if (B < 1 || chunks < 1 || chunks > 1024) return -1;
  if (chunks == 1) return 0;
  return (long long)B * (8ll * (chunks + BINS + 1) + 8ll * CAP * chunks + sizeof(Picked) +
                         4ll * (BINS + 4 + chunks));
}

int ko_sample(const void* logits, int f32, long long stride, int B, int V, const float* u,
              const float* temperature, float temperature1, const int* top_k, int top_k1,
              const float* top_p, float top_p1, const float* min_p, float min_p1, long long* ids,
              float* logprobs, void* scratch, long long scratch_bytes, int chunks, void* stream) {
  if (!logits || !u || !ids || B < 1 || V < 1 || stride < 0 || chunks < 1) return KO_EINVAL;
  if (V > 1 << 20 || chunks > 1024 || B > 65535) return KO_ERANGE;
  if (reinterpret_cast<uintptr_t>(logits) & (f32 ? 3 : 1)) return KO_EINVAL;
  if (chunks > 1 && (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15) ||
                     scratch_bytes < ko_sample_scratch(B, chunks)))
    return KO_EINVAL;
  Rows r;
  r.x = logits, r.stride = stride, r.V = V, r.chunks = chunks;
  r.u = u, r.temperature = temperature, r.top_p = top_p, r.min_p = min_p, r.top_k = top_k;
  r.temperature1 = temperature1, r.top_p1 = top_p1, r.min_p1 = min_p1, r.top_k1 = top_k1;
  r.ids = ids, r.logp = logprobs;
  r.best = static_cast<u64*>(scratch);
  r.mass = r.best + (long long)B * chunks;
  r.list = r.mass + (long long)B * (BINS + 1);
  r.picked = reinterpret_cast<Picked*>(r.list + (long long)B * chunks * CAP);
  r.count = reinterpret_cast<uint32_t*>(r.picked + B);
  r.found = r.count + (long long)B * (BINS + 4);
  const hipStream_t s = static_cast<hipStream_t>(stream);
#define KO_SAMPLE(F)                                                                    \
  if (chunks == 1) {                                                                    \
    hipLaunchKernelGGL(sample_kernel<F>, dim3(B), dim3(NT), 0, s, r);                   \
  } else {                                                                              \
    hipLaunchKernelGGL(maxima_kernel<F>, dim3(chunks, B), dim3(NT), 0, s, r);           \
    hipLaunchKernelGGL(bins_kernel<F>, dim3(chunks, B), dim3(NT), 0, s, r);             \
    hipLaunchKernelGGL(draw_kernel<F>, dim3(chunks, B), dim3(NT), 0, s, r);             \
  }
  if (f32) {
    KO_SAMPLE(true)
  } else {
    KO_SAMPLE(false)
  }
#undef KO_SAMPLE
  return KO_LAUNCH_STATUS();
}

}  // extern "C"
