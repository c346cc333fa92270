// One token for each row of logits by temperature, top-k, top-p and min-p from given random numbers.
//
// With the row's tokens in order of falling logit (ties: the lowest index first), every filter
// keeps a beginning of the order, and the drawn token is where the running mass passes u times
// the kept mass: all four are places in one order, found by count or by mass, and no sort of the row
// is needed. Masses are whole numbers, W = rint(2^42 exp((x - max) / T)) from an exp in 64
// bits: sums of up to 2^20 of them are exact in 64 bits in any order, so atomics and splits of a row do
// not show in the result. A token of probability below 2^-43 of the largest has mass 0.
//
// - maxima: the largest logit of each chunk of a row and its first index (greedy rows end here).
// - histogram: tokens by z = (max - x) log2(e) / T in 2048 bins over 44 octaves, counts and masses
//   (a row with a small top-k takes counts only: no exp for its whole vocabulary), first in LDS, then
//   added to the row's in memory. The last workgroup of a row finishes it: a running sum over the
//   bins gives the bin of a place, the bin's tokens are gathered from the row (in the caches by
//   now), sorted in LDS, and the place lies where their running sum says. A bin of more tokens
//   than LDS is given (equal logits, say) is narrowed down digit by digit of (logit, index) instead.
// A row that is one chunk does all of it in one workgroup and one launch.
#include "ko_common.h"

namespace {

using namespace ko;

typedef unsigned long long u64;

constexpr int NT = 1024, NW = NT / 64;
constexpr int BINS = 2048, CAP = 2048;
constexpr int SHIFT = 42;             // a mass of 1 is 2^42: 2^20 tokens sum below 2^63
constexpr float ZMAX = SHIFT + 2;     // octaves: masses from here on are 0
constexpr float PER_OCTAVE = BINS / ZMAX;
constexpr int K_COUNTED = 1024;       // top-k up to here: counts alone find the kept tokens
constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;

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
  u64* best;      // [B][chunks]: ordered logit << 32 | ~index
  u64* mass;      // [B][BINS + 1]: the last is min-p's
  uint32_t* count;   // [B][BINS + 1]: the last is the arrival counter
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
  // f(index, logit) for the elements of the vectors [v0, v1), U loads of a thread at a time.
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
  // -1: a token of mass 0 (a logit of -infinity or NaN among them).
  __device__ __forceinline__ int bin(float x) const {
    if (top == __builtin_huge_valf()) return x == top ? 0 : -1;
    const float z = fmaf(x, -0.5f, 0.5f * top) * inv;   // falls with x, roundings and all
    return z < ZMAX ? min((int)(z * PER_OCTAVE), BINS - 1) : -1;
  }
  __device__ __forceinline__ double octaves(float x) const {
    return x == top ? 0.0 : ((double)top - (double)x) * invd;
  }
  __device__ __forceinline__ u64 mass(float x, double* w) const {
    *w = exp2(-octaves(x));
    return (u64)(*w * (double)(1ull << SHIFT) + 0.5);
  }
};

struct Shared {
  uint32_t count[BINS];   // of each bin, then running
  u64 mass[BINS];
  u64 key[CAP], cum[CAP];
  u64 part[NW];
  u64 minp;
  u64 found, found_mass;
  uint32_t n;
  int at;
  u64 best;
};

__device__ __forceinline__ u64 shfl_up(u64 v, int d) {
  return ((u64)(uint32_t)__shfl_up((int)(v >> 32), d) << 32) | (uint32_t)__shfl_up((int)(uint32_t)v, d);
}
__device__ __forceinline__ u64 shfl_xor(u64 v, int d) {
  return ((u64)(uint32_t)__shfl_xor((int)(v >> 32), d) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)v, d);
}

// The sum of v over the threads up to and with this one.
__device__ u64 running(u64 v, u64* part) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = shfl_up(v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 63) part[wv] = v;
  __syncthreads();
  for (int i = 0; i < wv; ++i) v += part[i];
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
  u64 best = 0;   // nothing: no logit is a number above -infinity
  row.template each<4>(v0, v1, [&](int i, float x) {
    if (x > -__builtin_huge_valf()) {
      const u64 c = (u64)ordered(x) << 32 | (uint32_t)~i;
      best = c > best ? c : best;
    }
  });
  return block_max(best, part);
}

// Counts and masses of the vectors' tokens by bin, into s.
template <bool F32>
__device__ void histogram(const Row<F32>& row, int v0, int v1, const Scale& sc, bool masses, float mp,
                          Shared& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) s.count[i] = 0, s.mass[i] = 0;
  if (threadIdx.x == 0) s.minp = 0;
  __syncthreads();
  u64 kept = 0;
  row.template each<4>(v0, v1, [&](int, float x) {
    const int b = sc.bin(x);
    if (b < 0) return;
    atomicAdd(&s.count[b], 1u);
    if (masses) {
      double w;
      const u64 m = sc.mass(x, &w);
      atomicAdd(&s.mass[b], m);
      if (w >= (double)mp) kept += m;
    }
  });
  if (masses && mp > 0.f) atomicAdd(&s.minp, kept);
  __syncthreads();
}

// Bins to running sums.
__device__ void accumulate(Shared& s) {
  const int t = threadIdx.x;
  const uint32_t c0 = s.count[2 * t], c1 = s.count[2 * t + 1];
  const u64 m0 = s.mass[2 * t], m1 = s.mass[2 * t + 1];
  const u64 c = running(c0 + c1, s.part), m = running(m0 + m1, s.part);
  s.count[2 * t] = (uint32_t)c - c1, s.count[2 * t + 1] = (uint32_t)c;
  s.mass[2 * t] = m - m1, s.mass[2 * t + 1] = m;
  __syncthreads();
}

// The tokens of bins [b0, b1] into s.key, sorted by (falling logit, index); s.cum: their running
// mass. At most CAP.
template <bool F32>
__device__ void gather(const Row<F32>& row, const Scale& sc, int b0, int b1, Shared& s) {
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  row.template each<4>(0, row.vectors, [&](int i, float x) {
    const int b = sc.bin(x);
    if (b >= b0 && b <= b1) {
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < CAP) s.key[at] = (u64)~ordered(x) << 32 | (uint32_t)i;
    }
  });
  __syncthreads();
  const int n = min((int)s.n, CAP);
  int m = 64;
  while (m < n) m <<= 1;
  for (int i = n + threadIdx.x; i < m; i += NT) s.key[i] = ~0ull;
  __syncthreads();
  for (int size = 2; size <= m; size <<= 1)
    for (int d = size >> 1; d > 0; d >>= 1) {
      if ((int)threadIdx.x < m / 2) {
        const int i = ((int)threadIdx.x / d) * 2 * d + (int)threadIdx.x % d;
        const u64 a = s.key[i], b = s.key[i + d];
        if ((a > b) == ((i & size) == 0)) s.key[i] = b, s.key[i + d] = a;
      }
      __syncthreads();
    }
  u64 w[2];
  double unused;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = 2 * threadIdx.x + j;
    w[j] = i < n ? sc.mass(unordered(~(uint32_t)(s.key[i] >> 32)), &unused) : 0;
  }
  const u64 c = running(w[0] + w[1], s.part);
  s.cum[2 * threadIdx.x] = c - w[1], s.cum[2 * threadIdx.x + 1] = c;
  __syncthreads();
}

struct Place {
  u64 key, mass;   // the token, and the mass up to and with it
};

// The first token of the order at which the count or the mass reaches target >= 1 (the caller sees
// to it that one does).
template <bool F32>
__device__ Place find(const Row<F32>& row, const Scale& sc, bool by_count, u64 target, Shared& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) {
    const u64 here = by_count ? s.count[i] : s.mass[i];
    const u64 before = i ? (by_count ? s.count[i - 1] : s.mass[i - 1]) : 0;
    if (here >= target && before < target) s.at = i;
  }
  __syncthreads();
  const int b = s.at;
  const uint32_t c0 = b ? s.count[b - 1] : 0;
  const u64 m0 = b ? s.mass[b - 1] : 0;
  const int n = (int)(s.count[b] - c0);
  if (n <= CAP) {
    gather(row, sc, b, b, s);
    for (int i = threadIdx.x; i < n; i += NT) {
      const u64 here = by_count ? c0 + i + 1 : m0 + s.cum[i];
      const u64 before = by_count ? c0 + i : m0 + (i ? s.cum[i - 1] : 0);
      if (here >= target && before < target) s.found = s.key[i], s.found_mass = m0 + s.cum[i];
    }
    __syncthreads();
    return {s.found, s.found_mass};
  }
  // 8 bits of the key at a time, over the row; s.cum and s.key hold the digit's masses and counts
  u64 prefix = 0, known = 0, count = c0, mass = m0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    if (!F32 && (shift == 32 || shift == 40)) {
      // a bf16 logit's lower half is zeros: in the key ones, of a negative logit zeros
      if (!(prefix >> 63)) prefix |= 0xffull << shift;
      known |= 0xffull << shift;
      continue;
    }
    __syncthreads();
    if (threadIdx.x < 256) s.cum[threadIdx.x] = s.key[threadIdx.x] = 0;
    __syncthreads();
    row.template each<4>(0, row.vectors, [&](int i, float x) {
      if (sc.bin(x) != b) return;
      const u64 key = (u64)~ordered(x) << 32 | (uint32_t)i;
      if ((key & known) != prefix) return;
      double w;
      const int digit = (int)(key >> shift) & 255;
      atomicAdd(&s.key[digit], 1ull);
      atomicAdd(&s.cum[digit], sc.mass(x, &w));
    });
    __syncthreads();
    const u64 c = threadIdx.x < 256 ? s.key[threadIdx.x] : 0, m = threadIdx.x < 256 ? s.cum[threadIdx.x] : 0;
    const u64 rc = count + running(c, s.part), rm = mass + running(m, s.part);
    const u64 here = by_count ? rc : rm, before = by_count ? rc - c : rm - m;
    if (threadIdx.x < 256 && here >= target && before < target) {
      s.at = threadIdx.x;
      s.found = rc - c, s.found_mass = rm - m;
    }
    __syncthreads();
    const u64 digit = (u64)s.at;
    prefix |= digit << shift, known |= 0xffull << shift;
    count = s.found, mass = s.found_mass;
  }
  double w;
  const u64 own = sc.mass(unordered(~(uint32_t)(prefix >> 32)), &w);
  return {prefix, mass + own};
}

// u's place in a kept mass.
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

__device__ void result(const Rows& r, long long b, const Scale& sc, u64 key, u64 kept) {
  if (threadIdx.x) return;
  r.ids[b] = (uint32_t)key;
  if (r.logp) {
    const float x = unordered(~(uint32_t)(key >> 32));
    r.logp[b] = (float)(-sc.octaves(x) * LN2 - log((double)kept) + SHIFT * LN2);
  }
}

// The row's token from its bins (counts and, unless counted, masses) in s.
template <bool F32>
__device__ void finish(const Rows& r, long long b, const Row<F32>& row, const Settings& st,
                       const Scale& sc, Shared& s) {
  accumulate(s);
  const uint32_t total = s.count[BINS - 1];
  if (st.counted()) {
    const uint32_t k = min((uint32_t)st.k, total);
    for (int i = threadIdx.x; i < BINS; i += NT)
      if (s.count[i] >= k && (i ? s.count[i - 1] : 0) < k) s.at = i;
    __syncthreads();
    const int last = s.at;
    if (s.count[last] <= CAP) {
      // every token down to the k-th's bin, in order: all places are in s.cum
      gather(row, sc, 0, last, s);
      u64 kept = s.cum[k - 1];
      if (st.p < 1.f) {
        const u64 target = nucleus(st.p, kept);
        for (int i = threadIdx.x; i < (int)k; i += NT)
          if (s.cum[i] >= target && (i ? s.cum[i - 1] : 0) < target) s.found_mass = s.cum[i];
        __syncthreads();
        kept = s.found_mass;
      }
      if (st.mp > 0.f) {
        double w = 1.0, w1 = 0.0;
        for (int i = threadIdx.x; i < (int)k; i += NT) {
          sc.mass(unordered(~(uint32_t)(s.key[i] >> 32)), &w);
          if (i + 1 < (int)k) sc.mass(unordered(~(uint32_t)(s.key[i + 1] >> 32)), &w1);
          else w1 = -1.0;
          if ((w >= (double)st.mp || i == 0) && !(w1 >= (double)st.mp)) s.minp = s.cum[i];
        }
        __syncthreads();
        kept = s.minp < kept ? s.minp : kept;
      }
      const u64 target = draw(st.u, kept);
      for (int i = threadIdx.x; i < (int)k; i += NT)
        if (s.cum[i] >= target && (i ? s.cum[i - 1] : 0) < target) s.found = s.key[i];
      __syncthreads();
      result(r, b, sc, s.found, kept);
      return;
    }
    histogram(row, 0, row.vectors, sc, true, st.mp, s);
    accumulate(s);
  }
  u64 kept = s.mass[BINS - 1];
  if (st.k && (uint32_t)st.k < total) kept = find(row, sc, true, (u64)st.k, s).mass;
  if (st.p < 1.f) kept = find(row, sc, false, nucleus(st.p, kept), s).mass;
  if (st.mp > 0.f) {
    const u64 least = s.minp ? s.minp : 1ull << SHIFT;   // nothing reaches min_p > 1: the first token
    kept = least < kept ? least : kept;
  }
  const Place at = find(row, sc, false, draw(st.u, kept), s);
  result(r, b, sc, at.key, kept);
}

// What needs no more than the row's best; true if that was all.
__device__ bool decided(const Rows& r, long long b, const Settings& st, u64 best) {
  if (best && !st.first()) return false;
  if (threadIdx.x == 0) {
    r.ids[b] = best ? (long long)(uint32_t)~(uint32_t)best : -1;
    if (r.logp) r.logp[b] = best ? 0.f : -__builtin_huge_valf();
  }
  return true;
}

template <bool F32>
__global__ __launch_bounds__(NT) void sample_kernel(Rows r) {
  __shared__ Shared s;
  const long long b = blockIdx.x;
  const Row<F32> row(r, b);
  const Settings st(r, b);
  const u64 best = best_of(row, 0, row.vectors, s.part);
  if (decided(r, b, st, best)) return;
  const Scale sc(unordered((uint32_t)(best >> 32)), st.t);
  histogram(row, 0, row.vectors, sc, !st.counted(), st.mp, s);
  finish(r, b, row, st, sc, s);
}

template <bool F32>
__global__ __launch_bounds__(NT) void maxima_kernel(Rows r) {
  __shared__ u64 part[NW];
  const long long b = blockIdx.y;
  const int c = blockIdx.x;
  const Row<F32> row(r, b);
  const int per = (row.vectors + r.chunks - 1) / r.chunks;
  // the row's bins, to be added to by the next launch
  for (int i = c * NT + threadIdx.x; i <= BINS; i += r.chunks * NT)
    r.mass[b * (BINS + 1) + i] = 0, r.count[b * (BINS + 1) + i] = 0;
  const u64 best = best_of(row, min(c * per, row.vectors), min((c + 1) * per, row.vectors), part);
  if (threadIdx.x == 0) r.best[b * r.chunks + c] = best;
}

template <bool F32>
__global__ __launch_bounds__(NT) void bins_kernel(Rows r) {
  __shared__ Shared s;
  const long long b = blockIdx.y;
  const int c = blockIdx.x;
  const Row<F32> row(r, b);
  const Settings st(r, b);
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
  if (!best || st.first()) {
    if (c == 0) decided(r, b, st, best);
    return;
  }
  const Scale sc(unordered((uint32_t)(best >> 32)), st.t);
  const int per = (row.vectors + r.chunks - 1) / r.chunks;
  const bool masses = !st.counted();
  histogram(row, min(c * per, row.vectors), min((c + 1) * per, row.vectors), sc, masses, st.mp, s);
  u64* mass = r.mass + b * (BINS + 1);
  uint32_t* count = r.count + b * (BINS + 1);
  for (int i = threadIdx.x; i < BINS; i += NT) {
    if (!s.count[i]) continue;
    __hip_atomic_fetch_add(count + i, s.count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (masses) __hip_atomic_fetch_add(mass + i, s.mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (threadIdx.x == 0 && s.minp)
    __hip_atomic_fetch_add(mass + BINS, s.minp, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __builtin_amdgcn_s_waitcnt(0);   // this thread's additions are performed
  __syncthreads();
  if (threadIdx.x == 0)
    s.at = (int)__hip_atomic_fetch_add(count + BINS, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s.at != r.chunks - 1) return;
  for (int i = threadIdx.x; i < BINS; i += NT) {
    s.count[i] = __hip_atomic_load(count + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s.mass[i] = masses ? __hip_atomic_load(mass + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
  }
  if (threadIdx.x == 0) s.minp = __hip_atomic_load(mass + BINS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  finish(r, b, row, st, sc, s);
}

}  // namespace

extern "C" {

long long ko_sample_scratch(int B, int chunks) {
  if (B < 1 || chunks < 1 || chunks > 1024) return -1;
  if (chunks == 1) return 0;
  return (long long)B * (8 * chunks + 12 * (BINS + 1));
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
  r.count = reinterpret_cast<uint32_t*>(r.mass + (long long)B * (BINS + 1));
  const hipStream_t s = static_cast<hipStream_t>(stream);
#define KO_SAMPLE(F)                                                                    \
  if (chunks == 1) {                                                                    \
    hipLaunchKernelGGL(sample_kernel<F>, dim3(B), dim3(NT), 0, s, r);                   \
  } else {                                                                              \
    hipLaunchKernelGGL(maxima_kernel<F>, dim3(chunks, B), dim3(NT), 0, s, r);           \
    hipLaunchKernelGGL(bins_kernel<F>, dim3(chunks, B), dim3(NT), 0, s, r);             \
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
