// Decode attention over the 4-bit KV cache (kv4_core.h), for gfx950.
//
// Query row (t, h) of sequence b and KV head j, t of T tokens, sees the keys below len - T + t + 1:
//   score_k = scale sum_g (s_kg sum_{d in g} q_d (n_kd - 8) + c_kg sum_{d in g} q_d)
//   out_d   = sum_k p_k (c_kg + s_kg (n_kd - 8)) / sum_k p_k,  p_k = exp(score_k - max)
// A row that sees no key is zero.
#include "kv4_core.h"

using namespace ko;

namespace {

struct Kv4AttnArgs {
  const uint16_t* q;  // [B*T, nq*D]
  const uint8_t* cache;
  long long cb, ch;  // bytes
  const int* lens;
  int len_off, cap, B, T, nkv, G;
  float scale_log2;
  uint16_t* out;
};

// One workgroup per query row; wavefront w takes the blocks w, w + 4, ... Lane (key, half) forms
// half a score; lane l then owns the columns l and l + 64.
template <int D, int NG>
__global__ __launch_bounds__(256) void kv4_attn_kernel(Kv4AttnArgs a) {
  constexpr int HP = D / 64, GS = D / NG;
  __shared__ float qs[D], ps[4][32], om[4][2], oa[4][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int row = blockIdx.x;
  const int h = row % a.G;
  row /= a.G;
  const int j = row % a.nkv;
  row /= a.nkv;
  const int t = row % a.T, b = row / a.T;
  const long long qo = ((long long)(b * a.T + t) * a.nkv * a.G + j * a.G + h) * D;
  if (threadIdx.x < D) qs[threadIdx.x] = bf16_to_f32(a.q[qo + threadIdx.x]);
  __syncthreads();
  const long long total = min((long long)a.lens[b] + a.len_off, (long long)a.cap);
  const int lim = (int)max(total - a.T + t + 1, 0LL);  // keys this row sees
  const uint8_t* base = a.cache + b * a.cb + j * a.ch;
  float m = -3.0e38f, l = 0.f, acc[HP] = {};
  for (int blk = wave; blk * KV4_KEYS < lim; blk += 4) {
    const uint8_t* p = base + (long long)blk * kv4_block_bytes(D, NG);
    const uint32_t* ksc = reinterpret_cast<const uint32_t*>(p + 32 * D);
    const uint32_t* vsc = ksc + 32 * NG;
    const int key = lane & 31, half = lane >> 5;
    float s = 0.f;
    for (int dd = half * (D / 2); dd < (half + 1) * (D / 2); dd += 8) {
      const int i = dd / 32, kg = dd % 32 / 8;
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p + key * (D / 2) + kg * (D / 8) + 4 * i);
      const uint32_t sc = ksc[dd / GS * 32 + key];
      for (int e = 0; e < 8; ++e) {
        const int n = (w >> (4 * (e / 2) + 16 * (e & 1))) & 15;
        s = fmaf(qs[dd + e], fmaf(bf16lo(sc), (float)(n - 8), bf16hi(sc)), s);
      }
    }
    s = (s + __shfl_xor(s, 32, 64)) * a.scale_log2;
    if (blk * KV4_KEYS + key >= lim) s = -INFINITY;
    const float mn = fmaxf(m, wave_max(s));
    const float al = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    const float pr = __builtin_amdgcn_exp2f(s - m);
    l = l * al + 0.5f * wave_sum(pr);  // both halves hold every key
    __builtin_amdgcn_wave_barrier();
    ps[wave][key] = pr;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int keys = min(lim - blk * KV4_KEYS, KV4_KEYS);
    for (int c = 0; c < HP; ++c) {
      const int col = lane + 64 * c;
      const int jj = 2 * (col / 32) + (col & 1), n = col % 32 / 2;
      float o = acc[c] * al;
      for (int k = 0; k < keys; ++k) {
        const uint8_t* w = p + 16 * D + ((k / 8 * HP + jj / 4) * 16 + n) * 16 + k % 8 * 2;
        const int code = (*reinterpret_cast<const uint16_t*>(w) >> (4 * (jj & 3))) & 15;
        const uint32_t sc = vsc[col / GS * 32 + k];
        o = fmaf(ps[wave][k], fmaf(bf16lo(sc), (float)(code - 8), bf16hi(sc)), o);
      }
      acc[c] = o;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  if (lane == 0) om[wave][0] = m, om[wave][1] = l;
  for (int c = 0; c < HP; ++c) oa[wave][lane + 64 * c] = acc[c];
  __syncthreads();
  if (threadIdx.x < D) {
    float mx = om[0][0], L = 0.f, o = 0.f;
    for (int w = 1; w < 4; ++w) mx = fmaxf(mx, om[w][0]);
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(om[w][0] - mx);
      L += f * om[w][1];
      o += f * oa[w][threadIdx.x];
    }
    a.out[qo + threadIdx.x] = f32_to_bf16(L == 0.f ? 0.f : o / L);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" {

int ko_kv4_attn(const void* q, const void* cache, long long cache_b_stride,
                long long cache_h_stride, const int* kv_lens, int len_offset, int cap, int B,
                int T, int nq, int nkv, int d, int group, float scale, void* out, void* stream) {
  if (!q || !cache || !kv_lens || !out || B < 1 || T < 1 || nkv < 1 || nq < 1 || cap < 1)
    return KO_EINVAL;
  if (!kv4_served(d, group) || nq % nkv) return KO_ENOTSUP;
  if (!aligned16(q) || !aligned16(cache) || !aligned16(out) || (cache_b_stride & 15) ||
      (cache_h_stride & 15))
    return KO_EINVAL;
  const long long rows = (long long)B * T * nq;
  if (rows > (1LL << 24) - 1) return KO_ERANGE;
  const Kv4AttnArgs a = {static_cast<const uint16_t*>(q), static_cast<const uint8_t*>(cache),
                         cache_b_stride, cache_h_stride, kv_lens, len_offset, cap, B, T, nkv,
                         nq / nkv, scale * 1.4426950408889634f, static_cast<uint16_t*>(out)};
  const dim3 grid((unsigned)rows), block(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define CALL(D_, NG_) hipLaunchKernelGGL((kv4_attn_kernel<D_, NG_>), grid, block, 0, s, a);
  KV4_PICK(d, group, CALL)
#undef CALL
  return KO_LAUNCH_STATUS();
}

}  // extern "C"
