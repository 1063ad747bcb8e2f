// Attention over the 8-bit paged cache (codes and scales as kv_append writes
// them).
//
// Query i of sequence s (n new tokens, len cached ones, the new ones among
// them) sees cache indices c < len - n + i + 1 when causal, c < len otherwise:
//   s_c = scale kscale[page(c)] (q . kcode_c),  out = sum_c softmax(s)_c vscale[page(c)] vcode_c,
// lse = log sum_c exp(s_c); a row that sees nothing gets 0 and -inf.
#include <cuda_fp8.h>

#include "kernels.cuh"
#include "sm100.cuh"

namespace qa {

namespace {

constexpr int kPage = 64;

struct CacheAttnParams {
  const void* q;
  long long ldq, T;
  int nq, nkv;
  SeqMap seqs;
  const uint8_t *kpool, *vpool;
  int kv_pages;
  const float *kscale, *vscale;
  float scale;
  int causal;
  void* out;
  long long ldo;
  float* lse;
  unsigned* status;
};

__device__ __forceinline__ float e4m3_to_f32(uint8_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

// One warp per (query token, query head).
template <typename T, int HD>
__global__ void __launch_bounds__(128) cache_attn_simple(CacheAttnParams ap) {
  constexpr int kD = HD / 32;
  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.z, hq = blockIdx.y, lane = threadIdx.x & 31;
  const int i = blockIdx.x * 4 + threadIdx.x / 32;
  const SeqSpan sp = seq_span(ap.seqs, s, ap.T);
  if (!sp.ok) {
    if (i == 0 && hq == 0 && lane == 0 && ap.status) atomicOr(ap.status, kStatusBadShape);
    return;
  }
  if (i >= sp.n) return;
  const int h = hq / (ap.nq / ap.nkv);
  const long long t = sp.t0 + i;
  const T* qr = static_cast<const T*>(ap.q) + t * ap.ldq + static_cast<long long>(hq) * HD;
  float q[kD], o[kD], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int d = 0; d < kD; ++d) {
    q[d] = h2f<T>(qr[lane + 32 * d]);
    o[d] = 0.0f;
  }
  const int seen = ap.causal ? sp.len - sp.n + i + 1 : sp.len;
  for (int pg = 0; pg * kPage < seen; ++pg) {
    const int page = ap.seqs.block_tab[static_cast<long long>(s) * ap.seqs.max_pages + pg];
    if (page < 0 || page >= ap.kv_pages) {
      if (lane == 0 && ap.status) atomicOr(ap.status, kStatusBadShape);
      continue;
    }
    const long long ph = static_cast<long long>(page) * ap.nkv + h;
    const uint8_t* kp = ap.kpool + ph * (kPage * HD);
    const uint8_t* vp = ap.vpool + ph * (kPage * HD);
    const float ks = ap.kscale[ph] * ap.scale, vs = ap.vscale[ph];
    const int n = min(kPage, seen - pg * kPage);
    for (int c = 0; c < n; ++c) {
      float x = 0.0f;
#pragma unroll
      for (int d = 0; d < kD; ++d) x = fmaf(q[d], e4m3_to_f32(kp[c * HD + lane + 32 * d]), x);
#pragma unroll
      for (int o2 = 16; o2 > 0; o2 >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o2);
      x *= ks;
      const float nm = fmaxf(m, x);
      const float ref = nm == -INFINITY ? 0.0f : nm;  // a NaN score makes a NaN row
      const float a = __expf(m - ref), p = __expf(x - ref);
      m = nm;
      l = l * a + p;
#pragma unroll
      for (int d = 0; d < kD; ++d) o[d] = o[d] * a + p * vs * e4m3_to_f32(vp[c * HD + lane + 32 * d]);
    }
  }
  T* dst = static_cast<T*>(ap.out) + t * ap.ldo + static_cast<long long>(hq) * HD;
#pragma unroll
  for (int d = 0; d < kD; ++d) dst[lane + 32 * d] = f2h<T>(l == 0.0f ? 0.0f : o[d] / l);
  if (lane == 0 && ap.lse) ap.lse[t * ap.nq + hq] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

int cache_attention(const void* q, long long ldq, long long T, int nqh, int nkvh, int hd,
                    const SeqMap& seqs, int max_q, int max_kv, const void* kpool, const void* vpool,
                    int kv_pages, const float* kscale, const float* vscale, float scale, bool causal,
                    void* out, long long ldo, float* lse, bool bf16, unsigned* status,
                    cudaStream_t s) {
  if (T <= 0 || seqs.n_seqs <= 0 || max_q <= 0) return 0;
  CacheAttnParams ap{};
  ap.q = q;
  ap.ldq = ldq;
  ap.T = T;
  ap.nq = nqh;
  ap.nkv = nkvh;
  ap.seqs = seqs;
  ap.seqs.max_q = max_q;
  ap.kpool = static_cast<const uint8_t*>(kpool);
  ap.vpool = static_cast<const uint8_t*>(vpool);
  ap.kv_pages = kv_pages;
  ap.kscale = kscale;
  ap.vscale = vscale;
  ap.scale = scale;
  ap.causal = causal;
  ap.out = out;
  ap.ldo = ldo;
  ap.lse = lse;
  ap.status = status;
  if (nqh > 65535 || seqs.n_seqs > 65535) return (int)cudaErrorInvalidValue;
  const dim3 grid((max_q + 3) / 4, nqh, seqs.n_seqs);
  cudaError_t e;
  if (bf16)
    e = hd == 128 ? launch_pdl(cache_attn_simple<__nv_bfloat16, 128>, grid, dim3(128), 0, s, ap)
                  : launch_pdl(cache_attn_simple<__nv_bfloat16, 64>, grid, dim3(128), 0, s, ap);
  else
    e = hd == 128 ? launch_pdl(cache_attn_simple<__half, 128>, grid, dim3(128), 0, s, ap)
                  : launch_pdl(cache_attn_simple<__half, 64>, grid, dim3(128), 0, s, ap);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace qa
