// Rotation of new queries and keys, and the append of keys and values to a
// paged cache.
//
// Token t of sequence s has cache index c = kv_len[s] - n_s + (t - q_start[s])
// (n_s new tokens, kv_len counts them).  With h = hd / 2, p_j the position that
// frequency j goes by and x a query or key head (RMS-normalised first when a
// gain is given),
//   y[j]     = x[j] cos[p_j][j]     - x[j + h] sin[p_j][j]
//   y[j + h] = x[j + h] cos[p_j][j] + x[j] sin[p_j][j].
// p_j is c, or the token's position on the axis that frequency j belongs to.
//
// An 8-bit cache holds e4m3 codes and one f32 scale for each (page of 64
// tokens, head), a power of two: the least one >= 2^-64 for which the page's
// largest finite value is at most 448 scale.  So a larger value that arrives
// later only moves the exponent of what the page already holds (code * old /
// new): the 3-bit significand is rounded once, when a value is written, except
// where a code becomes subnormal.  A page's scale never shrinks while the page
// fills; the token in slot 0 starts it afresh, whatever a former user left.
//
// One CTA per (sequence, page the append touches, K/V head) holds the page's
// new keys and values in registers between the maximum and the codes, so every
// input is read once and nothing is written twice; it also rotates the group's
// query heads for the same tokens, with the same cos / sin rows.  A page and
// head belongs to one CTA: no atomics, the same bits every time.
#include <cuda_fp8.h>

#include "kernels.cuh"
#include "sm100.cuh"

namespace qa {

namespace {

constexpr int kPage = 64;
constexpr int kThreads = 256;
constexpr float kE4m3Max = 448.0f;

struct AppendParams {
  const void *q, *k, *v;
  long long ldq, ldk, ldv, ldqo;
  void* q_out;
  long long T;
  int group;  // query heads per K/V head
  int nkv;
  SeqMap seqs;
  int pages_per_seq;  // grid.x = n_seqs * pages_per_seq
  void *kpool, *vpool;
  int kv_pages;
  float *kscale, *vscale;
  RopeAxes rope;
  const float *qn, *kn;
  float eps;
  int vec;  // q, k, v and q_out rows can be read and written 16 bytes at a time
  unsigned* status;
};

// Eight consecutive 16-bit values.
template <typename T>
__device__ __forceinline__ uint4 load8(const T* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint4 r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = p[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, uint4 d, bool vec) {
  if (vec) {
    *reinterpret_cast<uint4*>(p) = d;
    return;
  }
  const T* e = reinterpret_cast<const T*>(&d);
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = e[i];
}
template <typename T>
__device__ __forceinline__ void widen8(uint4 d, float* f) {
  const T* e = reinterpret_cast<const T*>(&d);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = h2f<T>(e[i]);
}
template <typename T>
__device__ __forceinline__ uint4 narrow8(const float* f) {
  return make_uint4(cvt2_rn<T>(make_float2(f[0], f[1])), cvt2_rn<T>(make_float2(f[2], f[3])),
                    cvt2_rn<T>(make_float2(f[4], f[5])), cvt2_rn<T>(make_float2(f[6], f[7])));
}

// Least power of two s >= 2^-64 with m <= 448 s (m finite, >= 0).  448 is
// 1.75 * 2^8, so the exponent follows from m's own and one comparison.
__device__ __forceinline__ float page_scale(float m) {
  const int b = __float_as_int(m);
  const int e = (b >> 23) - 127 - 8 + ((b & 0x7FFFFF) > 0x600000 ? 1 : 0);
  return __int_as_float((max(e, -64) + 127) << 23);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;  // NaN and infinities do not size the scale
}

// Eight values as e4m3 codes of scale 1 / inv; non-finite values become NaN.
__device__ __forceinline__ uint2 codes8(const float* f, float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v = make_float2(f[2 * i] * inv, f[2 * i + 1] * inv);
    if (!(fabsf(f[2 * i]) < INFINITY)) v.x = NAN;
    if (!(fabsf(f[2 * i + 1]) < INFINITY)) v.y = NAN;
    w[i] = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// Codes of a page's first `rows` rows, multiplied by ratio < 1.
__device__ __forceinline__ void rescale_rows(uint8_t* page, int bytes, float ratio) {
  for (int i = threadIdx.x * 16; i < bytes; i += kThreads * 16) {
    uint4 d = *reinterpret_cast<uint4*>(page + i);
    __nv_fp8x2_storage_t* c = reinterpret_cast<__nv_fp8x2_storage_t*>(&d);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(c[j], __NV_E4M3);
      float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      f.x *= ratio;
      f.y *= ratio;
      c[j] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
    }
    *reinterpret_cast<uint4*>(page + i) = d;
  }
}

template <typename T, int HD, bool B8>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(AppendParams ap) {
  constexpr int kHalf = HD / 2;
  constexpr int kLanes = HD / 16;             // lanes of a row: 8 dims of each half per lane
  constexpr int kAtOnce = kThreads / kLanes;  // rows at once
  constexpr int kRounds = kPage / kAtOnce;
  __shared__ float s_max[2][kThreads / 32];

  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.x / ap.pages_per_seq, j = blockIdx.x % ap.pages_per_seq;
  const int h = blockIdx.y;
  const SeqSpan sp = seq_span(ap.seqs, s, ap.T);
  if (!sp.ok || sp.n > sp.len) {
    if (j == 0 && h == 0 && threadIdx.x == 0 && ap.status) atomicOr(ap.status, kStatusBadShape);
    return;
  }
  const int c0 = sp.len - sp.n;       // cache index of the first new token
  const int pg = c0 / kPage + j;      // page of the sequence
  const int lo = max(c0, pg * kPage), hi = min(sp.len, (pg + 1) * kPage);  // cache indices
  if (lo >= hi) return;
  const int page = ap.seqs.block_tab[static_cast<long long>(s) * ap.seqs.max_pages + pg];
  const bool page_ok = page >= 0 && page < ap.kv_pages;
  bool bad = !page_ok;

  const int row = threadIdx.x / kLanes, d0 = (threadIdx.x % kLanes) * 8;
  const bool vec = ap.vec;
  int ax[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) ax[i] = ap.rope.n_axes > 1 ? ap.rope.axis_of[d0 + i] & 3 : 0;

  float kx[B8 ? kRounds : 1][16];
  uint4 vx[B8 ? kRounds : 1][2];
  float kmax = 0.0f, vmax = 0.0f;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int rr = B8 ? r : 0;
    const int c = lo + r * kAtOnce + row;
    const bool on = c < hi;
    // lanes without a token follow along with the last one's, for the shuffles
    const long long t = sp.t0 + (min(c, hi - 1) - c0);
    float cs[8], sn[8];
    if (ap.rope.cos_t) {
      int p[4] = {static_cast<int>(t - sp.t0) + c0, 0, 0, 0};
      if (ap.rope.pos)
#pragma unroll
        for (int a = 0; a < 4; ++a)
          if (a < ap.rope.n_axes) p[a] = ap.rope.pos[a * ap.rope.pos_stride + t];
#pragma unroll
      for (int a = 0; a < 4; ++a)
        if (p[a] < 0 || p[a] >= ap.rope.rows) {
          bad = true;
          p[a] = 0;
        }
      if (ap.rope.n_axes > 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int pi = ax[i] == 0 ? p[0] : ax[i] == 1 ? p[1] : ax[i] == 2 ? p[2] : p[3];
          const long long at = static_cast<long long>(pi) * kHalf + d0 + i;
          cs[i] = ap.rope.cos_t[at];
          sn[i] = ap.rope.sin_t[at];
        }
      } else {
        const long long at = static_cast<long long>(p[0]) * kHalf + d0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          reinterpret_cast<float4*>(cs)[i] = reinterpret_cast<const float4*>(ap.rope.cos_t + at)[i];
          reinterpret_cast<float4*>(sn)[i] = reinterpret_cast<const float4*>(ap.rope.sin_t + at)[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cs[i] = 1.0f;
        sn[i] = 0.0f;
      }
    }
    // a row's 16 values of this lane: normalised, rotated
    auto turn = [&](uint4 a, uint4 b, const float* gain, float* y) {
      float x[16];
      widen8<T>(a, x);
      widen8<T>(b, x + 8);
      if (gain) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        const float inv = rsqrtf(ss * (1.0f / HD) + ap.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] *= inv * gain[d0 + i];
          x[8 + i] *= inv * gain[kHalf + d0 + i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = x[i] * cs[i] - x[8 + i] * sn[i];
        y[8 + i] = x[8 + i] * cs[i] + x[i] * sn[i];
      }
    };
    const T* kr = static_cast<const T*>(ap.k) + t * ap.ldk + h * HD + d0;
    const T* vr = static_cast<const T*>(ap.v) + t * ap.ldv + h * HD + d0;
    const uint4 ka = load8(kr, vec), kb = load8(kr + kHalf, vec);
    vx[rr][0] = load8(vr, vec);
    vx[rr][1] = load8(vr + kHalf, vec);
    turn(ka, kb, ap.kn, kx[rr]);
    if constexpr (B8) {
      if (on) {
        float vf[16];
        widen8<T>(vx[rr][0], vf);
        widen8<T>(vx[rr][1], vf + 8);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          kmax = fmaxf(kmax, finite_abs(kx[rr][i]));
          vmax = fmaxf(vmax, finite_abs(vf[i]));
        }
      }
    } else if (on && page_ok) {
      const long long at = ((static_cast<long long>(page) * ap.nkv + h) * kPage + c % kPage) * HD + d0;
      T* kd = static_cast<T*>(ap.kpool) + at;
      T* vd = static_cast<T*>(ap.vpool) + at;
      store8(kd, narrow8<T>(kx[rr]), true);
      store8(kd + kHalf, narrow8<T>(kx[rr] + 8), true);
      store8(vd, vx[rr][0], true);
      store8(vd + kHalf, vx[rr][1], true);
    }
#pragma unroll 2
    for (int g = 0; g < ap.group; ++g) {
      const long long col = static_cast<long long>(h * ap.group + g) * HD + d0;
      const T* qr = static_cast<const T*>(ap.q) + t * ap.ldq + col;
      const uint4 qa = load8(qr, vec), qb = load8(qr + kHalf, vec);
      float y[16];
      turn(qa, qb, ap.qn, y);
      if (on) {
        T* qd = static_cast<T*>(ap.q_out) + t * ap.ldqo + col;
        store8(qd, narrow8<T>(y), vec);
        store8(qd + kHalf, narrow8<T>(y + 8), vec);
      }
    }
  }
  if (bad && ap.status) atomicOr(ap.status, kStatusBadShape);
  if constexpr (B8) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      kmax = fmaxf(kmax, __shfl_xor_sync(0xFFFFFFFFu, kmax, o));
      vmax = fmaxf(vmax, __shfl_xor_sync(0xFFFFFFFFu, vmax, o));
    }
    if ((threadIdx.x & 31) == 0) {
      s_max[0][threadIdx.x / 32] = kmax;
      s_max[1][threadIdx.x / 32] = vmax;
    }
    if (!page_ok) return;
    const long long ph = static_cast<long long>(page) * ap.nkv + h;
    const int a = lo % kPage;  // rows of the page that were there before
    const float kold = a ? ap.kscale[ph] : 0.0f, vold = a ? ap.vscale[ph] : 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
      kmax = fmaxf(kmax, s_max[0][i]);
      vmax = fmaxf(vmax, s_max[1][i]);
    }
    const float ks = fmaxf(kold, page_scale(kmax)), vs = fmaxf(vold, page_scale(vmax));
    uint8_t* kp = static_cast<uint8_t*>(ap.kpool) + ph * (kPage * HD);
    uint8_t* vp = static_cast<uint8_t*>(ap.vpool) + ph * (kPage * HD);
    if (a && kold < ks) rescale_rows(kp, a * HD, kold / ks);
    if (a && vold < vs) rescale_rows(vp, a * HD, vold / vs);
    if (threadIdx.x == 0) {
      ap.kscale[ph] = ks;
      ap.vscale[ph] = vs;
    }
    const float kinv = 1.0f / ks, vinv = 1.0f / vs;  // exact: powers of two
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int c = lo + r * kAtOnce + row;
      if (c < hi) {
        float vf[16];
        widen8<T>(vx[r][0], vf);
        widen8<T>(vx[r][1], vf + 8);
        const int at = c % kPage * HD + d0;
        *reinterpret_cast<uint2*>(kp + at) = codes8(kx[r], kinv);
        *reinterpret_cast<uint2*>(kp + at + kHalf) = codes8(kx[r] + 8, kinv);
        *reinterpret_cast<uint2*>(vp + at) = codes8(vf, vinv);
        *reinterpret_cast<uint2*>(vp + at + kHalf) = codes8(vf + 8, vinv);
      }
    }
  }
}

template <typename T, int HD>
cudaError_t launch(const AppendParams& ap, dim3 grid, bool b8, cudaStream_t s) {
  return b8 ? launch_pdl(kv_append_kernel<T, HD, true>, grid, dim3(kThreads), 0, s, ap)
            : launch_pdl(kv_append_kernel<T, HD, false>, grid, dim3(kThreads), 0, s, ap);
}

}  // namespace

int kv_append(const void* q, long long ldq, const void* k, long long ldk, const void* v,
              long long ldv, void* q_out, long long ldqo, long long T, int nqh, int nkvh, int hd,
              const SeqMap& seqs, int max_q, PagedKV kv, int kv_pages, float* kscale, float* vscale,
              const RopeAxes& rope, const float* qn, const float* kn, float eps, bool bf16,
              unsigned* status, cudaStream_t s) {
  if (T <= 0 || seqs.n_seqs <= 0 || max_q <= 0) return 0;
  AppendParams ap{};
  ap.q = q;
  ap.k = k;
  ap.v = v;
  ap.q_out = q_out;
  ap.ldq = ldq;
  ap.ldk = ldk;
  ap.ldv = ldv;
  ap.ldqo = ldqo;
  ap.T = T;
  ap.group = nqh / nkvh;
  ap.nkv = nkvh;
  ap.seqs = seqs;
  ap.seqs.max_q = max_q;
  ap.pages_per_seq = (max_q + 2 * kPage - 2) / kPage;  // a run of max_q tokens from slot 63 on
  ap.kpool = kv.k;
  ap.vpool = kv.v;
  ap.kv_pages = kv_pages;
  ap.kscale = kscale;
  ap.vscale = vscale;
  ap.rope = rope;
  ap.qn = qn;
  ap.kn = kn;
  ap.eps = eps;
  ap.vec = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
             reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q_out)) % 16 == 0) &&
           ((ldq | ldk | ldv | ldqo) % 8 == 0);
  ap.status = status;
  const long long gx = static_cast<long long>(seqs.n_seqs) * ap.pages_per_seq;
  if (gx > 0x7FFFFFFFll || nkvh > 65535) return (int)cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(gx), nkvh);
  cudaError_t e;
  if (bf16)
    e = hd == 128 ? launch<__nv_bfloat16, 128>(ap, grid, kscale != nullptr, s)
                  : launch<__nv_bfloat16, 64>(ap, grid, kscale != nullptr, s);
  else
    e = hd == 128 ? launch<__half, 128>(ap, grid, kscale != nullptr, s)
                  : launch<__half, 64>(ap, grid, kscale != nullptr, s);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace qa
