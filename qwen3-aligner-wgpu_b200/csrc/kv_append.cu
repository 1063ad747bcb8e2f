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
// A CTA takes one (sequence, page the append touches, K/V head) and some of the
// group's query heads, which turn by the same cos / sin rows; the first of a
// group's CTAs also takes the keys and values.  Each thread copies what it will
// use itself into shared memory (cp.async), all of it before the first use, so
// that the loads in flight cost no registers and no barrier; the new keys stay in
// registers between the page's maximum and the codes.  Every input is read once,
// nothing is written twice, a page and head belongs to one CTA: no atomics, the
// same bits every time.
//
// Bound by bytes for long prompts, by the latency of a chain of dependent loads
// (maps, positions, rows) and the launch for few tokens.  Measured on a B200: four
// prompts of up to 8192 tokens into the 16-bit cache (16/8 heads of 128) 68 us,
// 4.9 TB/s; 24 ragged sequences (14/2 heads of 64, three axes, 8 bits) 16.5 us, 3.5
// TB/s, 26 with the inputs in registers and a loop over the heads; 64 sequences of
// one token 9.4 us in the kernel, 18 with CTAs of 256 threads.
#include <cuda_fp8.h>

#include <algorithm>

#include "kernels.cuh"
#include "sm100.cuh"

namespace qa {

namespace {

constexpr int kPage = 64;
constexpr int kThreads = 256;                    // at most
constexpr uint32_t kStage = 72 * 1024;           // staged by a CTA: three CTAs an SM

struct AppendParams {
  const void *q, *k, *v;
  long long ldq, ldk, ldv, ldqo;
  void* q_out;
  long long T;
  int group;  // query heads per K/V head
  int nkv;
  int heads;          // query heads of a CTA
  int head_ctas;      // CTAs that share a group's query heads
  int ctas;           // nkv * head_ctas, for one run of tokens
  int rounds;         // in which a CTA goes through its tokens
  SeqMap seqs;
  int runs_per_seq;   // CTAs along a sequence's new tokens, at most
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

__device__ __forceinline__ void load_f8(const float* p, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    reinterpret_cast<float4*>(f)[i] = reinterpret_cast<const float4*>(p)[i];
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

// The first `bytes` codes of a page, multiplied by ratio < 1.
__device__ __forceinline__ void rescale_rows(uint8_t* page, int bytes, float ratio) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) {
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

// Tokens of a CTA.  A page's scales need all of its new tokens in one place; the
// 16-bit cache has none, and takes what one round of threads covers.
template <int HD, bool B8>
constexpr int tokens() {
  return B8 ? kPage : kThreads / (HD / 16);
}

template <typename T, int HD, bool B8>
__global__ void __launch_bounds__(kThreads, B8 ? (HD == 128 ? 2 : 3) : 4)
    kv_append_kernel(AppendParams ap) {
  constexpr int kHalf = HD / 2;
  constexpr int kLanes = HD / 16;  // of a token: 8 dims of each half per lane
  constexpr int kTokens = tokens<HD, B8>();
  constexpr int kRounds = kTokens * kLanes / kThreads;  // at most
  extern __shared__ __align__(16) uint4 stage[];  // [slot][round][half][thread]
  __shared__ float s_max[2][kThreads / 32];

  pdl_wait();
  pdl_trigger();
  // heads first: CTAs that run together read neighbouring columns of the same rows
  const int y = blockIdx.x % ap.ctas, x = blockIdx.x / ap.ctas;
  const int s = x / ap.runs_per_seq, j = x % ap.runs_per_seq;
  const int h = y / ap.head_ctas, g0 = y % ap.head_ctas * ap.heads;
  const int heads = min(ap.heads, ap.group - g0);
  const SeqSpan sp = seq_span(ap.seqs, s, ap.T);
  if (!sp.ok || sp.n > sp.len) {
    if (j == 0 && y == 0 && threadIdx.x == 0 && ap.status) atomicOr(ap.status, kStatusBadShape);
    return;
  }
  const int c0 = sp.len - sp.n;       // cache index of the first new token
  const int run = c0 / kTokens + j;
  const int lo = max(c0, run * kTokens), hi = min(sp.len, (run + 1) * kTokens);  // cache indices
  if (lo >= hi) return;

  const int rows = blockDim.x / kLanes;  // tokens of a round
  const int row = threadIdx.x / kLanes, d0 = (threadIdx.x % kLanes) * 8;
  const int warp_row = threadIdx.x / 32 * (32 / kLanes);
  const bool vec = ap.vec, with_kv = g0 == 0;
  const long long col = static_cast<long long>(h * ap.group + g0) * HD + d0;

  // slots: the query heads, then k, then v
  auto staged = [&](int slot, int r, int half) {
    return stage + ((slot * ap.rounds + r) * 2 + half) * blockDim.x + threadIdx.x;
  };
  auto fetch = [&](int slot, int r, const T* p) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (vec)
        cp_async16(smem_u32(staged(slot, r, i)), p + i * kHalf, 16);
      else
        *staged(slot, r, i) = load8(p + i * kHalf, false);
    }
  };
  for (int r = 0; r < ap.rounds; ++r) {
    const int c = lo + r * rows + row;
    if (c < hi) {
      const long long t = sp.t0 + (c - c0);
      if (with_kv) {
        fetch(heads, r, static_cast<const T*>(ap.k) + t * ap.ldk + h * HD + d0);
        fetch(heads + 1, r, static_cast<const T*>(ap.v) + t * ap.ldv + h * HD + d0);
      }
      const T* qr = static_cast<const T*>(ap.q) + t * ap.ldq + col;
      for (int g = 0; g < heads; ++g) fetch(g, r, qr + g * HD);
    }
    cp_async_commit();
  }

  bool bad = false, page_ok = true;
  int page = 0;
  if (with_kv) {
    page = ap.seqs.block_tab[static_cast<long long>(s) * ap.seqs.max_pages + lo / kPage];
    page_ok = page >= 0 && page < ap.kv_pages;
    bad = !page_ok;
  }
  uint32_t axes = 0;  // 2 bits for each of this lane's frequencies
  if (ap.rope.cos_t && ap.rope.n_axes > 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int a = ap.rope.axis_of[d0 + i];
      const bool there = a >= 0 && a < ap.rope.n_axes;
      bad |= !there;
      axes |= static_cast<uint32_t>(there ? a : 0) << (2 * i);
    }

  float kx[B8 ? kRounds : 1][16];
  float kmax = 0.0f, vmax = 0.0f;
  // Whole warps leave, so that the shuffles below always have theirs.
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (r >= ap.rounds || lo + r * rows + warp_row >= hi) break;
    const int rr = B8 ? r : 0;
    const int c = lo + r * rows + row;
    const bool on = c < hi;
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
      load_f8(ap.rope.cos_t + static_cast<long long>(p[0]) * kHalf + d0, cs);
      load_f8(ap.rope.sin_t + static_cast<long long>(p[0]) * kHalf + d0, sn);
      // Another axis's row as a whole, only where its position differs: single
      // elements would cost the load unit a pass per token each.
#pragma unroll
      for (int a = 1; a < 4; ++a)
        if (a < ap.rope.n_axes && p[a] != p[0]) {
          const long long at = static_cast<long long>(p[a]) * kHalf + d0;
          float c2[8], s2[8];
          load_f8(ap.rope.cos_t + at, c2);
          load_f8(ap.rope.sin_t + at, s2);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if ((axes >> (2 * i) & 3) == a) {
              cs[i] = c2[i];
              sn[i] = s2[i];
            }
        }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cs[i] = 1.0f;
        sn[i] = 0.0f;
      }
    }
    // a head's 16 values of this lane: normalised, rotated
    auto turn = [&](int slot, const float* gain, float* x) {
      widen8<T>(*staged(slot, r, 0), x);
      widen8<T>(*staged(slot, r, 1), x + 8);
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
        const float a = x[i], b = x[8 + i];
        x[i] = a * cs[i] - b * sn[i];
        x[8 + i] = b * cs[i] + a * sn[i];
      }
    };
    if (r + 1 < ap.rounds)
      asm volatile("cp.async.wait_group %0;" ::"n"(kRounds - 1) : "memory");
    else
      cp_async_wait_all();
    if (with_kv) {  // uniform in the CTA
      turn(heads, ap.kn, kx[rr]);
      if constexpr (B8) {
        if (on) {
          float vf[16];
          widen8<T>(*staged(heads + 1, r, 0), vf);
          widen8<T>(*staged(heads + 1, r, 1), vf + 8);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            kmax = fmaxf(kmax, finite_abs(kx[rr][i]));
            vmax = fmaxf(vmax, finite_abs(vf[i]));
          }
        }
      } else if (on && page_ok) {
        const long long at =
            ((static_cast<long long>(page) * ap.nkv + h) * kPage + c % kPage) * HD + d0;
        T* kd = static_cast<T*>(ap.kpool) + at;
        T* vd = static_cast<T*>(ap.vpool) + at;
        store8(kd, narrow8<T>(kx[rr]), true);
        store8(kd + kHalf, narrow8<T>(kx[rr] + 8), true);
        store8(vd, *staged(heads + 1, r, 0), true);
        store8(vd + kHalf, *staged(heads + 1, r, 1), true);
      }
    }
    T* qd = static_cast<T*>(ap.q_out) + t * ap.ldqo + col;
#pragma unroll 1
    for (int g = 0; g < heads; ++g) {
      float z[16];
      turn(g, ap.qn, z);
      if (on) {
        store8(qd + g * HD, narrow8<T>(z), vec);
        store8(qd + g * HD + kHalf, narrow8<T>(z + 8), vec);
      }
    }
  }
  if (bad && ap.status) atomicOr(ap.status, kStatusBadShape);
  if constexpr (B8) {
    if (!with_kv || !page_ok) return;  // uniform in the CTA
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      kmax = fmaxf(kmax, __shfl_xor_sync(0xFFFFFFFFu, kmax, o));
      vmax = fmaxf(vmax, __shfl_xor_sync(0xFFFFFFFFu, vmax, o));
    }
    if ((threadIdx.x & 31) == 0) {
      s_max[0][threadIdx.x / 32] = kmax;
      s_max[1][threadIdx.x / 32] = vmax;
    }
    const long long ph = static_cast<long long>(page) * ap.nkv + h;
    const int a = lo % kPage;  // rows of the page that were there before
    const float kold = a ? ap.kscale[ph] : 0.0f, vold = a ? ap.vscale[ph] : 0.0f;
    __syncthreads();
    for (int i = 0; i < static_cast<int>(blockDim.x) / 32; ++i) {
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
      const int c = lo + r * rows + row;
      if (r < ap.rounds && c < hi) {
        float vf[16];
        widen8<T>(*staged(heads + 1, r, 0), vf);
        widen8<T>(*staged(heads + 1, r, 1), vf + 8);
        const int at = c % kPage * HD + d0;
        *reinterpret_cast<uint2*>(kp + at) = codes8(kx[r], kinv);
        *reinterpret_cast<uint2*>(kp + at + kHalf) = codes8(kx[r] + 8, kinv);
        *reinterpret_cast<uint2*>(vp + at) = codes8(vf, vinv);
        *reinterpret_cast<uint2*>(vp + at + kHalf) = codes8(vf + 8, vinv);
      }
    }
  }
}

template <typename T, int HD, bool B8>
cudaError_t launch(AppendParams& ap, cudaStream_t s) {
  constexpr int kTokens = tokens<HD, B8>();
  ap.runs_per_seq = static_cast<int>((ap.seqs.max_q + 2ll * kTokens - 2) / kTokens);  // from a run's last slot on
  const int work = min(ap.seqs.max_q, kTokens) * (HD / 16);
  const int threads = min(kThreads, (work + 31) / 32 * 32);
  ap.rounds = (work + threads - 1) / threads;
  const uint32_t slot = ap.rounds * 2 * threads * 16;
  const int most = kStage / slot - 2;
  ap.head_ctas = (ap.group + most - 1) / most;
  ap.heads = (ap.group + ap.head_ctas - 1) / ap.head_ctas;
  ap.ctas = ap.nkv * ap.head_ctas;
  const long long ctas = static_cast<long long>(ap.seqs.n_seqs) * ap.runs_per_seq * ap.ctas;
  if (ctas > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  const uint32_t bytes = (ap.heads + 2) * slot;
  if (bytes > 47 * 1024) {  // 48 KB without it, the kernel's own variables among them
    const cudaError_t e = cudaFuncSetAttribute(kv_append_kernel<T, HD, B8>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kStage);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(kv_append_kernel<T, HD, B8>, dim3(static_cast<unsigned>(ctas)),
                    dim3(threads), bytes, s, ap);
}
template <typename T>
cudaError_t launch(AppendParams& ap, int hd, bool b8, cudaStream_t s) {
  if (hd == 128) return b8 ? launch<T, 128, true>(ap, s) : launch<T, 128, false>(ap, s);
  return b8 ? launch<T, 64, true>(ap, s) : launch<T, 64, false>(ap, s);
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
  ap.seqs.max_q = static_cast<int>(std::min<long long>(max_q, T));  // no sequence has more
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
  const cudaError_t e = bf16 ? launch<__nv_bfloat16>(ap, hd, kscale != nullptr, s)
                             : launch<__half>(ap, hd, kscale != nullptr, s);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace qa
