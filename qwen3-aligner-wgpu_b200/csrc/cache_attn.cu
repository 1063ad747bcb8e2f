// Attention over the 8-bit paged cache (codes and scales as kv_append writes
// them).
//
// Query i of sequence s (n new tokens, len cached ones, the new ones among
// them) sees cache indices c < len - n + i + 1 when causal, c < len otherwise:
//   s_c = scale kscale[page(c)] (q . kcode_c),  out = sum_c softmax(s)_c vscale[page(c)] vcode_c,
// lse = log sum_c exp(s_c); a row that sees nothing gets 0 and -inf.
#include <cuda_fp8.h>

#include "gemm_tc.cuh"
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
  int vec;      // q and out rows can be read and written 16 bytes at a time
  int cluster;  // CTAs that share a sequence's tokens
  unsigned* status;
};

// ------------------------------------------------------------ few query rows
// A query row is one (new token, head of the K/V head's group); row r of a
// sequence is token r / group, head r % group.  A CTA takes up to 8 * NT rows of
// one sequence and K/V head; a cluster of CTAs splits the cached tokens.
//
// Bound: the cache's bytes, read once (2 hd a token and head), so what matters
// is bytes in flight and instructions a byte.  Each of the CTA's warps streams
// its own slabs of 16 tokens through a private ring of kStages slabs
// (cp.async), without any CTA-wide barrier in the loop: 12 warps and three slabs
// of 4 KB each keep 144 KB in flight on an SM.
//
// Tokens are the M = 16 side of both products, so 8 rows cost one mma.sync
// m16n8k16 a 16x16 block and nothing is padded to 16 rows:
//   S^T [16 tokens][8 rows] = K [16][hd] . Q^T,
//   O^T [hd][8 rows]       += V^T [hd][16 tokens] . P^T.
// The order of the dims inside S^T's sum, and of the dims along O^T's rows, is
// free; it is chosen so that a thread reads its K and V operands as whole
// 16-byte units (16-byte units XOR-swizzled by token: no bank conflicts).
// V's pairs of tokens are formed bytewise before the conversion to f16 (one
// PRMT per two pairs); P^T comes from S^T's layout by movmatrix.
//
// e4m3 codes are exact in f16.  So are bf16 queries once a row is scaled by a
// power of two that brings its largest component to [2^14, 2^15): what falls
// into f16's subnormals lies 2^-39 below that.  P is rounded to f16.
//
// Softmax in base 2 with x = s log2(e): the running reference M of a row is
// over x + log2(vscale), so the page's scale goes into the exponent and P . V
// needs no scaling:  p = 2^(x + log2 vscale + kLift - M),  O = sum p vcode,
// l = sum p / vscale,  out = O / l.  M moves only when a value exceeds it by
// 2^kSlack (any reference gives the same quotient), so a slab usually needs one
// vote instead of a maximum across lanes; kLift keeps the small p of a long
// cache out of f16's subnormals and kLift + kSlack below its largest value.
constexpr int kWarps = 4;
constexpr int kStages = 4;
constexpr int kSlab = 16;  // tokens
constexpr float kLift = 8.0f, kSlack = 6.0f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxCluster = 16;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 8x8 transpose of 16-bit values across the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Two e4m3 codes (low byte first) as f16x2.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t w16) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w16), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
// 4 bytes global -> shared.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Base-2 logarithm and reciprocal of a page's V scale; a scale of 0 (a page of
// zeros written by someone else) counts as 2^-100.
__device__ __forceinline__ float usable_vscale(float v) { return fmaxf(v, 7.8886090522101181e-31f); }

// Four output values of a row.
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v, bool vec) {
  const uint32_t a = cvt2_rn<T>(make_float2(v.x, v.y)), b = cvt2_rn<T>(make_float2(v.z, v.w));
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(a, b);
  } else {
    const uint32_t w[2] = {a, b};
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = e[i];
  }
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kWarps * 32) cache_attn_rows(CacheAttnParams ap) {
  constexpr int R = 8 * NT;          // rows of a tile
  constexpr int kCpr = HD / 16;      // 16-byte units of a token
  constexpr int kKc = HD / 64;       // units of K a thread reads a token
  constexpr int kMt = HD / 16;       // 16-dim blocks of O^T
  constexpr int kPart = kSlab * HD;  // bytes of a slab's K (or V)
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_head[kWarps][kStages][4];  // K scale, V scale, tokens that may be seen
  __shared__ float s_m[kWarps][R], s_l[kWarps][R];
  __shared__ float s_cm[R], s_cl[R];            // the CTA's
  __shared__ float s_w[kMaxCluster][R], s_inv[R];

  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % ap.cluster, item = blockIdx.x / ap.cluster;
  const int s = item % ap.seqs.n_seqs, tile = item / ap.seqs.n_seqs;
  const int h = blockIdx.y;
  const SeqSpan sp = seq_span(ap.seqs, s, ap.T);
  if (!sp.ok) {
    if (tile == 0 && h == 0 && rank == 0 && threadIdx.x == 0 && ap.status) atomicOr(ap.status, kStatusBadShape);
    return;
  }
  const int group = ap.nq / ap.nkv;
  const int rows = min(R, sp.n * group - tile * R);
  if (rows <= 0) return;
  // tokens that the tile's last row sees, and the CTAs that share them
  const int past = sp.len - sp.n;  // + i + 1: seen by new token i
  const int seen = ap.causal ? min(sp.len, max(0, past + (tile * R + rows - 1) / group + 1)) : sp.len;
  const int slabs = (seen + kSlab - 1) / kSlab;
  const int cta = min(ap.cluster, max(1, (slabs + 2 * kWarps - 1) / (2 * kWarps)));
  if (rank >= cta) {
    if (cta > 1) {  // the cluster's barriers count this CTA too
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  // ---- queries: B operands, f16
  uint32_t qf[NT][HD / 16][2];
  float fac[NT][2];  // scale log2(e), undoing the row's own scaling, of columns 2t, 2t + 1
  int lim[NT][2];    // tokens that they see
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g, row = tile * R + r;
    float shift = 1.0f, undo = 1.0f;
    if (r < rows) {
      const T* qr = static_cast<const T*>(ap.q) + (sp.t0 + row / group) * ap.ldq +
                    static_cast<long long>(h * group + row % group) * HD;
      uint4 raw[kKc][2];
#pragma unroll
      for (int i = 0; i < kKc; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const T* src = qr + 16 * (kKc * t + i) + 8 * j;
          if (ap.vec) {
            raw[i][j] = *reinterpret_cast<const uint4*>(src);
          } else {
            T* e = reinterpret_cast<T*>(&raw[i][j]);
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = src[k];
          }
        }
      if constexpr (H16Traits<T>::kBf16) {
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < kKc; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int k = 0; k < 8; ++k)
              big = fmaxf(big, fabsf(h2f<T>(reinterpret_cast<const T*>(&raw[i][j])[k])));
        const unsigned quad = 0xFu << (lane & 28);
        big = fmaxf(big, __shfl_xor_sync(quad, big, 1));
        big = fmaxf(big, __shfl_xor_sync(quad, big, 2));
        const int e = (__float_as_int(big) >> 23) - 127;  // 2^e <= big
        // 2^(14 - e), in reach of a float for every finite row
        if (big > 0.0f && e < 128) {
          const int up = min(14 - e, 126);
          shift = __int_as_float((up + 127) << 23);
          undo = __int_as_float((127 - up) << 23);
        }
#pragma unroll
        for (int i = 0; i < kKc; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&raw[i][j]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const T* e2 = reinterpret_cast<const T*>(&w[k]);
              w[k] = cvt2_rn<__half>(make_float2(h2f<T>(e2[0]) * shift, h2f<T>(e2[1]) * shift));
            }
          }
      }
#pragma unroll
      for (int i = 0; i < kKc; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          qf[nt][4 * i + 2 * j][0] = raw[i][j].x;
          qf[nt][4 * i + 2 * j][1] = raw[i][j].y;
          qf[nt][4 * i + 2 * j + 1][0] = raw[i][j].z;
          qf[nt][4 * i + 2 * j + 1][1] = raw[i][j].w;
        }
    } else {
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) qf[nt][k][0] = qf[nt][k][1] = 0u;
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      fac[nt][c] = __shfl_sync(0xFFFFFFFFu, undo, 8 * t + 4 * c) * (ap.scale * kLog2e);
      const int cr = nt * 8 + 2 * t + c;
      // columns without a row: zeros that nothing masks and nobody reads
      lim[nt][c] = cr >= rows ? 0x7FFFFFFF : ap.causal ? max(0, past + (tile * R + cr) / group + 1) : sp.len;
    }
  }
  int all = 0x7FFFFFFF;  // tokens that every row sees
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) all = min(all, min(lim[nt][0], lim[nt][1]));
  all = __reduce_min_sync(0xFFFFFFFFu, all);

  // ---- the ring
  const uint32_t ring = smem_u32(smem) + warp * (kStages * 2 * kPart);
  const uint32_t head = smem_u32(&s_head[warp][0][0]);
  const int* bt = ap.seqs.block_tab + static_cast<long long>(s) * ap.seqs.max_pages;
  const int step = cta * kWarps;
  const int first = rank * kWarps + warp;
  auto fetch = [&](int slab, int stage) {
    if (slab < slabs) {
      int page = bt[slab / (kPage / kSlab)];
      int have = min(kSlab, sp.len - slab * kSlab);
      if (page < 0 || page >= ap.kv_pages) {
        if (lane == 0 && ap.status) atomicOr(ap.status, kStatusBadShape);
        page = have = 0;
      }
      const long long ph = static_cast<long long>(page) * ap.nkv + h;
      const long long at = ph * (kPage * HD) + (slab % (kPage / kSlab)) * kPart;
      const uint32_t dst = ring + stage * (2 * kPart);
#pragma unroll
      for (int i = 0; i < kSlab * kCpr / 32; ++i) {
        const int row = i * (32 / kCpr) + lane / kCpr, c = lane % kCpr;
        const uint32_t to = row * HD + 16 * (c ^ (HD == 128 ? row & 7 : (row >> 1) & 3));
        const uint32_t n = row < have ? 16 : 0;  // tokens past the end become zeros
        cp_async16(dst + to, ap.kpool + at + row * HD + 16 * c, n);
        cp_async16(dst + kPart + to, ap.vpool + at + row * HD + 16 * c, n);
      }
      if (lane < 2) cp_async4(head + stage * 16 + 4 * lane, (lane ? ap.vscale : ap.kscale) + ph);
      if (lane == 2) s_head[warp][stage][2] = __int_as_float(have);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(first + i * step, i);

  float o[kMt][NT][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < kMt; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
  }

  int stage = 0;
  for (int slab = first; slab < slabs; slab += step) {
    cp_async_wait<kStages - 2>();
    __syncwarp();  // this slab has landed; the slot refilled below was read by all
    fetch(slab + (kStages - 1) * step, (stage + kStages - 1) % kStages);
    const uint32_t kb = ring + stage * (2 * kPart), vb = kb + kPart;
    const float ks = s_head[warp][stage][0], vs = usable_vscale(s_head[warp][stage][1]);
    const int have = __float_as_int(s_head[warp][stage][2]);
    const float lv = log2f(vs), ivs = 1.0f / vs;

    float c[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.0f;
#pragma unroll
    for (int i = 0; i < kKc; ++i) {
      const int u = (kKc * t + i) ^ (HD == 128 ? g & 7 : (g >> 1) & 3);
      const uint4 ka = lds128(kb + g * HD + 16 * u), kc = lds128(kb + (g + 8) * HD + 16 * u);
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wc[4] = {kc.x, kc.y, kc.z, kc.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a[4] = {e4m3x2_f16x2(wa[j] & 0xFFFFu), e4m3x2_f16x2(wc[j] & 0xFFFFu),
                               e4m3x2_f16x2(wa[j] >> 16), e4m3x2_f16x2(wc[j] >> 16)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(c[nt], a, qf[nt][4 * i + j][0], qf[nt][4 * i + j][1]);
      }
    }

    // ---- softmax of tokens tok, tok + 8 (c[0..1], c[2..3]) for columns 2t, 2t + 1
    const int tok = slab * kSlab + g;
    const bool partial = (slab + 1) * kSlab > all || have < kSlab;
    bool over = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = fmaf(c[nt][e], ks * fac[nt][e & 1], lv);
        if (partial && (tok + (e >> 1) * 8 >= lim[nt][e & 1] || g + (e >> 1) * 8 >= have)) x = -INFINITY;
        c[nt][e] = x;
        over |= x > m[nt][e & 1] + kSlack;
      }
    if (__any_sync(0xFFFFFFFFu, over)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float big = fmaxf(c[nt][e], c[nt][e + 2]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, w));
          if (big > m[nt][e]) {
            const float a = ex2_approx(m[nt][e] - big);
            m[nt][e] = big;
            l[nt][e] *= a;
#pragma unroll
            for (int i = 0; i < kMt; ++i) {
              o[i][nt][e] *= a;
              o[i][nt][e + 2] *= a;
            }
          }
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float ref = m[nt][e & 1] == -INFINITY ? 0.0f : m[nt][e & 1];
        p[e] = ex2_approx(c[nt][e] + (kLift - ref));
        l[nt][e & 1] = fmaf(p[e], ivs, l[nt][e & 1]);
      }
      pb[nt][0] = movmatrix_trans(cvt2_rn<__half>(make_float2(p[0], p[1])));
      pb[nt][1] = movmatrix_trans(cvt2_rn<__half>(make_float2(p[2], p[3])));
    }

    // ---- O^T += V^T P^T: tokens 2t, 2t + 1, 2t + 8, 2t + 9 of dims 2 kMt g ..
    uint32_t v[4][HD / 32];  // the four tokens' codes
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = 2 * t + (k & 1) + (k >> 1) * 8;
      if constexpr (HD == 128) {
        const uint4 d = lds128(vb + row * HD + 16 * (g ^ (row & 7)));
        v[k][0] = d.x;
        v[k][1] = d.y;
        v[k][2] = d.z;
        v[k][3] = d.w;
      } else {
        const uint32_t at = vb + row * HD + 16 * ((g >> 1) ^ ((row >> 1) & 3)) + 8 * (g & 1);
        asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v[k][0]), "=r"(v[k][1]) : "r"(at));
      }
    }
    if (partial) {
      // 0 . NaN is NaN: a NaN code that some rows do not see is taken out, and
      // put into the results of the rows that do
      uint32_t nan[4];  // a bit for each of the thread's dims
      bool any = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        nan[k] = 0;
#pragma unroll
        for (int w = 0; w < HD / 32; ++w)
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (((v[k][w] >> (8 * b)) & 0x7Fu) == 0x7Fu) {
              nan[k] |= 1u << (4 * w + b);
              v[k][w] &= ~(0xFFu << (8 * b));
            }
        any |= nan[k] != 0;
      }
      if (__any_sync(0xFFFFFFFFu, any)) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          for (int from = 0; from < 4; ++from) {
            const uint32_t bits = __shfl_sync(0xFFFFFFFFu, nan[k], (lane & 28) + from);
            const int at = 2 * from + (k & 1) + (k >> 1) * 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (slab * kSlab + at < lim[nt][e] && at < have)
#pragma unroll
                  for (int i = 0; i < kMt; ++i) {
                    if (bits >> (2 * i) & 1) o[i][nt][e] = NAN;
                    if (bits >> (2 * i + 1) & 1) o[i][nt][e + 2] = NAN;
                  }
          }
      }
    }
#pragma unroll
    for (int w = 0; w < HD / 32; ++w)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t lo = __byte_perm(v[0][w], v[1][w], half ? 0x7362 : 0x5140);
        const uint32_t hi = __byte_perm(v[2][w], v[3][w], half ? 0x7362 : 0x5140);
        const uint32_t a[4] = {e4m3x2_f16x2(lo & 0xFFFFu), e4m3x2_f16x2(lo >> 16),
                               e4m3x2_f16x2(hi & 0xFFFFu), e4m3x2_f16x2(hi >> 16)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(o[2 * w + half][nt], a, pb[nt][0], pb[nt][1]);
      }
    stage = (stage + 1) % kStages;
  }

  // ---- join the warps: O [warp][row][dim] over the ring, scaled to one reference
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], w);
      if (g == 0) {
        s_m[warp][nt * 8 + 2 * t + e] = m[nt][e];
        s_l[warp][nt * 8 + 2 * t + e] = l[nt][e];
      }
    }
  cp_async_wait<0>();
  __syncthreads();
  float* obuf = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * t + e;
      float big = s_m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) big = fmaxf(big, s_m[w][r]);
      const float ref = big == -INFINITY ? 0.0f : big;
      const float a = ex2_approx(m[nt][e] - ref);
      float* dst = obuf + (warp * R + r) * HD + 2 * kMt * g;
#pragma unroll
      for (int i = 0; i < kMt / 2; ++i)
        *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(
            o[2 * i][nt][e] * a, o[2 * i][nt][e + 2] * a, o[2 * i + 1][nt][e] * a, o[2 * i + 1][nt][e + 2] * a);
      if (warp == 0 && g == 0) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += s_l[w][r] * ex2_approx(s_m[w][r] - ref);
        s_cm[r] = big;
        s_cl[r] = sum;
      }
    }
  __syncthreads();
  if (cta > 1) {
    for (int i = threadIdx.x; i < R * HD / 4; i += kWarps * 32) {
      float4 v = reinterpret_cast<float4*>(obuf)[i];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 x = reinterpret_cast<float4*>(obuf + w * R * HD)[i];
        v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
      }
      reinterpret_cast<float4*>(obuf)[i] = v;
    }
    cluster_sync();  // every part is in its CTA's shared memory
  }
  // ---- join the cluster: each CTA finishes a share of the values, parts in rank order
  if (threadIdx.x < rows) {
    const int r = threadIdx.x;
    float big = s_cm[r], sum = s_cl[r];
    if (cta > 1) {
      const uint32_t am = smem_u32(&s_cm[r]), al = smem_u32(&s_cl[r]);
      big = -INFINITY;
      for (int k = 0; k < cta; ++k) big = fmaxf(big, ld_cluster_f32(mapa_shared(am, k)));
      const float ref = big == -INFINITY ? 0.0f : big;
      sum = 0.0f;
      for (int k = 0; k < cta; ++k) {
        const float a = ex2_approx(ld_cluster_f32(mapa_shared(am, k)) - ref);
        s_w[k][r] = a;
        sum += a * ld_cluster_f32(mapa_shared(al, k));
      }
    }
    s_inv[r] = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (rank == 0 && ap.lse) {
      const int row = tile * R + r;
      ap.lse[(sp.t0 + row / group) * ap.nq + h * group + row % group] =
          sum == 0.0f ? -INFINITY : (big - kLift + log2f(sum)) * 0.69314718055994531f;
    }
  }
  __syncthreads();
  for (int i = rank * (kWarps * 32) + threadIdx.x; i < rows * (HD / 4); i += cta * (kWarps * 32)) {
    const int r = i / (HD / 4), row = tile * R + r;
    float4 v;
    if (cta > 1) {
      v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const uint32_t at = smem_u32(obuf + 4 * i);
      for (int k = 0; k < cta; ++k) {
        const float4 x = ld_cluster_f32x4(mapa_shared(at, k));
        const float a = s_w[k][r];
        v = make_float4(fmaf(a, x.x, v.x), fmaf(a, x.y, v.y), fmaf(a, x.z, v.z), fmaf(a, x.w, v.w));
      }
    } else {
      v = reinterpret_cast<float4*>(obuf)[i];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 x = reinterpret_cast<float4*>(obuf + w * R * HD)[i];
        v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
      }
    }
    const float inv = s_inv[r];
    store4(static_cast<T*>(ap.out) + (sp.t0 + row / group) * ap.ldo +
               static_cast<long long>(h * group + row % group) * HD + 4 * (i % (HD / 4)),
           make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), ap.vec);
  }
  if (cta > 1) cluster_sync();  // nobody leaves while its part is being read
}

template <typename T, int HD, int NT>
cudaError_t launch_rows(CacheAttnParams ap, int max_q, int max_kv, cudaStream_t s) {
  constexpr int R = 8 * NT;
  constexpr int kSmem = kWarps * kStages * 2 * kSlab * HD;  // = the joined O, 4 * kWarps * R * HD at NT = 4
  static_assert(kSmem >= 4 * kWarps * R * HD, "the warps' O fits the ring");
  const int group = ap.nq / ap.nkv;
  const long long tiles = (static_cast<long long>(max_q) * group + R - 1) / R;
  const long long x = tiles * ap.seqs.n_seqs;
  // Split until the machine is several times full, while a warp keeps enough slabs.
  const long long base = x * ap.nkv;
  const long long want = 12ll * device_sm_count();
  int c = 1;
  while (c < kMaxCluster && base * c < want && static_cast<long long>(c) * 2 * kWarps * kSlab * 2 <= max_kv) c *= 2;
  ap.cluster = c;
  if (x * c > 0x7FFFFFFFll || ap.nkv > 65535) return cudaErrorInvalidValue;
  auto k = cache_attn_rows<T, HD, NT>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e == cudaSuccess && c > 8) e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(x * c), ap.nkv);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = c;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k, ap);
}

template <typename T, int HD>
cudaError_t launch_any(const CacheAttnParams& ap, int max_q, int max_kv, cudaStream_t s) {
  const long long rows = static_cast<long long>(max_q) * (ap.nq / ap.nkv);
  if (rows <= 8) return launch_rows<T, HD, 1>(ap, max_q, max_kv, s);
  if (rows <= 16) return launch_rows<T, HD, 2>(ap, max_q, max_kv, s);
  if (rows <= 24) return launch_rows<T, HD, 3>(ap, max_q, max_kv, s);
  return launch_rows<T, HD, 4>(ap, max_q, max_kv, s);
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
  ap.vec = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0) &&
           ((ldq | ldo) % 8 == 0);
  cudaError_t e;
  if (bf16)
    e = hd == 128 ? launch_any<__nv_bfloat16, 128>(ap, max_q, max_kv, s)
                  : launch_any<__nv_bfloat16, 64>(ap, max_q, max_kv, s);
  else
    e = hd == 128 ? launch_any<__half, 128>(ap, max_q, max_kv, s)
                  : launch_any<__half, 64>(ap, max_q, max_kv, s);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace qa
