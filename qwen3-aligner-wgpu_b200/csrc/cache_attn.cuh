// What the two kernels of cache_attention share: its parameters, the codes'
// conversion, where results go, and the kernel that joins the parts of a sequence.
#pragma once

#include <algorithm>

#include "kernels.cuh"
#include "sm100.cuh"

namespace qa {

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
  int tiles_max;       // tiles of a sequence of max_q tokens
  float* parts;        // workspace: place_floats for each unit (few-row kernel), or each sequence and K/V head
  long long cap_units; // such places in the workspace
  long long place_floats;
  int cap_parts;       // parts a unit of the few-row kernel has place for
  int part_rows, part_stride;  // most rows of a part, its floats
  int half_stride;     // floats of a part of one tile of rows (tcgen05 kernel)
  unsigned* status;
};

namespace {

constexpr int kPage = 64;
constexpr float kLog2e = 1.4426950408889634f;

// Softmax in base 2 with x = s log2(e): the running reference M of a row is over
// x + log2(vscale), so the page's scale goes into the exponent and P . V needs no
// scaling:  p = 2^(x + log2 vscale + kLift - M),  O = sum p vcode,
// l = sum p / vscale,  out = O / l.  M moves only when a value exceeds it by
// 2^kSlack (any reference gives the same quotient); kLift keeps the small p of a
// long cache out of f16's subnormals, and 2^(kLift + kSlack) is below its largest
// value.
//
// P is f16 because the matrix instructions take 16 bits and V's codes are exact in
// f16; m, l and O stay in f32.  A p is off by 2^-11 of itself, or by 2^-25 where it
// is below 2^-14, which is 2^-22 or less of the row's largest: a token that counts
// that little beside another (its probability times its page's V scale) keeps fewer
// bits, and is lost below 2^-33.  Against 64 bits, outputs of 421 tokens are off by
// 2.3e-4 of their norm in f16 (2.1e-4 with P in 32 bits: the outputs' own rounding)
// and by 1.7e-3 in bf16 either way.
constexpr float kLift = 8.0f, kSlack = 6.0f;

// Four e4m3 codes (low byte first) as two f16x2; NaN codes stay NaN.
__device__ __forceinline__ void e4m3x4_f16x2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// A tile's rows of one sequence and K/V head.
struct UnitAt {
  int s, tile, h;
  long long t0;  // the sequence's first row of q and out
};

// A unit's parts: m and l of l_at rows (a multiple of four), O.
struct PartsAt {
  float* base;
  int stride, l_at;
};
__host__ __device__ __forceinline__ int padded_rows(int rows) { return (rows + 3) & ~3; }
__host__ __device__ __forceinline__ int part_floats(int rows, int hd) { return 2 * padded_rows(rows) + rows * hd; }

// Row `row` of a sequence is done: its lse; returns what its O is multiplied by.
__device__ __forceinline__ float close_row(const CacheAttnParams& ap, const UnitAt& at, int row,
                                           float big, float sum) {
  const int group = ap.nq / ap.nkv;
  if (ap.lse)
    ap.lse[(at.t0 + row / group) * ap.nq + at.h * group + row % group] =
        sum == 0.0f ? -INFINITY : (big - kLift + log2f(sum)) * 0.69314718055994531f;
  return sum == 0.0f ? 0.0f : 1.0f / sum;
}

template <typename T, int HD>
__device__ __forceinline__ void finish_row(const CacheAttnParams& ap, const UnitAt& at, int row, int dim,
                                           float4 v, float inv) {
  const int group = ap.nq / ap.nkv;
  store4(static_cast<T*>(ap.out) + (at.t0 + row / group) * ap.ldo +
             static_cast<long long>(at.h * group + row % group) * HD + dim,
         make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), ap.vec);
}

// Joins the parts of the units that left any (Plan::parts), four dims of a row a
// lane (hd 64: two parts a warp at a time).  Few rows of many parts (the few-row
// kernel's): a CTA's warps share a row, each summing every eighth part, and are
// then summed in turn.  Many rows of few parts (kAlone): a warp a row.  Bound by
// latency: a part's row is one line of 4 hd bytes.
constexpr int kJoinWarps = 8;
// Parts up to which a warp joins a row alone.  24 rows a head (16/8 heads of 128), in
// all, against a CTA a row: 16 sessions over 8192 tokens, 11 parts, 103 and 124 us;
// over 24,576, 32 parts, 259 and 276, but one session 36 and 32.  More parts: one
// session over 50,000, 66 parts, 73 and 60; four over 100,000 292 and 276.
constexpr int kJoinAlone = 32;

// grid: (sequences x tiles, K/V heads, rows, or rows / 8)
template <typename T, int HD, typename Plan>
__global__ void __launch_bounds__(kJoinWarps * 32, Plan::kAlone ? 4 : 2) cache_attn_join(const __grid_constant__ CacheAttnParams ap) {
  constexpr int kLanes = HD / 4, kPer = 32 / kLanes;  // lanes of a part, parts of a warp at once
  __shared__ float s_l[kJoinWarps];
  __shared__ float4 s_o[kJoinWarps][kLanes];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, s = blockIdx.x / ap.tiles_max, tile = blockIdx.x % ap.tiles_max;
  pdl_wait();
  pdl_trigger();
  const int group = ap.nq / ap.nkv;
  const SeqSpan sp = seq_span(ap.seqs, s, ap.T);
  if (!sp.ok) return;
  const int rows = min(Plan::kRows, sp.n * group - tile * Plan::kRows);
  if (rows <= 0) return;
  const int n = Plan::parts(ap, sp, s, tile);
  if (n == 0) return;
  constexpr bool alone = Plan::kAlone;
  const UnitAt at{s, tile, h, sp.t0};
  const PartsAt parts = Plan::place(ap, sp, at);
  // the CTA's warps share row blockIdx.z, or take rows of their own
  for (int r = alone ? kJoinWarps * blockIdx.z + warp : blockIdx.z; r < rows; r += (alone ? kJoinWarps : 1) * gridDim.z) {
  const int o_at = 2 * parts.l_at + r * HD;
  const int first = (alone ? 0 : warp * kPer) + lane / kLanes, step = alone ? kPer : kPer * kJoinWarps;
  const int d = lane % kLanes;
  float big = -INFINITY;
  for (int k = alone ? lane : threadIdx.x; k < n; k += alone ? 32 : 32 * kJoinWarps)
    big = fmaxf(big, __ldcg(parts.base + static_cast<long long>(k) * parts.stride + r));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
  if constexpr (!alone) {
    if (lane == 0) s_l[warp] = big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) big = fmaxf(big, s_l[w]);
    __syncthreads();
  }
  const float ref = big == -INFINITY ? 0.0f : big;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
  constexpr int kBatch = alone ? 4 : 8;  // parts whose loads are in flight together
  for (int k0 = first; k0 < n; k0 += kBatch * step) {
    float4 y[kBatch];
    float pm[kBatch], pl[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float* part = parts.base + static_cast<long long>(k0 + i * step) * parts.stride;
      y[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      pm[i] = pl[i] = 0.0f;
      if (k0 + i * step < n) {
        y[i] = __ldcg(reinterpret_cast<const float4*>(part + o_at + 4 * d));
        pm[i] = __ldcg(part + r);
        pl[i] = __ldcg(part + parts.l_at + r);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (k0 + i * step < n) {
        const float a = ex2_approx(pm[i] - ref);
        sum = fmaf(a, pl[i], sum);
        v = make_float4(fmaf(a, y[i].x, v.x), fmaf(a, y[i].y, v.y), fmaf(a, y[i].z, v.z), fmaf(a, y[i].w, v.w));
      }
  }
  if constexpr (kPer == 2) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
    v = make_float4(v.x + __shfl_xor_sync(0xFFFFFFFFu, v.x, 16), v.y + __shfl_xor_sync(0xFFFFFFFFu, v.y, 16),
                    v.z + __shfl_xor_sync(0xFFFFFFFFu, v.z, 16), v.w + __shfl_xor_sync(0xFFFFFFFFu, v.w, 16));
  }
  if constexpr (!alone) {
    if (lane < kLanes) s_o[warp][d] = v;
    if (lane == 0) s_l[warp] = sum;
    __syncthreads();
    if (warp > 0) return;
    v = s_o[0][d];
    sum = s_l[0];
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) {
      const float4 y = s_o[w][d];
      v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
      sum += s_l[w];
    }
  }
  if (lane < kLanes) {
    const int row = tile * Plan::kRows + r;
    if (d == 0) close_row(ap, at, row, big, sum);
    finish_row<T, HD>(ap, at, row, 4 * d, v, sum == 0.0f ? 0.0f : 1.0f / sum);
  }
  }
}

template <typename T, int HD, typename Plan>
cudaError_t launch_join(const CacheAttnParams& ap, cudaStream_t s) {
  const long long x = static_cast<long long>(ap.seqs.n_seqs) * ap.tiles_max;
  if (x > 0x7FFFFFFFll || ap.nkv > 65535) return cudaErrorInvalidValue;
  const int z = Plan::kAlone ? std::min((ap.part_rows - 1) / kJoinWarps + 1, 8) : ap.part_rows;
  return launch_pdl(cache_attn_join<T, HD, Plan>, dim3(static_cast<unsigned>(x), ap.nkv, z), dim3(kJoinWarps * 32), 0,
                    s, ap);
}

}  // namespace

// Bytes of units * nkvh places, at most 1 GiB: sequences past it are not split.
inline long long places_bytes(long long units, int nkvh, long long place_floats) {
  constexpr long long kMost = 1ll << 30;
  const long long one = 4 * place_floats;
  return units > kMost / one / nkvh ? kMost : units * nkvh * one;
}

// The two kernels' launches, and the workspace that each asks for.
int cache_attention_rows(const CacheAttnParams& ap, int hd, bool bf16, int max_kv, void* ws,
                         long long ws_bytes, cudaStream_t s);
int cache_attention_tiles(const CacheAttnParams& ap, int hd, bool bf16, int max_kv, void* ws,
                          long long ws_bytes, cudaStream_t s);
long long cache_rows_workspace(int nqh, int nkvh, int hd, int n_seqs, int max_q, int max_kv);
long long cache_tiles_workspace(int nqh, int nkvh, int hd, int n_seqs, int max_q, int max_kv);

}  // namespace qa
