// y = x W^T (+ bias) with W in 4 bits:
//   W[n][k] = scale[n][k / g] (code[n][k] - zero[n][k / g]),   zero = 8 where none is given.
// wq [N][K / 2] bytes, the even k of a pair in the low nibble.
//
// Built for few rows of x, where the weights' bytes are the bound (K / 2 a row
// of W, each read once).  A warp owns 16 rows of W (one mma.sync M block) and
// walks K in steps of 128: a thread's 16 bytes of a W row are 32 weights, a
// quad's four threads cover the step, and eight rows a load keep whole 64-byte
// lines in use.  The codes become 16-bit integers by bit work (the mantissa of
// 1024 or, for bf16, 128) less the zero, exactly; x is a 16-bit operand as it is;
// a group's sum is exact products in f32 and is scaled in f32, so nothing is
// rounded before the output.
//
// The order of k inside a step is free as long as both operands agree.  A word's
// nibbles leave the bit work as the pairs (0,4) (1,5) (2,6) (3,7); x is put in
// that order once, when the CTA copies its slice of x into shared memory, 16
// bytes to a thread and word.
//
// The CTA's warps split K (slices of whole steps) and their sums are joined in
// shared memory in warp order: no atomics, the same bits each time.
#include <algorithm>

#include "gemm_tc.cuh"
#include "kernels.cuh"
#include "sm100.cuh"

namespace qa {

namespace {

constexpr int kStep = 128;  // k of a step
constexpr int kRows = 16;   // rows of W a warp

struct W4Params {
  const void* x;
  long long ldx;
  int M, N, K, group;
  const uint8_t* wq;
  long long ldw;  // bytes
  const void* scales;
  const uint8_t* zeros;
  const float* bias;
  void* out;
  long long ldo;
  int vec_x, vec_w;  // rows of x / W can be read 16 bytes at a time
};

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (H16Traits<T>::kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Nibbles i and i + 4 of w (already shifted right by 4 i) less the zero, as two
// 16-bit values.  1024 + code is exact in f16, 128 + code in bf16, and so is the
// difference of two such values.
template <typename T>
__device__ __forceinline__ uint32_t nibbles(uint32_t w, uint32_t zero2) {
  constexpr uint32_t kBase = H16Traits<T>::kBf16 ? 0x43004300u : 0x64006400u;
  const uint32_t v = (w & 0x000F000Fu) | kBase;
  if constexpr (H16Traits<T>::kBf16) {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                     *reinterpret_cast<const __nv_bfloat162*>(&zero2));
    return *reinterpret_cast<const uint32_t*>(&d);
  } else {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&zero2));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t zero_pair(uint32_t z) {
  constexpr uint32_t kBase = H16Traits<T>::kBf16 ? 0x4300u : 0x6400u;
  return (kBase | z) * 0x10001u;
}

// x in shared memory: for each step and token, 16 chunks of 16 bytes (word w,
// quad lane t at chunk 4 w + t), a token's 256 bytes followed by the next's;
// tokens are 272 bytes apart, so that the eight lanes of a 16-byte access (two
// tokens, four chunks) touch 32 different banks.
constexpr int kXTok = 272;

template <typename T, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) w4_kernel(W4Params wp) {
  constexpr int kTok = 8 * NT;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * kTok;
  const int steps = (wp.K + kStep - 1) / kStep, groups = wp.K / wp.group;
  const int gps = kStep / wp.group;  // groups of a step: 1, 2 or 4
  const int n0 = blockIdx.x * kRows + g;
  pdl_wait();
  pdl_trigger();

  float acc[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;

  // rows past the end read the last row; their sums are not stored
  const int r0 = min(n0, wp.N - 1), r1 = min(n0 + 8, wp.N - 1);
  const uint8_t* w0 = wp.wq + r0 * wp.ldw + 16 * t;
  const uint8_t* w1 = wp.wq + r1 * wp.ldw + 16 * t;
  const T* s0 = static_cast<const T*>(wp.scales) + static_cast<long long>(r0) * groups;
  const T* s1 = static_cast<const T*>(wp.scales) + static_cast<long long>(r1) * groups;
  const uint8_t* z0 = wp.zeros ? wp.zeros + static_cast<long long>(r0) * groups : nullptr;
  const uint8_t* z1 = wp.zeros ? wp.zeros + static_cast<long long>(r1) * groups : nullptr;

  // 32 weights from k on; past K nothing is read (x is zero there)
  auto load_w = [&](const uint8_t* p, int step) {
    const int k = step * kStep + 32 * t;
    uint4 d = make_uint4(0, 0, 0, 0);
    if (k < wp.K) {
      if (wp.vec_w) {
        d = __ldg(reinterpret_cast<const uint4*>(p + step * (kStep / 2)));
      } else {
        uint8_t* b = reinterpret_cast<uint8_t*>(&d);
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = p[step * (kStep / 2) + i];
      }
    }
    return d;
  };
  uint8_t* xs = smem + warp * (kTok * kXTok);  // the warp's current step of x
  for (int step = warp; step < steps; step += WARPS) {
    const uint4 wa = load_w(w0, step), wb = load_w(w1, step);
    // the step's x: chunk c of a token holds k = 32 (c % 4) + 8 (c / 4) .. + 8
    __syncwarp();
    for (int i = lane; i < kTok * 16; i += 32) {
      const int m = i / 16, c = i % 16, k = step * kStep + 32 * (c & 3) + 8 * (c >> 2);
      uint4 d = make_uint4(0, 0, 0, 0);
      if (m0 + m < wp.M && k < wp.K) {
        const T* src = static_cast<const T*>(wp.x) + (m0 + m) * wp.ldx + k;
        if (wp.vec_x) {
          d = __ldg(reinterpret_cast<const uint4*>(src));
        } else {
          T* e = reinterpret_cast<T*>(&d);
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = src[j];
        }
        // (0 1)(2 3)(4 5)(6 7) -> (0 4)(1 5)(2 6)(3 7)
        d = make_uint4(__byte_perm(d.x, d.z, 0x5410), __byte_perm(d.x, d.z, 0x7632),
                       __byte_perm(d.y, d.w, 0x5410), __byte_perm(d.y, d.w, 0x7632));
      }
      *reinterpret_cast<uint4*>(xs + m * kXTok + 16 * c) = d;
    }
    __syncwarp();
    const uint32_t va[4] = {wa.x, wa.y, wa.z, wa.w}, vb[4] = {wb.x, wb.y, wb.z, wb.w};
    // A lane's 32 weights lie in one group (32, 64 or 128 of them), but the four
    // lanes' may lie in several: a group's sum then needs its lanes alone, so the
    // scale is applied to the operand's products by splitting the step's MMAs by
    // lane: lanes of other groups feed zeros.
    for (int gi = 0; gi < gps; ++gi) {
      const int gr = step * gps + gi;
      if (gr >= groups) break;
      const bool mine = gps == 1 || (gps == 2 ? (t >> 1) == gi : t == gi);
      const uint32_t za = zero_pair<T>(z0 ? z0[gr] : 8u), zb = zero_pair<T>(z1 ? z1[gr] : 8u);
      float c[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a0[4], a1[4];
        a0[0] = mine ? nibbles<T>(va[w], za) : 0u;
        a0[1] = mine ? nibbles<T>(vb[w], zb) : 0u;
        a0[2] = mine ? nibbles<T>(va[w] >> 4, za) : 0u;
        a0[3] = mine ? nibbles<T>(vb[w] >> 4, zb) : 0u;
        a1[0] = mine ? nibbles<T>(va[w] >> 8, za) : 0u;
        a1[1] = mine ? nibbles<T>(vb[w] >> 8, zb) : 0u;
        a1[2] = mine ? nibbles<T>(va[w] >> 12, za) : 0u;
        a1[3] = mine ? nibbles<T>(vb[w] >> 12, zb) : 0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 b = *reinterpret_cast<const uint4*>(xs + (8 * nt + g) * kXTok + 16 * (4 * w + t));
          mma_16816<T>(c[nt], a0, b.x, b.y);
          mma_16816<T>(c[nt], a1, b.z, b.w);
        }
      }
      const float sa = h2f<T>(s0[gr]), sb = h2f<T>(s1[gr]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        acc[nt][0] = fmaf(sa, c[nt][0], acc[nt][0]);
        acc[nt][1] = fmaf(sa, c[nt][1], acc[nt][1]);
        acc[nt][2] = fmaf(sb, c[nt][2], acc[nt][2]);
        acc[nt][3] = fmaf(sb, c[nt][3], acc[nt][3]);
      }
    }
  }
  // ---- join the warps' sums: [warp][row][token]
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      red[(warp * kTok + 8 * nt + 2 * t + (e & 1)) * kRows + g + (e >> 1) * 8] = acc[nt][e];
  __syncthreads();
  for (int i = threadIdx.x; i < kTok * kRows; i += WARPS * 32) {
    const int m = m0 + i / kRows, n = blockIdx.x * kRows + i % kRows;
    if (m >= wp.M || n >= wp.N) continue;
    float v = red[i];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) v += red[w * (kTok * kRows) + i];
    static_cast<T*>(wp.out)[m * wp.ldo + n] = f2h<T>(v + (wp.bias ? wp.bias[n] : 0.0f));
  }
}

template <typename T, int NT, int WARPS>
cudaError_t launch(const W4Params& wp, cudaStream_t s) {
  const dim3 grid((wp.N + kRows - 1) / kRows, (wp.M + 8 * NT - 1) / (8 * NT));
  constexpr int kSmem = WARPS * 8 * NT * kXTok;
  static_assert(kSmem >= WARPS * 8 * NT * kRows * 4, "the sums fit x's place");
  if (grid.y > 65535) return cudaErrorInvalidValue;
  auto k = w4_kernel<T, NT, WARPS>;
  if (kSmem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(k, grid, dim3(WARPS * 32), kSmem, s, wp);
}

template <typename T>
cudaError_t launch_any(const W4Params& wp, cudaStream_t s) {
  if (wp.M <= 8) return launch<T, 1, 4>(wp, s);
  if (wp.M <= 16) return launch<T, 2, 4>(wp, s);
  return launch<T, 4, 4>(wp, s);
}

}  // namespace

int w4_linear(const void* x, long long ldx, int M, int K, const uint8_t* wq, long long ldw, int N,
              int group, const void* scales, const uint8_t* zeros, const float* bias, void* out,
              long long ldo, bool bf16, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  W4Params wp{x, ldx, M, N, K, group, wq, ldw, scales, zeros, bias, out, ldo, 0, 0};
  wp.vec_x = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0;
  wp.vec_w = reinterpret_cast<uintptr_t>(wq) % 16 == 0 && ldw % 16 == 0;
  const cudaError_t e = bf16 ? launch_any<__nv_bfloat16>(wp, s) : launch_any<__half>(wp, s);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace qa
