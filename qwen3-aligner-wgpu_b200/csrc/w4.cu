// y = x W^T (+ bias) with W in 4 bits:
//   W[n][k] = scale[n][k / g] (code[n][k] - zero[n][k / g]),   zero = 8 where none is given.
// wq [N][K / 2] bytes, the even k of a pair in the low nibble.
//
// Built for few rows of x, where the weights' bytes are the bound (K / 2 a row
// of W, each read once).  A warp takes 32 rows of W (two mma.sync M blocks) and
// walks K in steps of 128: a thread's 16 bytes of a W row are 32 weights, a
// quad's four threads cover the step, and a load of eight rows keeps whole
// 64-byte pieces in use; kAhead steps are on their way in registers.  The codes
// become 16-bit integers by bit work (in the mantissa of a power of two) less the
// zero, exactly; x is a 16-bit operand as it is; a group's sum is exact products
// in f32 and is scaled in f32, so nothing is rounded before the output.
//
// The order of k inside a step is free as long as both operands agree.  A word's
// nibbles leave the bit work as the pairs (0,4) (1,5) (2,6) (3,7); x is put in
// that order when the CTA copies it into shared memory, as the 16 bytes that a
// thread needs for a word.  x stays there for all rows that the CTA takes, if it
// fits; a longer K goes through in chunks.
//
// With few rows of W a CTA's eight warps share 32 rows and split K, and their
// sums are joined in shared memory in warp order; with many each warp has rows
// of its own.  No atomics, the same bits each time.
#include <algorithm>
#include <type_traits>

#include "gemm_tc.cuh"
#include "kernels.cuh"
#include "sm100.cuh"

namespace qa {

namespace {

constexpr int kStep = 128;   // k of a step
constexpr int kRows = 32;    // rows of W a warp
constexpr int kWarps = 8;
constexpr int kAhead = 2;    // steps of W on their way
constexpr int kXBytes = 96 * 1024;  // most of x in shared memory: two CTAs an SM

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
  int slices;        // warps that share rows of W: 1, 2, 4 or 8
  int per;           // steps of a slice
  int chunk;         // steps of every slice that have x in shared memory at a time
  int vec_o;         // eight adjacent outputs can be written at once
};

// c = a b (FIRST) or c += a b
template <typename T, bool FIRST>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  const float i0 = FIRST ? 0.0f : c[0], i1 = FIRST ? 0.0f : c[1], i2 = FIRST ? 0.0f : c[2], i3 = FIRST ? 0.0f : c[3];
  if constexpr (H16Traits<T>::kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(i0), "f"(i1), "f"(i2), "f"(i3));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(i0), "f"(i1), "f"(i2), "f"(i3));
}

// The pairs of nibbles (0,4) (1,5) (2,6) (3,7) of a word, less the zero, as
// 16-bit values.  f16: 1024 + code with the code in the low four bits of the
// mantissa, 64 + code with it four bits higher, so one shift serves two pairs.
// bf16: 128 + code.  All exact, and so are the differences.
template <typename T>
struct Zero {  // base + zero, twice
  uint32_t lo, hi;
  __device__ __forceinline__ explicit Zero(uint32_t z) {
    if constexpr (H16Traits<T>::kBf16) {
      lo = hi = (0x4300u | z) * 0x10001u;
    } else {
      lo = (0x6400u | z) * 0x10001u;
      hi = (0x5400u | z << 4) * 0x10001u;
    }
  }
};
// The masks and bases in registers: an instruction takes one constant, and
// (w & mask) | base is one instruction only when the other operand is a register.
template <typename T>
struct Bits {
  uint32_t mask_lo, base_lo, mask_hi, base_hi;
  __device__ __forceinline__ Bits() {
    asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(mask_lo));
    asm volatile("mov.b32 %0, %1;" : "=r"(base_lo) : "n"(H16Traits<T>::kBf16 ? 0x43004300 : 0x64006400));
    asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(mask_hi));
    asm volatile("mov.b32 %0, 0x54005400;" : "=r"(base_hi));
  }
};
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t base) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(base));
  return d;
}
template <typename T>
__device__ __forceinline__ void weights8(uint32_t w, const Zero<T>& z, const Bits<T>& k, uint32_t (&out)[4]) {
  if constexpr (H16Traits<T>::kBf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = and_or(w >> (4 * i), k.mask_lo, k.base_lo);
      const __nv_bfloat162 d =
          __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&z.lo));
      out[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = i < 2 ? w : w >> 8;
      const uint32_t v = i & 1 ? and_or(u, k.mask_hi, k.base_hi) : and_or(u, k.mask_lo, k.base_lo);
      const __half2 d =
          __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(i & 1 ? &z.hi : &z.lo));
      out[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

// GPS: groups of a step, 1, 2 or 4 (group 128, 64, 32).  FAST: rows of x and W can
// be read 16 bytes at a time, a step's scales and zeros at once, and K is whole
// steps.
template <typename T, int NT, int GPS, bool FAST>
__global__ void __launch_bounds__(kWarps * 32, GPS * NT <= 2 ? 2 : 1) w4_kernel(const __grid_constant__ W4Params wp) {
  constexpr int kTok = 8 * NT;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * kTok, toks = min(kTok, wp.M - m0);
  const int steps = (wp.K + kStep - 1) / kStep, groups = wp.K / wp.group;
  const int slice = warp % wp.slices, tiles = kWarps / wp.slices;
  // x: [slice][step][token][16 units of 16 bytes: word w of lane t at 4 w + t, odd
  // tokens with w ^ 1], so that an access of eight lanes (two tokens, four units)
  // meets 32 different banks; then the warps' sums
  constexpr int kTokBytes = 2 * kStep;
  const int step_bytes = toks * kTokBytes, slice_bytes = wp.chunk * step_bytes;
  float* red = reinterpret_cast<float*>(smem + wp.slices * slice_bytes);
  const Bits<T> bits;
  pdl_wait();
  pdl_trigger();

  // steps [l0, l0 + chunk) of every slice; a thread has one unit and token
  auto stage = [&](int l0) {
    const int c = threadIdx.x % 16;
    for (int m = threadIdx.x / 16; m < toks; m += kWarps * 2) {
      const T* row = static_cast<const T*>(wp.x) + (m0 + m) * wp.ldx + 32 * (c & 3) + 8 * (c >> 2);
      uint8_t* to = smem + m * kTokBytes + 16 * (c ^ 4 * (m & 1));
      for (int sl = 0; sl < wp.slices; ++sl) {
        const int n = min(wp.chunk, wp.per - l0), st0 = sl * wp.per + l0;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
          const int k = (st0 + i) * kStep;
          uint4 d = make_uint4(0, 0, 0, 0);  // past K
          if (FAST ? st0 + i < steps : k + 32 * (c & 3) + 8 * (c >> 2) < wp.K) {
            if (FAST || wp.vec_x) {
              d = __ldg(reinterpret_cast<const uint4*>(row + k));
            } else {
              T* e = reinterpret_cast<T*>(&d);
#pragma unroll
              for (int j = 0; j < 8; ++j) e[j] = row[k + j];
            }
          }
          // (0 1)(2 3)(4 5)(6 7) -> (0 4)(1 5)(2 6)(3 7)
          *reinterpret_cast<uint4*>(to + sl * slice_bytes + i * step_bytes) =
              make_uint4(__byte_perm(d.x, d.z, 0x5410), __byte_perm(d.x, d.z, 0x7632),
                         __byte_perm(d.y, d.w, 0x5410), __byte_perm(d.y, d.w, 0x7632));
        }
      }
    }
  };

  const bool once = wp.chunk >= wp.per;  // x stays for all rows
  const int first = slice * wp.per, own = min(wp.per, steps - first);  // own may be < 1
  const uint8_t* xs = smem + slice * slice_bytes + g * kTokBytes + 16 * t;
  const int even = 64 * (g & 1), odd = -even;  // of the words w
  const int all_tiles = (wp.N + kRows - 1) / kRows;
  bool staged = false;
  for (int tile0 = blockIdx.x * tiles; tile0 < all_tiles; tile0 += gridDim.x * tiles) {
    const int row0 = (tile0 + warp / wp.slices) * kRows;
    // rows g, g + 8 of the two blocks; past N the last row is read and not stored
    const uint8_t* wr[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) wr[r] = wp.wq + min(row0 + g + 8 * r, wp.N - 1) * wp.ldw + 16 * t;
    // lane t fetches the scales and zeros of the quad's row g + 8 t
    const long long sr = static_cast<long long>(min(row0 + g + 8 * t, wp.N - 1)) * groups;
    const T* srow = static_cast<const T*>(wp.scales) + sr;
    const uint8_t* zrow = wp.zeros ? wp.zeros + sr : nullptr;
    auto load_w = [&](int r, int step) {
      if constexpr (FAST) step = min(step, steps - 1);  // past the end: nobody uses it
      const uint8_t* p = wr[r] + step * (kStep / 2);
      if constexpr (FAST) return __ldg(reinterpret_cast<const uint4*>(p));
      uint4 d = make_uint4(0, 0, 0, 0);
      if (step * kStep + 32 * t < wp.K) {
        if (wp.vec_w) {
          d = __ldg(reinterpret_cast<const uint4*>(p));
        } else {
          uint8_t* b = reinterpret_cast<uint8_t*>(&d);
#pragma unroll
          for (int i = 0; i < 16; ++i) b[i] = p[i];
        }
      }
      return d;
    };
    using Packed = std::conditional_t<GPS == 4, uint64_t, uint32_t>;  // a step's scales of a row
    auto load_s = [&](int step) {
      if constexpr (FAST) step = min(step, steps - 1);
      const T* p = srow + step * GPS;
      Packed d = 0;
      if constexpr (FAST) {
        if constexpr (GPS == 1) d = *reinterpret_cast<const uint16_t*>(p);
        else d = *reinterpret_cast<const Packed*>(p);
      } else {
#pragma unroll
        for (int q = 0; q < GPS; ++q)
          if (step * GPS + q < groups)
            d |= static_cast<Packed>(reinterpret_cast<const uint16_t*>(p)[q]) << (16 * q);
      }
      return d;
    };
    auto load_z = [&](int step) {
      uint32_t d = 0x08080808u;
      if (zrow) {
        if constexpr (FAST) step = min(step, steps - 1);
        const uint8_t* p = zrow + step * GPS;
        if constexpr (FAST) {
          d = GPS == 1 ? *p : GPS == 2 ? *reinterpret_cast<const uint16_t*>(p) : *reinterpret_cast<const uint32_t*>(p);
        } else {
          d = 0;
#pragma unroll
          for (int q = 0; q < GPS; ++q)
            if (step * GPS + q < groups) d |= static_cast<uint32_t>(p[q]) << (8 * q);
        }
      }
      return d;
    };
    uint4 ring[kAhead][4];
    Packed ring_s[kAhead];
    uint32_t ring_z[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) ring[i][r] = load_w(r, first + i);
      ring_s[i] = load_s(first + i);
      ring_z[i] = load_z(first + i);
    }
    float acc[2][NT][4];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[b][nt][0] = acc[b][nt][1] = acc[b][nt][2] = acc[b][nt][3] = 0.0f;

    int li = 0;  // step of the slice
    for (int l0 = 0; l0 < wp.per; l0 += wp.chunk) {
      if (!staged) {
        __syncthreads();  // the last chunk has been read
        stage(l0);
        __syncthreads();
        staged = once;
      }
      for (const int stop = min(own, l0 + wp.chunk); li < stop; li += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int st = first + li + i;
          uint4 wv[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            wv[r] = ring[i][r];
            ring[i][r] = load_w(r, st + kAhead);
          }
          const Packed sv = ring_s[i];
          const uint32_t zv = ring_z[i];
          ring_s[i] = load_s(st + kAhead);
          ring_z[i] = load_z(st + kAhead);
          if (li + i >= own) continue;
          float sc[4][GPS];
          Zero<T> zr[4] = {Zero<T>(8u), Zero<T>(8u), Zero<T>(8u), Zero<T>(8u)};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const Packed four = __shfl_sync(0xFFFFFFFFu, sv, (lane & 28) + r);
#pragma unroll
            for (int q = 0; q < GPS; ++q) {
              const uint16_t bits = static_cast<uint16_t>(four >> (16 * q));
              sc[r][q] = h2f<T>(*reinterpret_cast<const T*>(&bits));
            }
            // a lane's 32 weights lie in one group
            if (wp.zeros) zr[r] = Zero<T>(__shfl_sync(0xFFFFFFFFu, zv, (lane & 28) + r) >> (8 * (t * GPS / 4)) & 0xFFu);
          }
          float c[GPS][2][NT][4];
          const uint8_t* xst = xs + (li + i - l0) * step_bytes;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a[4][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint32_t word = w == 0 ? wv[r].x : w == 1 ? wv[r].y : w == 2 ? wv[r].z : wv[r].w;
              weights8<T>(word, zr[r], bits, a[r]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint4 x = make_uint4(0, 0, 0, 0);
              if (8 * nt + g < toks) x = *reinterpret_cast<const uint4*>(xst + 8 * nt * kTokBytes + 64 * w + (w & 1 ? odd : even));
#pragma unroll
              for (int q = 0; q < GPS; ++q) {
                // with several groups in the step, x of the other groups' lanes is
                // left out: a code times 0 is 0
                const bool in = GPS == 1 || t * GPS / 4 == q;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                  const uint32_t a0[4] = {a[2 * b][0], a[2 * b + 1][0], a[2 * b][1], a[2 * b + 1][1]};
                  const uint32_t a1[4] = {a[2 * b][2], a[2 * b + 1][2], a[2 * b][3], a[2 * b + 1][3]};
                  if (w == 0)
                    mma_16816<T, true>(c[q][b][nt], a0, in ? x.x : 0u, in ? x.y : 0u);
                  else
                    mma_16816<T, false>(c[q][b][nt], a0, in ? x.x : 0u, in ? x.y : 0u);
                  mma_16816<T, false>(c[q][b][nt], a1, in ? x.z : 0u, in ? x.w : 0u);
                }
              }
            }
          }
#pragma unroll
          for (int q = 0; q < GPS; ++q)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  acc[b][nt][e] = fmaf(sc[2 * b + (e >> 1)][q], c[q][b][nt][e], acc[b][nt][e]);
        }
      }
    }
    // ---- sums [warp][token][row], joined over the slices in their order; eight
    // rows of a token are a unit of the output
    constexpr int kSums = kTok * kRows;
    float* mine = red + warp * kSums;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mine[(8 * nt + 2 * t + (e & 1)) * kRows + 16 * b + g + (e >> 1) * 8] = acc[b][nt][e];
    auto put = [&](const float* from, int unit, int row) {  // unit of a tile that begins at row `row`
      const int m = unit / (kRows / 8), n = row + unit % (kRows / 8) * 8;
      if (m >= toks || n >= wp.N) return;
      float v[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) *reinterpret_cast<float4*>(v + 4 * j) = *reinterpret_cast<const float4*>(from + unit * 8 + 4 * j);
      for (int w = 1; w < wp.slices; ++w)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 y = *reinterpret_cast<const float4*>(from + w * kSums + unit * 8 + 4 * j);
          v[4 * j] += y.x;
          v[4 * j + 1] += y.y;
          v[4 * j + 2] += y.z;
          v[4 * j + 3] += y.w;
        }
      T* to = static_cast<T*>(wp.out) + (m0 + m) * wp.ldo + n;
      if (wp.bias)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += n + j < wp.N ? wp.bias[n + j] : 0.0f;
      if (wp.vec_o && n + 8 <= wp.N) {
        *reinterpret_cast<uint4*>(to) =
            make_uint4(cvt2_rn<T>(make_float2(v[0], v[1])), cvt2_rn<T>(make_float2(v[2], v[3])),
                       cvt2_rn<T>(make_float2(v[4], v[5])), cvt2_rn<T>(make_float2(v[6], v[7])));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (n + j < wp.N) to[j] = f2h<T>(v[j]);
      }
    };
    if (wp.slices == 1) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kSums / 8 / 32; ++i) put(mine, lane + 32 * i, row0);
      __syncwarp();
    } else {
      __syncthreads();
      for (int i = threadIdx.x; i < tiles * (kSums / 8); i += kWarps * 32) {
        const int tile = i / (kSums / 8);
        put(red + tile * wp.slices * kSums, i % (kSums / 8), (tile0 + tile) * kRows);
      }
      __syncthreads();
    }
  }
}

template <typename T, int NT, int GPS, bool FAST>
cudaError_t launch(W4Params wp, cudaStream_t s) {
  constexpr int kRed = kWarps * 8 * NT * kRows * 4;
  const int toks = std::min(8 * NT, wp.M), step_bytes = toks * 2 * kStep;
  const int steps = (wp.K + kStep - 1) / kStep, tiles = (wp.N + kRows - 1) / kRows;
  const int y = (wp.M + 8 * NT - 1) / (8 * NT);
  if (y > 65535) return cudaErrorInvalidValue;
  // split K until there are about 16 warps an SM, while each has a step
  wp.slices = 1;
  while (wp.slices < kWarps && static_cast<long long>(tiles) * y * wp.slices < 16ll * device_sm_count() &&
         2 * wp.slices <= steps)
    wp.slices *= 2;
  wp.per = (steps + wp.slices - 1) / wp.slices;
  wp.chunk = std::max(kAhead, (kXBytes - kRed) / (step_bytes * wp.slices) / kAhead * kAhead);
  wp.chunk = std::min(wp.chunk, wp.per);
  const int smem = wp.slices * wp.chunk * step_bytes + kRed;
  auto k = w4_kernel<T, NT, GPS, FAST>;
  static int set[64] = {0};  // per instantiation and device
  int dev = 0;
  cudaGetDevice(&dev);
  if (set[dev & 63] < smem) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    set[dev & 63] = smem;
  }
  const int per = kWarps / wp.slices;
  const int grid = std::min((tiles + per - 1) / per, std::max(1, (GPS * NT <= 2 ? 2 : 1) * device_sm_count() / y));
  return launch_pdl(k, dim3(grid, y), dim3(kWarps * 32), smem, s, wp);
}

template <typename T, int NT, int GPS>
cudaError_t launch_form(const W4Params& wp, cudaStream_t s) {
  const bool fast = wp.vec_x && wp.vec_w && wp.K % kStep == 0 && reinterpret_cast<uintptr_t>(wp.scales) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(wp.zeros) % 4 == 0;
  return fast ? launch<T, NT, GPS, true>(wp, s) : launch<T, NT, GPS, false>(wp, s);
}

template <typename T, int NT>
cudaError_t launch_group(const W4Params& wp, cudaStream_t s) {
  return wp.group == 128  ? launch_form<T, NT, 1>(wp, s)
         : wp.group == 64 ? launch_form<T, NT, 2>(wp, s)
                          : launch_form<T, NT, 4>(wp, s);
}

template <typename T>
cudaError_t launch_any(const W4Params& wp, cudaStream_t s) {
  return wp.M <= 8 ? launch_group<T, 1>(wp, s) : launch_group<T, 2>(wp, s);
}

}  // namespace

int w4_linear(const void* x, long long ldx, int M, int K, const uint8_t* wq, long long ldw, int N,
              int group, const void* scales, const uint8_t* zeros, const float* bias, void* out,
              long long ldo, bool bf16, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  W4Params wp{x, ldx, M, N, K, group, wq, ldw, scales, zeros, bias, out, ldo, 0, 0, 1, 1, 1, 0};
  wp.vec_x = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0;
  wp.vec_w = reinterpret_cast<uintptr_t>(wq) % 16 == 0 && ldw % 16 == 0;
  wp.vec_o = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ldo % 8 == 0;
  const cudaError_t e = bf16 ? launch_any<__nv_bfloat16>(wp, s) : launch_any<__half>(wp, s);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace qa
