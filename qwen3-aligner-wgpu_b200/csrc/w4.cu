// y = x W^T (+ bias) with W in 4 bits:
//   W[n][k] = scale[n][k / g] (code[n][k] - zero[n][k / g]),   zero = 8 where none is given.
// wq [N][K / 2] bytes, the even k of a pair in the low nibble.
//
// Built for few rows of x, where the weights' bytes are the bound (K / 2 a row
// of W, each read once).  A warp takes 16 RB rows of W (RB mma.sync M blocks) and
// walks K in steps of 128: a thread's 16 bytes of a W row are 32 weights, a
// quad's four threads cover the step, and a load of eight rows keeps whole
// 64-byte pieces in use; 4 KB of steps, of the next rows too, are on their way
// in registers.  The codes become 16-bit integers by bit work (in the mantissa of
// a power of two) less the zero, exactly; x is a 16-bit operand as it is; a
// group's sum is exact products in f32 and is scaled in f32, so nothing is
// rounded before the output.
//
// A word (8 weights) of all lanes lies in one group: of a step's 128 k a lane has
// 16 bytes in a row with groups of 128, 8 bytes in each of two groups of 64, 4 in
// each of four groups of 32.
//
// The order of k inside a step is free as long as both operands agree.  A word's
// nibbles leave the bit work as the pairs (0,4) (1,5) (2,6) (3,7); x is put in
// that order in shared memory, as the 16 bytes that a thread needs for a word.
// x stays there for all rows that the CTA takes, if it fits; a longer K goes
// through in chunks.
//
// With few rows of W a cluster of 2, 4 or 8 CTAs shares rows and splits K (so that
// a CTA needs its part of x only), and the sums are joined through distributed
// shared memory in the CTAs' order.  No atomics, the same bits each time.
//
// Bound by the latency of a warp's step (copies, bit work, products and scales in
// one chain, 16 warps an SM; 32 to 42 % of the issue slots are used, and 19 to 29 % of
// DRAM's time).  Measured on a B200: 4096 x 1024, one row, 8.5 us a call (10.2 without
// the split of K); 8191 x 8192, 5 rows, groups of 64 with zeros, 20.2 us (63 without
// the split); 151936 x 1024, 16 rows, 30 us, 2.8 TB/s.  W through a ring in shared memory
// came out the same or slower (22 and 30 us), 24 warps with fewer registers too (29
// and 35).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gemm_tc.cuh"
#include "kernels.cuh"
#include "sm100.cuh"

namespace qa {

namespace {

constexpr int kStep = 128;   // k of a step
constexpr int kWarps = 8;
constexpr int kXBytes = 96 * 1024;  // most of x in shared memory: two CTAs an SM

// For 8 NT tokens: M blocks a warp takes (more share each operand of x, as far as
// the registers reach) and steps of W in registers, one in use and the others on
// their way: 4 or 3 KB a warp.
template <int NT>
struct Form {
  static constexpr int kRb = NT == 1 ? 2 : 1, kRows = 16 * kRb, kAhead = 3, kCtas = 2;
};

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
  int slices;        // CTAs of a cluster, which share rows of W: 1, 2, 4 or 8
  int per;           // steps of a slice
  int chunk;         // steps of the slice that have x in shared memory at a time
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
// 16-bit values, by bit work in the mantissa of a power of two.  f16 has 1024 + code
// in its low four bits and 64 + 15 - code four bits higher, so one shift serves two
// pairs; bf16 has 128 + 15 - code.  For every byte 1024 + zero, 64 + 15 - zero and
// 128 + 15 - zero are exact (base + zero is not: no odd numbers above 256 in bf16,
// and no room for it in the mantissa above 64), and so are the differences
//   code - zero = (1024 + code) - (1024 + zero) = (base + 15 - zero) - (base + 15 - code).
template <typename T>
struct Zero {  // f16: 1024 + zero and 79 - zero; bf16: 143 - zero; twice
  uint32_t lo, hi;
  __device__ __forceinline__ Zero() {
    if constexpr (H16Traits<T>::kBf16) {
      lo = hi = 0x43074307u;  // 135
    } else {
      lo = 0x64086408u;  // 1032
      hi = 0x54705470u;  // 71
    }
  }
  // the zero is byte `at` of w
  __device__ __forceinline__ Zero(uint32_t w, int at) {
    if constexpr (H16Traits<T>::kBf16) {
      // 2^23 + zero, byte by byte; the difference is exact
      const float f = 8388608.0f + 143.0f - __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7640u | at));
      lo = hi = cvt2_rn<T>(make_float2(f, f));
    } else {
      lo = __byte_perm(w, 0x00000064u, 0x4040u | at * 0x101u);
      const __half2 h = __hsub2(__half2half2(__ushort_as_half(0x644F)), *reinterpret_cast<const __half2*>(&lo));  // 1103 -
      hi = *reinterpret_cast<const uint32_t*>(&h);
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
__device__ __forceinline__ uint32_t andn_or(uint32_t a, uint32_t mask, uint32_t base) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xAE;" : "=r"(d) : "r"(a), "r"(mask), "r"(base));  // (~a & mask) | base
  return d;
}
template <typename T>
__device__ __forceinline__ void weights8(uint32_t w, const Zero<T>& z, const Bits<T>& k, uint32_t (&out)[4]) {
  if constexpr (H16Traits<T>::kBf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = andn_or(w >> (4 * i), k.mask_lo, k.base_lo);
      const __nv_bfloat162 d =
          __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&z.lo), *reinterpret_cast<const __nv_bfloat162*>(&v));
      out[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = i < 2 ? w : w >> 8;
      const uint32_t v = i & 1 ? andn_or(u, k.mask_hi, k.base_hi) : and_or(u, k.mask_lo, k.base_lo);
      const __half2 c = *reinterpret_cast<const __half2*>(&v);
      const __half2 d = i & 1 ? __hsub2(*reinterpret_cast<const __half2*>(&z.hi), c)
                              : __hsub2(c, *reinterpret_cast<const __half2*>(&z.lo));
      out[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

// GPS: groups of a step, 1, 2 or 4 (group 128, 64, 32).  FAST: rows of x and W can
// be read 16 bytes at a time, a step's scales and zeros at once, and K is whole
// steps.

// First k, in its step, of word w of lane t.
template <int GPS>
__device__ __forceinline__ int word_k(int w, int t) {
  return GPS == 1 ? 32 * t + 8 * w : GPS == 2 ? 64 * (w >> 1) + 16 * t + 8 * (w & 1) : 32 * w + 8 * t;
}

template <typename T, int NT, int GPS, bool ZEROS, bool FAST>
__global__ void __launch_bounds__(kWarps * 32, Form<NT>::kCtas) w4_kernel(const __grid_constant__ W4Params wp) {
  constexpr int kTok = 8 * NT, kRb = Form<NT>::kRb, kRows = Form<NT>::kRows, kAhead = Form<NT>::kAhead;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * kTok, toks = min(kTok, wp.M - m0);
  const int steps = (wp.K + kStep - 1) / kStep, groups = wp.K / wp.group;
  const int slice = wp.slices > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int cta = blockIdx.x / wp.slices, ctas = gridDim.x / wp.slices;
  // x: [step][token][16 units of 16 bytes: word w of lane t at 4 w + t, odd
  // tokens with w ^ 1], so that an access of eight lanes (two tokens, four units)
  // meets 32 different banks; then the warps' sums
  constexpr int kTokBytes = 2 * kStep;
  const int step_bytes = toks * kTokBytes;
  float* red = reinterpret_cast<float*>(smem + wp.chunk * step_bytes);
  const Bits<T> bits;
  pdl_wait();
  pdl_trigger();

  // ---- W, its scales and zeros: `flat` counts this warp's steps over all its tiles
  const int first = slice * wp.per, own = min(wp.per, steps - first);  // own may be < 1
  const int row_step = ctas * kWarps * kRows, all_rows = wp.N;
  const int row_first = (cta * kWarps + warp) * kRows;
  using Packed = std::conditional_t<GPS == 4, uint64_t, uint32_t>;  // a step's scales of a row
  struct Ahead {
    uint4 w[2 * kRb];
    Packed s;
    uint32_t z;
  };
  const uint8_t* wr[2 * kRb];  // rows g, g + 8, .. of the tile being fetched; past N the last row
  long long sr = 0;            // where lane t's row (one of the quad's) has its scales
  auto at_tile = [&](int row0) {
#pragma unroll
    for (int r = 0; r < 2 * kRb; ++r)
      wr[r] = wp.wq + static_cast<long long>(min(row0 + g + 8 * r, all_rows - 1)) * wp.ldw + word_k<GPS>(0, t) / 2;
    sr = static_cast<long long>(min(row0 + g + 8 * (t % (2 * kRb)), all_rows - 1)) * groups;
  };
  int f_row = row_first, f_step = first;  // to be fetched next
  at_tile(f_row);
  auto fetch = [&](Ahead& a) {
    const int st = f_step;
    if constexpr (FAST) {
#pragma unroll
      for (int r = 0; r < 2 * kRb; ++r) {
        const uint8_t* p = wr[r] + st * (kStep / 2);
        if constexpr (GPS == 1) {
          a.w[r] = __ldg(reinterpret_cast<const uint4*>(p));
        } else if constexpr (GPS == 2) {
          const uint2 lo = __ldg(reinterpret_cast<const uint2*>(p)), hi = __ldg(reinterpret_cast<const uint2*>(p + 32));
          a.w[r] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          a.w[r] = make_uint4(__ldg(reinterpret_cast<const uint32_t*>(p)), __ldg(reinterpret_cast<const uint32_t*>(p + 16)),
                              __ldg(reinterpret_cast<const uint32_t*>(p + 32)), __ldg(reinterpret_cast<const uint32_t*>(p + 48)));
        }
      }
      const T* sp = static_cast<const T*>(wp.scales) + sr + st * GPS;
      if constexpr (GPS == 1) a.s = *reinterpret_cast<const uint16_t*>(sp);
      else a.s = *reinterpret_cast<const Packed*>(sp);
      if constexpr (ZEROS) {
        const uint8_t* zp = wp.zeros + sr + st * GPS;
        a.z = GPS == 1 ? *zp : GPS == 2 ? *reinterpret_cast<const uint16_t*>(zp) : *reinterpret_cast<const uint32_t*>(zp);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 2 * kRb; ++r) {
        uint8_t* b = reinterpret_cast<uint8_t*>(&a.w[r]);
        const uint8_t* p = wr[r] + st * (kStep / 2) - word_k<GPS>(0, t) / 2;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int k = word_k<GPS>(w, t);
#pragma unroll
          for (int i = 0; i < 4; ++i) b[4 * w + i] = st * kStep + k < wp.K ? p[k / 2 + i] : 0;
        }
      }
      a.s = 0;
      a.z = 0;
#pragma unroll
      for (int q = 0; q < GPS; ++q)
        if (st * GPS + q < groups) {
          a.s |= static_cast<Packed>(static_cast<const uint16_t*>(wp.scales)[sr + st * GPS + q]) << (16 * q);
          if (ZEROS) a.z |= static_cast<uint32_t>(wp.zeros[sr + st * GPS + q]) << (8 * q);
        }
    }
    if (++f_step == first + own) {
      f_step = first;
      f_row += row_step;  // past N: the last row again, which nobody uses
      at_tile(min(f_row, all_rows - 1));
    }
  };
  Ahead ring[kAhead];
  if (own > 0)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(ring[i]);

  // ---- x: steps [l0, l0 + chunk) of the slice.  A thread has one unit of one
  // token, and with few tokens every `apart`-th step
  const int apart = max(1, 2 * kWarps / toks), x_m = threadIdx.x / 16 % toks, x_from = threadIdx.x / 16 / toks;
  auto stage = [&](int l0) {
    const int c = threadIdx.x % 16;
    auto each = [&](auto f) {  // f(place, token, k) for the thread's units
      if (x_from >= apart) return;
      uint8_t* to = smem + x_m * kTokBytes + 16 * (c ^ 4 * (x_m & 1));
      const int n = min(wp.chunk, wp.per - l0);
#pragma unroll 2
      for (int i = x_from; i < n; i += apart)
        f(to + i * step_bytes, x_m, (first + l0 + i) * kStep + word_k<GPS>(c >> 2, c & 3));
    };
    if (FAST || wp.vec_x) {
      each([&](uint8_t* to, int m, int k) {  // zeros past K
        const T* src = static_cast<const T*>(wp.x) + (m0 + m) * wp.ldx;
        cp_async16(smem_u32(to), k < wp.K ? src + k : src, k < wp.K ? 16 : 0);
      });
      cp_async_commit();
      cp_async_wait_all();
    } else {
      each([&](uint8_t* to, int m, int k) {
        const T* src = static_cast<const T*>(wp.x) + (m0 + m) * wp.ldx + k;
        T* e = reinterpret_cast<T*>(to);
        for (int j = 0; j < 8; ++j) e[j] = k < wp.K ? src[j] : f2h<T>(0.0f);
      });
    }
    // (0 1)(2 3)(4 5)(6 7) -> (0 4)(1 5)(2 6)(3 7)
    each([&](uint8_t* to, int, int) {
      const uint4 d = *reinterpret_cast<const uint4*>(to);
      *reinterpret_cast<uint4*>(to) = make_uint4(__byte_perm(d.x, d.z, 0x5410), __byte_perm(d.x, d.z, 0x7632),
                                                 __byte_perm(d.y, d.w, 0x5410), __byte_perm(d.y, d.w, 0x7632));
    });
  };

  const bool once = wp.chunk >= wp.per;  // x stays for all rows
  // where this lane's token has its even and odd words; columns past the tokens
  // take the last one's x, and nobody reads their sums
  const uint8_t *x_even[NT], *x_odd[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int m = min(8 * nt + g, toks - 1);
    x_even[nt] = smem + m * kTokBytes + 16 * t + 64 * (m & 1);
    x_odd[nt] = smem + m * kTokBytes + 16 * t - 64 * (m & 1);
  }
  bool staged = false;
  int slot = 0;  // of the ring
  for (int row_cta = cta * kWarps * kRows; row_cta < all_rows; row_cta += row_step) {
    float acc[kRb][NT][4];
#pragma unroll
    for (int b = 0; b < kRb; ++b)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[b][nt][0] = acc[b][nt][1] = acc[b][nt][2] = acc[b][nt][3] = 0.0f;

    // one step, with what `a` brought; then a's place is filled again
    auto take = [&](Ahead& a, int at) {
      float c[kRb][NT][4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int q = w * GPS / 4;  // the word's group
        const bool opens = w % (4 / GPS) == 0, closes = (w + 1) % (4 / GPS) == 0;
        uint32_t k[2 * kRb][4];
#pragma unroll
        for (int r = 0; r < 2 * kRb; ++r) {
          Zero<T> zero;
          if constexpr (ZEROS) zero = Zero<T>(__shfl_sync(0xFFFFFFFFu, a.z, (lane & 28) + r), q);
          const uint32_t word = w == 0 ? a.w[r].x : w == 1 ? a.w[r].y : w == 2 ? a.w[r].z : a.w[r].w;
          weights8<T>(word, zero, bits, k[r]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 x = *reinterpret_cast<const uint4*>((w & 1 ? x_odd[nt] : x_even[nt]) + at + 64 * w);
#pragma unroll
          for (int b = 0; b < kRb; ++b) {
            const uint32_t a0[4] = {k[2 * b][0], k[2 * b + 1][0], k[2 * b][1], k[2 * b + 1][1]};
            const uint32_t a1[4] = {k[2 * b][2], k[2 * b + 1][2], k[2 * b][3], k[2 * b + 1][3]};
            if (opens)
              mma_16816<T, true>(c[b][nt], a0, x.x, x.y);
            else
              mma_16816<T, false>(c[b][nt], a0, x.x, x.y);
            mma_16816<T, false>(c[b][nt], a1, x.z, x.w);
          }
        }
        if (!closes) continue;
#pragma unroll
        for (int r = 0; r < 2 * kRb; ++r) {
          const uint16_t h = static_cast<uint16_t>(__shfl_sync(0xFFFFFFFFu, a.s, (lane & 28) + r) >> (16 * q));
          const float sc = h2f<T>(*reinterpret_cast<const T*>(&h));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 2 * (r & 1); e < 2 * (r & 1) + 2; ++e) acc[r / 2][nt][e] = fmaf(sc, c[r / 2][nt][e], acc[r / 2][nt][e]);
        }
      }
      fetch(a);
    };

    int li = 0;  // step of the slice
    for (int l0 = 0; l0 < wp.per; l0 += wp.chunk) {
      if (!staged) {
        __syncthreads();  // the last chunk has been read
        stage(l0);
        __syncthreads();
        staged = once;
      }
      const int stop = min(own, l0 + wp.chunk);
      while (li < stop) {
        // the ring goes on over tiles, its place in the loop's unrolled body does not
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (slot == i && li < stop) {
            take(ring[i], (li - l0) * step_bytes);
            ++li;
            slot = (i + 1) % kAhead;
          }
      }
    }
    // ---- sums [warp][token][row]; eight rows of a token are a unit of the output
    constexpr int kSums = kTok * kRows, kUnits = kSums / 8;
    float* mine = red + warp * kSums;
#pragma unroll
    for (int b = 0; b < kRb; ++b)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mine[(8 * nt + 2 * t + (e & 1)) * kRows + 16 * b + g + (e >> 1) * 8] = acc[b][nt][e];
    auto put = [&](float (&v)[8], int m, int n) {
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
      for (int i = 0; i < kUnits; i += 32) {
        const int u = i + lane, m = u / (kRows / 8), n = row_cta + warp * kRows + u % (kRows / 8) * 8;
        if (m < toks && n < all_rows) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 2; ++j) *reinterpret_cast<float4*>(v + 4 * j) = *reinterpret_cast<const float4*>(mine + 8 * u + 4 * j);
          put(v, m, n);
        }
      }
      __syncwarp();
    } else {
      cluster_sync();  // the cluster's sums are there; each CTA joins its share of the units
      for (int i = slice * (kWarps * 32) + threadIdx.x; i < kWarps * kUnits; i += wp.slices * (kWarps * 32)) {
        const int u = i % kUnits, m = u / (kRows / 8), n = row_cta + i / kUnits * kRows + u % (kRows / 8) * 8;
        if (m >= toks || n >= all_rows) continue;
        const uint32_t at = smem_u32(red + 8 * i);
        float v[8] = {};
        for (int r = 0; r < wp.slices; ++r) {
          const uint32_t from = mapa_shared(at, r);
          const float4 y = ld_cluster_f32x4(from), z = ld_cluster_f32x4(from + 16);
          v[0] += y.x;
          v[1] += y.y;
          v[2] += y.z;
          v[3] += y.w;
          v[4] += z.x;
          v[5] += z.y;
          v[6] += z.z;
          v[7] += z.w;
        }
        put(v, m, n);
      }
      cluster_sync();  // read before they are written again, or the CTA ends
    }
  }
}

template <typename T, int NT, int GPS, bool ZEROS, bool FAST>
cudaError_t launch(W4Params wp, cudaStream_t s) {
  constexpr int kRows = Form<NT>::kRows, kRed = kWarps * 8 * NT * kRows * 4;
  constexpr int kCtas = Form<NT>::kCtas;
  const int toks = std::min(8 * NT, wp.M), step_bytes = toks * 2 * kStep;
  const int steps = (wp.K + kStep - 1) / kStep, tiles = (wp.N - 1) / kRows + 1;
  const int y = (wp.M - 1) / (8 * NT) + 1;
  if (y > 65535 || wp.N > 0x40000000) return cudaErrorInvalidValue;
  // split K until the GPU is full, while each CTA has a step
  const int groups = (tiles - 1) / kWarps + 1;
  wp.slices = 1;
  while (wp.slices < 8 && static_cast<long long>(groups) * y * wp.slices < kCtas * device_sm_count() &&
         2 * wp.slices <= steps)
    wp.slices *= 2;
  wp.per = (steps + wp.slices - 1) / wp.slices;
  wp.chunk = std::min(wp.per, std::max(1, (kXBytes - kRed) / step_bytes));
  const int smem = wp.chunk * step_bytes + kRed;
  auto k = w4_kernel<T, NT, GPS, ZEROS, FAST>;
  static std::atomic<bool> set[64];  // per instantiation and device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kXBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) set[dev] = true;
  }
  const int ctas = std::min(groups, std::max(1, kCtas * device_sm_count() / (y * wp.slices)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas * wp.slices, y);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = wp.slices;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = wp.slices > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k, wp);
}

template <typename T, int NT, int GPS>
cudaError_t launch_form(const W4Params& wp, cudaStream_t s) {
  const bool fast = wp.vec_x && wp.vec_w && wp.K % kStep == 0 && reinterpret_cast<uintptr_t>(wp.scales) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(wp.zeros) % 4 == 0;
  if (wp.zeros) return fast ? launch<T, NT, GPS, true, true>(wp, s) : launch<T, NT, GPS, true, false>(wp, s);
  return fast ? launch<T, NT, GPS, false, true>(wp, s) : launch<T, NT, GPS, false, false>(wp, s);
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
  // a grid's y holds 65535 blocks of rows
  constexpr int kMost = 65535 * 16;
  for (long long m = 0; m < M; m += kMost) {
    wp.x = static_cast<const uint8_t*>(x) + 2 * m * ldx;
    wp.out = static_cast<uint8_t*>(out) + 2 * m * ldo;
    wp.M = static_cast<int>(std::min<long long>(kMost, M - m));
    const cudaError_t e = bf16 ? launch_any<__nv_bfloat16>(wp, s) : launch_any<__half>(wp, s);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)cudaGetLastError();
}

}  // namespace qa
