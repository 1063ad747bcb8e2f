// y = x W^T (+ bias) with W in 4 bits:
//   W[n][k] = scale[n][k / g] (code[n][k] - zero[n][k / g]),   zero = 8 where none is given.
// wq [N][K / 2] bytes, the even k of a pair in the low nibble.
#include "kernels.cuh"
#include "sm100.cuh"

namespace qa {

namespace {

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
};

// One warp per output value.
template <typename T>
__global__ void __launch_bounds__(256) w4_simple(W4Params wp) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long n = static_cast<long long>(blockIdx.x) * 8 + threadIdx.x / 32;
  if (n >= wp.N) return;
  const int groups = wp.K / wp.group;
  for (int m = blockIdx.y; m < wp.M; m += gridDim.y) {
    const T* x = static_cast<const T*>(wp.x) + m * wp.ldx;
    float acc = 0.0f;
    for (int k = lane * 2; k < wp.K; k += 64) {
      const int g = k / wp.group;
      const float s = h2f<T>(static_cast<const T*>(wp.scales)[n * groups + g]);
      const float z = wp.zeros ? static_cast<float>(wp.zeros[n * groups + g]) : 8.0f;
      const uint8_t b = wp.wq[n * wp.ldw + k / 2];
      acc += s * ((static_cast<float>(b & 15) - z) * h2f<T>(x[k]) +
                  (static_cast<float>(b >> 4) - z) * h2f<T>(x[k + 1]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xFFFFFFFFu, acc, o);
    if (lane == 0)
      static_cast<T*>(wp.out)[m * wp.ldo + n] = f2h<T>(acc + (wp.bias ? wp.bias[n] : 0.0f));
  }
}

}  // namespace

int w4_linear(const void* x, long long ldx, int M, int K, const uint8_t* wq, long long ldw, int N,
              int group, const void* scales, const uint8_t* zeros, const float* bias, void* out,
              long long ldo, bool bf16, cudaStream_t s) {
  if (M <= 0 || N <= 0) return 0;
  const W4Params wp{x, ldx, M, N, K, group, wq, ldw, scales, zeros, bias, out, ldo};
  const dim3 grid((N + 7) / 8, M < 65535 ? M : 65535);
  const cudaError_t e = bf16 ? launch_pdl(w4_simple<__nv_bfloat16>, grid, dim3(256), 0, s, wp)
                             : launch_pdl(w4_simple<__half>, grid, dim3(256), 0, s, wp);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace qa
