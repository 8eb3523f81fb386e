// Dropout with the mask drawn from a counter (hyc_philox.cuh), with or without the add of a residual:
//     y = residual + (keep ? x / (1 - p) : 0)
// computed in fp32 and rounded once.  What is dropped is selected away, not multiplied by zero: an infinity or a NaN in a
// dropped place does not reach y.  The backward pass is the same kernel on the arriving gradient.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hyc_host.cuh"
#include "hyc_philox.cuh"

namespace hyc {

struct DropoutArgs {
  const void *x, *residual;
  void* y;
  long long rows, cols, x_stride, residual_stride;
  const long long* rng;
  DropRate rate;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// one thread: the four elements of one counter block
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutArgs a) {
  const Philox gen = Philox::load(a.rng);
  const long long n = a.rows * a.cols, blocks = (n + 3) >> 2;
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  for (long long b = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; b < blocks;
       b += static_cast<long long>(gridDim.x) * blockDim.x) {
    const uint4 w4 = gen.block(static_cast<unsigned long long>(b));
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long long i = 4 * b + e;
      if (i >= n) break;
      const long long row = i / a.cols, col = i - row * a.cols;
      const float base = RES ? to_float<T>(res[row * a.residual_stride + col]) : 0.f;
      const float v = to_float<T>(x[row * a.x_stride + col]);
      y[i] = from_float<T>(a.rate.keep(w[e]) ? fmaf(v, a.rate.scale, base) : base);
    }
  }
}

__global__ void rng_take_kernel(unsigned long long* state, long long* used) {
  used[0] = static_cast<long long>(state[0]);
  used[1] = static_cast<long long>(atomicAdd(state + 1, 1ull));
}

template <typename T>
static int launch_dropout(const DropoutArgs& a, cudaStream_t stream) {
  const long long blocks = (a.rows * a.cols + 1023) / 1024;
  const int grid = static_cast<int>(blocks < 1 << 30 ? blocks : 1 << 30);
  if (a.residual)
    dropout_kernel<T, true><<<grid, 256, 0, stream>>>(a);
  else
    dropout_kernel<T, false><<<grid, 256, 0, stream>>>(a);
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "dropout_kernel");
}

}  // namespace hyc

using namespace hyc;

extern "C" {

int hyc_rng_take(int64_t* state, int64_t* used, void* stream) {
  if (!state || !used) return HYC_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(state) & 7u) || (reinterpret_cast<uintptr_t>(used) & 7u)) return HYC_ERR_ALIGN;
  rng_take_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(reinterpret_cast<unsigned long long*>(state),
                                                                  reinterpret_cast<long long*>(used));
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "rng_take_kernel");
}

int hyc_dropout(const hyc_dropout_args* args, void* stream) {
  if (!args) return HYC_ERR_NULL;
  if (args->rows < 0 || args->cols < 0 || (args->cols && args->rows > (1LL << 50) / args->cols)) return HYC_ERR_SHAPE;
  if (args->dtype != HYC_F32 && args->dtype != HYC_BF16) return HYC_ERR_DTYPE;
  if (!(args->p >= 0.0 && args->p <= 1.0)) return HYC_ERR_VALUE;
  if (args->rows == 0 || args->cols == 0) return HYC_OK;
  if (!args->x || !args->y || !args->rng) return HYC_ERR_NULL;
  const uintptr_t es = args->dtype == HYC_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(args->x) % es || reinterpret_cast<uintptr_t>(args->y) % es ||
      reinterpret_cast<uintptr_t>(args->residual) % es || (reinterpret_cast<uintptr_t>(args->rng) & 7u))
    return HYC_ERR_ALIGN;
  if (args->x_stride < 0 || args->residual_stride < 0) return HYC_ERR_SHAPE;
  DropoutArgs a;
  a.x = args->x; a.residual = args->residual; a.y = args->y;
  a.rows = args->rows; a.cols = args->cols; a.x_stride = args->x_stride; a.residual_stride = args->residual_stride;
  a.rng = reinterpret_cast<const long long*>(args->rng);
  a.rate = DropRate::make(args->p);
  return args->dtype == HYC_BF16 ? launch_dropout<__nv_bfloat16>(a, static_cast<cudaStream_t>(stream))
                                 : launch_dropout<float>(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
