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

// Any addresses and strides.  One thread: the four elements of one counter block.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_any_kernel(const DropoutArgs a) {
  const Philox gen = Philox::load(a.rng);
  const long long n = a.rows * a.cols, blocks = (n + 3) >> 2;
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  for (long long b = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; b < blocks;
       b += static_cast<long long>(gridDim.x) * blockDim.x) {
    const uint4 w4 = gen.block(static_cast<unsigned long long>(b));
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
    long long row = 4 * b / a.cols, col = 4 * b - row * a.cols;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (4 * b + e >= n) break;
      const float base = RES ? to_float<T>(res[row * a.residual_stride + col]) : 0.f;
      const float v = to_float<T>(x[row * a.x_stride + col]);
      y[4 * b + e] = T(a.rate.keep(w[e]) ? fmaf(v, a.rate.scale, base) : base);
      if (++col == a.cols) { col = 0; ++row; }
    }
  }
}

// One flat run of elements at 16-byte aligned addresses.  A thread takes kDropUnits pieces of eight elements (two counter
// blocks each) that lie a CTA's width apart, all loads before the first use.  What bounds it is DRAM as long as the ten
// rounds of the generator (about 11 instructions per element) stay under the issue slots that the traffic leaves: 22 per
// element for bf16 without a residual.
constexpr int kDropUnits = 2;

template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_flat_kernel(const DropoutArgs a) {
  const Philox gen = Philox::load(a.rng);
  const long long units = a.cols >> 3;
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  const long long first = static_cast<long long>(blockIdx.x) * (256 * kDropUnits) + threadIdx.x;
  float v[kDropUnits][8], r[kDropUnits][8];
#pragma unroll
  for (int u = 0; u < kDropUnits; ++u) {
    const long long unit = first + u * 256;
    if (unit < units) {
      load8_stream(x + unit * 8, v[u]);
      if (RES) load8_stream(res + unit * 8, r[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < kDropUnits; ++u) {
    const long long unit = first + u * 256;
    if (unit < units) {
      const uint4 lo = gen.block(2ull * unit), hi = gen.block(2ull * unit + 1);
      const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float base = RES ? r[u][e] : 0.f;
        v[u][e] = a.rate.keep(w[e]) ? fmaf(v[u][e], a.rate.scale, base) : base;
      }
      store8<T>(y + unit * 8, 0, v[u]);
    }
  }
  // the last elements, fewer than eight
  const long long e = units * 8 + threadIdx.x;
  if (blockIdx.x == 0 && e < a.cols) {
    const uint4 w = gen.block(static_cast<unsigned long long>(e >> 2));
    const int lane = static_cast<int>(e & 3);
    const float base = RES ? to_float<T>(res[e]) : 0.f;
    const bool keep = a.rate.keep(lane == 0 ? w.x : lane == 1 ? w.y : lane == 2 ? w.z : w.w);
    y[e] = T(keep ? fmaf(to_float<T>(x[e]), a.rate.scale, base) : base);
  }
}

__global__ void rng_take_kernel(unsigned long long* state, long long* used) {
  used[0] = static_cast<long long>(state[0]);
  used[1] = static_cast<long long>(atomicAdd(state + 1, 1ull));
}

template <typename T>
static int launch_dropout(const DropoutArgs& a, cudaStream_t stream) {
  const bool flat = a.rows == 1 && aligned16(a.x) && aligned16(a.y) && aligned16(a.residual);
  const long long per_block = flat ? 256 * 8 * kDropUnits : 1024, blocks = (a.rows * a.cols + per_block - 1) / per_block;
  if (flat && blocks <= 0x7fffffffLL) {
    if (a.residual)
      dropout_flat_kernel<T, true><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
    else
      dropout_flat_kernel<T, false><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
  } else {
    const int grid = static_cast<int>(blocks < 1 << 30 ? blocks : 1 << 30);
    if (a.residual)
      dropout_any_kernel<T, true><<<grid, 256, 0, stream>>>(a);
    else
      dropout_any_kernel<T, false><<<grid, 256, 0, stream>>>(a);
  }
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "dropout kernel");
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
