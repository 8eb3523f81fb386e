// Layer norm of a residual sum, forward and backward, with dropout on the branch that joins the residual:
//     z = residual + dropout(x),  y = (z - mean(z)) * rstd(z) * weight + bias
//     with u = (z - mean) * rstd and g = dy * weight:
//     dz = (g - mean(g) - u * mean(g * u)) * rstd [+ the gradient that reaches z from elsewhere]
//     dx = keep ? dz / (1 - p) : 0, dresidual = dz, dweight = sum over rows of dy * u, dbias = sum over rows of dy
// Statistics, sums and gradients are held in fp32; every output is rounded once.  The forward pass normalises the unrounded
// sum; the backward pass starts from z as it was stored.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hyc_host.cuh"
#include "hyc_philox.cuh"

namespace hyc {

struct LnFwdArgs {
  const void *x, *residual, *weight, *bias;
  void *y, *z;
  float *mean, *rstd;
  long long rows, x_stride, residual_stride;
  int cols;
  float eps;
  const long long* rng;     // NULL: no dropout
  DropRate rate;
};

struct LnBwdArgs {
  const void *dy, *z, *dz, *weight;
  const float *mean, *rstd;
  void *dresidual, *dx, *dweight, *dbias;
  float* partials;          // [parts, 2, cols]
  long long rows, dy_stride, z_stride, dz_stride;
  int cols, parts;
  const long long* rng;
  DropRate rate;
};

template <typename T>
__device__ __forceinline__ float ln_load(const void* p, long long i) { return static_cast<const T*>(p)[i]; }
template <typename T>
__device__ __forceinline__ void ln_store(void* p, long long i, float v) { static_cast<T*>(p)[i] = T(v); }

__device__ __forceinline__ bool ln_keep(const Philox& gen, const DropRate& rate, unsigned long long element) {
  const uint4 w = gen.block(element >> 2);
  const uint32_t lane = static_cast<uint32_t>(element & 3);
  return rate.keep(lane == 0 ? w.x : lane == 1 ? w.y : lane == 2 ? w.z : w.w);
}

template <typename T, typename P>
__global__ void __launch_bounds__(256) ln_fwd_kernel(const LnFwdArgs a) {
  __shared__ float slot[3][64];
  Philox gen = {};
  if (a.rng) gen = Philox::load(a.rng);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    auto sum = [&](int c) {
      float v = ln_load<T>(a.x, row * a.x_stride + c);
      if (a.rng) v = ln_keep(gen, a.rate, static_cast<unsigned long long>(row) * a.cols + c) ? v * a.rate.scale : 0.f;
      if (a.residual) v += ln_load<T>(a.residual, row * a.residual_stride + c);
      return v;
    };
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) s[0] += sum(c);
    block_reduce<1>(s, slot[0], OpSum());
    const float mean = s[0] / a.cols;
    float q[1] = {0.f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float d = sum(c) - mean;
      q[0] += d * d;
    }
    block_reduce<1>(q, slot[1], OpSum());
    const float rstd = rsqrtf(q[0] / a.cols + a.eps);
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float v = sum(c);
      float y = (v - mean) * rstd;
      if (a.weight) y *= ln_load<P>(a.weight, c);
      if (a.bias) y += ln_load<P>(a.bias, c);
      ln_store<T>(a.y, row * a.cols + c, y);
      if (a.z) ln_store<T>(a.z, row * a.cols + c, v);
    }
    if (threadIdx.x == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
    __syncthreads();
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(256) ln_bwd_kernel(const LnBwdArgs a) {
  __shared__ float slot[64];
  Philox gen = {};
  if (a.rng) gen = Philox::load(a.rng);
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float g = ln_load<T>(a.dy, row * a.dy_stride + c) * (a.weight ? ln_load<P>(a.weight, c) : 1.f);
      s[0] += g;
      s[1] += g * (ln_load<T>(a.z, row * a.z_stride + c) - mean) * rstd;
    }
    block_reduce<2>(s, slot, OpSum());
    const float c2 = s[0] / a.cols, c1 = s[1] / a.cols;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float g = ln_load<T>(a.dy, row * a.dy_stride + c) * (a.weight ? ln_load<P>(a.weight, c) : 1.f);
      const float u = (ln_load<T>(a.z, row * a.z_stride + c) - mean) * rstd;
      float d = (g - c2 - u * c1) * rstd;
      if (a.dz) d += ln_load<T>(a.dz, row * a.dz_stride + c);
      ln_store<T>(a.dresidual, row * a.cols + c, d);
      if (a.dx)
        ln_store<T>(a.dx, row * a.cols + c,
                    ln_keep(gen, a.rate, static_cast<unsigned long long>(row) * a.cols + c) ? d * a.rate.scale : 0.f);
    }
    __syncthreads();
  }
}

// partial column sums: block y takes every gridDim.y-th row
template <typename T>
__global__ void __launch_bounds__(128) ln_partial_kernel(const LnBwdArgs a) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= a.cols) return;
  float w = 0.f, b = 0.f;
  for (long long row = blockIdx.y; row < a.rows; row += a.parts) {
    const float dy = ln_load<T>(a.dy, row * a.dy_stride + c);
    w += dy * ((ln_load<T>(a.z, row * a.z_stride + c) - a.mean[row]) * a.rstd[row]);
    b += dy;
  }
  a.partials[static_cast<long long>(blockIdx.y) * 2 * a.cols + c] = w;
  a.partials[(static_cast<long long>(blockIdx.y) * 2 + 1) * a.cols + c] = b;
}

template <typename P>
__global__ void __launch_bounds__(128) ln_finish_kernel(const LnBwdArgs a) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= a.cols) return;
  float w = 0.f, b = 0.f;
  for (int part = 0; part < a.parts; ++part) {
    w += a.partials[static_cast<long long>(part) * 2 * a.cols + c];
    b += a.partials[(static_cast<long long>(part) * 2 + 1) * a.cols + c];
  }
  if (a.dweight) ln_store<P>(a.dweight, c, w);
  if (a.dbias) ln_store<P>(a.dbias, c, b);
}

constexpr int kLnMaxCols = 16384;

static int ln_parts(long long rows) {
  const long long parts = (rows + 31) / 32;
  return static_cast<int>(parts < 1 ? 1 : parts > 148 ? 148 : parts);
}

static int check_ln(int64_t rows, int32_t cols, int32_t dtype, int32_t param_dtype, double p) {
  if (rows < 0 || rows > (1LL << 40) || cols < 1) return HYC_ERR_SHAPE;
  if (cols > kLnMaxCols) return HYC_ERR_CAPACITY;
  if ((dtype != HYC_F32 && dtype != HYC_BF16) || (param_dtype != HYC_F32 && param_dtype != HYC_BF16)) return HYC_ERR_DTYPE;
  if (!(p >= 0.0 && p <= 1.0)) return HYC_ERR_VALUE;
  return HYC_OK;
}

static bool misaligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

template <typename T, typename P>
static int launch_ln_fwd(const LnFwdArgs& a, cudaStream_t stream) {
  const int grid = static_cast<int>(a.rows < 148 * 8 ? a.rows : 148 * 8);
  ln_fwd_kernel<T, P><<<grid, 256, 0, stream>>>(a);
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "ln_fwd_kernel");
}

template <typename T, typename P>
static int launch_ln_bwd(const LnBwdArgs& a, cudaStream_t stream) {
  const int grid = static_cast<int>(a.rows < 148 * 8 ? a.rows : 148 * 8);
  ln_bwd_kernel<T, P><<<grid, 256, 0, stream>>>(a);
  HYC_LAUNCHED();
  if (a.dweight || a.dbias) {
    const int blocks = (a.cols + 127) / 128;
    ln_partial_kernel<T><<<dim3(blocks, a.parts), 128, 0, stream>>>(a);
    HYC_LAUNCHED();
    ln_finish_kernel<P><<<blocks, 128, 0, stream>>>(a);
    HYC_LAUNCHED();
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "ln_bwd_kernel");
}

}  // namespace hyc

using namespace hyc;

extern "C" {

int hyc_layer_norm(const hyc_layer_norm_args* q, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!q) return HYC_ERR_NULL;
  const int rc = check_ln(q->rows, q->cols, q->dtype, q->param_dtype, q->p);
  if (rc) return rc;
  if (q->rows == 0) return HYC_OK;
  if (!q->x || !q->y || !q->mean || !q->rstd || (q->p > 0.0 && !q->rng)) return HYC_ERR_NULL;
  if (q->x_stride < 0 || q->residual_stride < 0) return HYC_ERR_SHAPE;
  const uintptr_t es = q->dtype == HYC_BF16 ? 2 : 4, ps = q->param_dtype == HYC_BF16 ? 2 : 4;
  if (misaligned(q->x, es) || misaligned(q->residual, es) || misaligned(q->y, es) || misaligned(q->z, es) ||
      misaligned(q->weight, ps) || misaligned(q->bias, ps) || misaligned(q->mean, 4) || misaligned(q->rstd, 4) ||
      misaligned(q->rng, 8))
    return HYC_ERR_ALIGN;
  LnFwdArgs a;
  a.x = q->x; a.residual = q->residual; a.weight = q->weight; a.bias = q->bias; a.y = q->y; a.z = q->z;
  a.mean = q->mean; a.rstd = q->rstd; a.rows = q->rows; a.x_stride = q->x_stride; a.residual_stride = q->residual_stride;
  a.cols = q->cols; a.eps = q->eps;
  a.rng = q->p > 0.0 ? reinterpret_cast<const long long*>(q->rng) : nullptr;
  a.rate = DropRate::make(q->p);
  if (q->dtype == HYC_BF16)
    return q->param_dtype == HYC_BF16 ? launch_ln_fwd<__nv_bfloat16, __nv_bfloat16>(a, stream)
                                      : launch_ln_fwd<__nv_bfloat16, float>(a, stream);
  return q->param_dtype == HYC_BF16 ? launch_ln_fwd<float, __nv_bfloat16>(a, stream) : launch_ln_fwd<float, float>(a, stream);
}

int64_t hyc_layer_norm_bwd_scratch_floats(int64_t rows, int32_t cols) {
  if (rows < 0 || cols < 1) return HYC_ERR_SHAPE;
  if (cols > kLnMaxCols) return HYC_ERR_CAPACITY;
  return 2LL * ln_parts(rows) * cols;
}

int hyc_layer_norm_bwd(const hyc_layer_norm_bwd_args* q, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!q) return HYC_ERR_NULL;
  const int rc = check_ln(q->rows, q->cols, q->dtype, q->param_dtype, q->p);
  if (rc) return rc;
  const uintptr_t es = q->dtype == HYC_BF16 ? 2 : 4, ps = q->param_dtype == HYC_BF16 ? 2 : 4;
  if (misaligned(q->dweight, ps) || misaligned(q->dbias, ps)) return HYC_ERR_ALIGN;
  if (q->rows == 0) {
    for (void* p : {q->dweight, q->dbias}) {
      if (!p) continue;
      const cudaError_t e = cudaMemsetAsync(p, 0, static_cast<size_t>(q->cols) * ps, stream);
      if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync(parameter gradient)");
    }
    return HYC_OK;
  }
  if (!q->dy || !q->z || !q->mean || !q->rstd || !q->dresidual || (q->p > 0.0 && (!q->rng || !q->dx))) return HYC_ERR_NULL;
  if ((q->dweight || q->dbias) && !q->partials) return HYC_ERR_NULL;
  if (q->dy_stride < 0 || q->z_stride < 0 || q->dz_stride < 0) return HYC_ERR_SHAPE;
  if (misaligned(q->dy, es) || misaligned(q->z, es) || misaligned(q->dz, es) || misaligned(q->dresidual, es) ||
      misaligned(q->dx, es) || misaligned(q->weight, ps) || misaligned(q->mean, 4) || misaligned(q->rstd, 4) ||
      misaligned(q->rng, 8) || misaligned(q->partials, 16))
    return HYC_ERR_ALIGN;
  LnBwdArgs a;
  a.dy = q->dy; a.z = q->z; a.dz = q->dz; a.weight = q->weight; a.mean = q->mean; a.rstd = q->rstd;
  a.dresidual = q->dresidual; a.dx = q->p > 0.0 ? q->dx : nullptr; a.dweight = q->dweight; a.dbias = q->dbias;
  a.partials = q->partials; a.rows = q->rows; a.dy_stride = q->dy_stride; a.z_stride = q->z_stride; a.dz_stride = q->dz_stride;
  a.cols = q->cols; a.parts = ln_parts(q->rows);
  a.rng = q->p > 0.0 ? reinterpret_cast<const long long*>(q->rng) : nullptr;
  a.rate = DropRate::make(q->p);
  if (q->dtype == HYC_BF16)
    return q->param_dtype == HYC_BF16 ? launch_ln_bwd<__nv_bfloat16, __nv_bfloat16>(a, stream)
                                      : launch_ln_bwd<__nv_bfloat16, float>(a, stream);
  return q->param_dtype == HYC_BF16 ? launch_ln_bwd<float, __nv_bfloat16>(a, stream) : launch_ln_bwd<float, float>(a, stream);
}

}  // extern "C"
