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
  int param_bf16;
  float eps;
  const long long* rng;     // NULL: no dropout
  DropRate rate;
};

struct LnBwdArgs {
  const void *dy, *z, *dz, *weight;
  const float *mean, *rstd;
  void *dresidual, *dx, *dweight, *dbias;
  float* partials;          // [parts, 2, cols], NULL: no parameter gradients
  long long rows, dy_stride, z_stride, dz_stride;
  int cols, parts, param_bf16;
  const long long* rng;
  DropRate rate;
};

// ---------------------------------------------------------------- how a row is held
// A row belongs to G threads (a warp, or a group of warps with a named barrier of its own) that keep it in registers: one read
// of the row, statistics in two exact passes over registers, one write.  VEC: thread t owns the 8-element pieces t, t + G, ...
// (16-byte accesses; every address of every row 16-byte aligned).  Otherwise it owns the elements t, t + G, ... (coalesced
// accesses of single elements, for odd widths and unaligned tensors).

template <typename T>
__device__ __forceinline__ float ln_load(const void* p, long long i) { return static_cast<const T*>(p)[i]; }
template <typename T>
__device__ __forceinline__ void ln_store(void* p, long long i, float v) { static_cast<T*>(p)[i] = T(v); }

template <int G, bool VEC>
__device__ __forceinline__ int ln_col(int t, int v, int j) { return VEC ? (v * G + t) * 8 + j : (v * 8 + j) * G + t; }

// the eight elements of slot v of thread t, `fill` beyond the row's end
template <typename T, int G, bool VEC>
__device__ __forceinline__ void ln_get(const void* row, int t, int v, int cols, float (&f)[8]) {
  if (VEC) {
    const int c = (v * G + t) * 8;
    if (c < cols) {
      load8_stream(static_cast<const T*>(row) + c, f);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = (v * 8 + j) * G + t;
      f[j] = c < cols ? static_cast<float>(static_cast<const T*>(row)[c]) : 0.f;
    }
  }
}

template <typename T, int G, bool VEC>
__device__ __forceinline__ void ln_put(void* row, int t, int v, int cols, const float (&f)[8]) {
  if (VEC) {
    const int c = (v * G + t) * 8;
    if (c < cols) store8<T>(static_cast<T*>(row) + c, 0, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = (v * 8 + j) * G + t;
      if (c < cols) static_cast<T*>(row)[c] = T(f[j]);
    }
  }
}

// weight or bias: read again for every row (L1 keeps them), as fp32
template <int G, bool VEC>
__device__ __forceinline__ void ln_param(const void* p, bool bf16, int t, int v, int cols, float fill, float (&f)[8]) {
  if (VEC) {
    const int c = (v * G + t) * 8;
    if (p && c < cols) {
      if (bf16) load8<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(p), c, f);
      else load8<float>(static_cast<const float*>(p), c, f);
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = fill;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = (v * 8 + j) * G + t;
      f[j] = fill;
      if (p && c < cols) f[j] = bf16 ? ln_load<__nv_bfloat16>(p, c) : static_cast<const float*>(p)[c];
    }
  }
}

// which of the eight elements of a slot are kept; `first` is the index of the row's first element in the tensor
template <int G, bool VEC>
__device__ __forceinline__ uint32_t ln_kept(const Philox& gen, const DropRate& rate, unsigned long long first, int t, int v) {
  uint32_t kept = 0;
  if (VEC) {                                   // rows of a multiple of eight elements: two whole counter blocks
    const unsigned long long block = (first + static_cast<unsigned>((v * G + t) * 8)) >> 2;
    const uint4 lo = gen.block(block), hi = gen.block(block + 1);
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) kept |= rate.keep(w[j]) ? 1u << j : 0u;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned long long element = first + static_cast<unsigned>((v * 8 + j) * G + t);
      const uint4 w = gen.block(element >> 2);
      const uint32_t lane = static_cast<uint32_t>(element & 3);
      kept |= rate.keep(lane == 0 ? w.x : lane == 1 ? w.y : lane == 2 ? w.z : w.w) ? 1u << j : 0u;
    }
  }
  return kept;
}

template <int G>
__device__ __forceinline__ void group_sync() {
  if (G == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / G), "n"(G) : "memory");
}

// Sums of N values over the G threads of a group, the same bits in every thread.  `slot` is the group's own, N * 32 floats,
// and is not used again before the group has met at another barrier.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if (G == 32) return;
  const int warp = (threadIdx.x % G) >> 5;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slot[i * 32 + warp] = v[i];
  }
  group_sync<G>();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float r = 0.f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) r += slot[i * 32 + w];
    v[i] = r;
  }
}

// ---------------------------------------------------------------- forward

// One row per group of G threads, CTAs of at least 256 threads.  Traffic is what the formula needs; the loads of a whole
// row are in flight before the first sum, and rows of other groups on the SM cover the two reductions.
template <typename T, int G, int VPT, bool DROP, bool VEC>
__global__ void __launch_bounds__(G < 256 ? 256 : G) ln_fwd_kernel(const LnFwdArgs a) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G;
  __shared__ float slots[kGroups][2][32];
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  const long long row = static_cast<long long>(blockIdx.x) * kGroups + group;
  if (row >= a.rows) return;
  const void* x = static_cast<const T*>(a.x) + row * a.x_stride;
  float z[VPT][8];
#pragma unroll
  for (int v = 0; v < VPT; ++v) ln_get<T, G, VEC>(x, t, v, a.cols, z[v]);
  if (a.residual) {
    const void* res = static_cast<const T*>(a.residual) + row * a.residual_stride;
    float r[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v) ln_get<T, G, VEC>(res, t, v, a.cols, r[v]);
    if (DROP) {
      const Philox gen = Philox::load(a.rng);
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const uint32_t kept = ln_kept<G, VEC>(gen, a.rate, static_cast<unsigned long long>(row) * a.cols, t, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[v][j] = kept >> j & 1 ? fmaf(z[v][j], a.rate.scale, r[v][j]) : r[v][j];
      }
    } else {
#pragma unroll
      for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) z[v][j] += r[v][j];
    }
  } else if (DROP) {
    const Philox gen = Philox::load(a.rng);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const uint32_t kept = ln_kept<G, VEC>(gen, a.rate, static_cast<unsigned long long>(row) * a.cols, t, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[v][j] = kept >> j & 1 ? z[v][j] * a.rate.scale : 0.f;
    }
  }
  float s[1] = {0.f};
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const float(&p)[8] = z[v];                       // zero beyond the row's end
    s[0] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
  }
  group_sum<G, 1>(s, slots[group][0]);
  const float mean = s[0] / a.cols;
  float q[1] = {0.f};
#pragma unroll
  for (int v = 0; v < VPT; ++v)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = z[v][j] - mean;
      if (ln_col<G, VEC>(t, v, j) < a.cols) q[0] = fmaf(d, d, q[0]);
    }
  group_sum<G, 1>(q, slots[group][1]);
  const float rstd = rsqrtf(q[0] / a.cols + a.eps);
  if (t == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  void* y = static_cast<T*>(a.y) + row * a.cols;
  if (a.z) {
    void* zp = static_cast<T*>(a.z) + row * a.cols;
#pragma unroll
    for (int v = 0; v < VPT; ++v) ln_put<T, G, VEC>(zp, t, v, a.cols, z[v]);
  }
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    float w[8], b[8];
    ln_param<G, VEC>(a.weight, a.param_bf16, t, v, a.cols, 1.f, w);
    ln_param<G, VEC>(a.bias, a.param_bf16, t, v, a.cols, 0.f, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = fmaf((z[v][j] - mean) * rstd, w[j], b[j]);
    ln_put<T, G, VEC>(y, t, v, a.cols, w);
  }
}

// ---------------------------------------------------------------- backward

// Where the parameter gradients of a thread's own columns add up over its rows: registers, or (rows so wide that they would
// not fit beside the row) shared memory, one conflict-free column of it per thread.
template <int VPT, bool SMEM, int THREADS>
struct LnAcc {
  float w[VPT][8], b[VPT][8];
  __device__ __forceinline__ void init(float*) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) w[v][j] = b[v][j] = 0.f;
  }
  __device__ __forceinline__ void add(int v, int j, float dw, float db) { w[v][j] += dw; b[v][j] += db; }
  __device__ __forceinline__ float2 get(int v, int j) const { return make_float2(w[v][j], b[v][j]); }
};
template <int VPT, int THREADS>
struct LnAcc<VPT, true, THREADS> {
  float2* own;
  __device__ __forceinline__ void init(float* smem) {
    own = reinterpret_cast<float2*>(smem) + threadIdx.x;
    for (int i = 0; i < VPT * 8; ++i) own[i * THREADS] = make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ void add(int v, int j, float dw, float db) {
    float2 s = own[(v * 8 + j) * THREADS];
    s.x += dw;
    s.y += db;
    own[(v * 8 + j) * THREADS] = s;
  }
  __device__ __forceinline__ float2 get(int v, int j) const { return own[(v * 8 + j) * THREADS]; }
};

// Persistent groups: group g of CTA b takes the rows b * kGroups + g, + gridDim * kGroups, ...  A row is read once; its
// gradient is written while the columns' sums stay with their thread, and leave once per CTA as a row of partial sums.
template <typename T, int G, int VPT, bool DROP, bool VEC, bool SMEM>
__global__ void __launch_bounds__(G < 256 ? 256 : G) ln_bwd_kernel(const LnBwdArgs a) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G;
  extern __shared__ float dynamic[];
  __shared__ float slots[kGroups][2][2][32];
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  LnAcc<VPT, SMEM, kThreads> acc;
  acc.init(dynamic);
  Philox gen = {};
  if (DROP) gen = Philox::load(a.rng);
  int turn = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * kGroups + group; row < a.rows;
       row += static_cast<long long>(gridDim.x) * kGroups, turn ^= 1) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[VPT][8], u[VPT][8];
    const void* dyp = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const void* zp = static_cast<const T*>(a.z) + row * a.z_stride;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      ln_get<T, G, VEC>(dyp, t, v, a.cols, g[v]);
      ln_get<T, G, VEC>(zp, t, v, a.cols, u[v]);
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float w[8];
      ln_param<G, VEC>(a.weight, a.param_bf16, t, v, a.cols, 1.f, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (ln_col<G, VEC>(t, v, j) >= a.cols) { u[v][j] = 0.f; continue; }
        u[v][j] = (u[v][j] - mean) * rstd;
        acc.add(v, j, g[v][j] * u[v][j], g[v][j]);
        g[v][j] *= w[j];
        s[0] += g[v][j];
        s[1] = fmaf(g[v][j], u[v][j], s[1]);
      }
    }
    group_sum<G, 2>(s, &slots[group][turn][0][0]);
    const float c2 = s[0] / a.cols, c1 = s[1] / a.cols;
    void* out = static_cast<T*>(a.dresidual) + row * a.cols;
    void* dx = static_cast<T*>(a.dx) + row * a.cols;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float d[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = (g[v][j] - c2 - u[v][j] * c1) * rstd;
      if (a.dz) {
        float e[8];
        ln_get<T, G, VEC>(static_cast<const T*>(a.dz) + row * a.dz_stride, t, v, a.cols, e);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] += e[j];
      }
      ln_put<T, G, VEC>(out, t, v, a.cols, d);
      if (DROP) {
        const uint32_t kept = ln_kept<G, VEC>(gen, a.rate, static_cast<unsigned long long>(row) * a.cols, t, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = kept >> j & 1 ? d[j] * a.rate.scale : 0.f;
        ln_put<T, G, VEC>(dx, t, v, a.cols, d);
      }
    }
  }
  if (!a.partials) return;
  float* part = a.partials + static_cast<long long>(blockIdx.x) * 2 * a.cols;
  if (kGroups == 1) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = ln_col<G, VEC>(t, v, j);
        const float2 p = acc.get(v, j);
        if (c < a.cols) { part[c] = p.x; part[a.cols + c] = p.y; }
      }
    return;
  }
  // the groups of a CTA, summed in their order through shared memory: [group][slot][thread]
  float2* all = reinterpret_cast<float2*>(dynamic);
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) all[(group * 8 + j) * G + t] = acc.get(v, j);
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * G; i += kThreads) {
      float2 sum = all[i];
      for (int k = 1; k < kGroups; ++k) {
        const float2 p = all[k * 8 * G + i];
        sum.x += p.x;
        sum.y += p.y;
      }
      const int c = ln_col<G, VEC>(i % G, v, i / G);
      if (c < a.cols) { part[c] = sum.x; part[a.cols + c] = sum.y; }
    }
  }
}

// The partial rows, summed in a fixed order: 32 columns per CTA, eight lanes of rows.
__global__ void __launch_bounds__(256) ln_finish_kernel(const LnBwdArgs a) {
  __shared__ float sums[8][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
  float s = 0.f;
  if (c < 2 * a.cols) {
#pragma unroll 8
    for (int part = lane; part < a.parts; part += 8) s += a.partials[static_cast<long long>(part) * 2 * a.cols + c];
  }
  sums[lane][threadIdx.x & 31] = s;
  __syncthreads();
  if (lane == 0 && c < 2 * a.cols) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sums[k][threadIdx.x & 31];
    void* out = c < a.cols ? a.dweight : a.dbias;
    const int at = c < a.cols ? c : c - a.cols;
    if (out) {
      if (a.param_bf16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(s);
      else static_cast<float*>(out)[at] = s;
    }
  }
}

constexpr int kLnMaxCols = 16384;

constexpr int kLnMaxParts = 148 * 3;

// most partial rows that a call of so many rows writes (the scratch a caller brings)
static int ln_max_parts(long long rows) { return static_cast<int>(rows < 1 ? 1 : rows < kLnMaxParts ? rows : kLnMaxParts); }

static int check_ln(int64_t rows, int32_t cols, int32_t dtype, int32_t param_dtype, double p) {
  if (rows < 0 || cols < 1) return HYC_ERR_SHAPE;
  if (cols > kLnMaxCols || rows > 0x7fffffffLL) return HYC_ERR_CAPACITY;
  if ((dtype != HYC_F32 && dtype != HYC_BF16) || (param_dtype != HYC_F32 && param_dtype != HYC_BF16)) return HYC_ERR_DTYPE;
  if (!(p >= 0.0 && p <= 1.0)) return HYC_ERR_VALUE;
  return HYC_OK;
}

static bool misaligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

static bool rows_aligned(const void* p, long long stride, uintptr_t es) { return !p || (aligned16(p) && stride * es % 16 == 0); }

template <typename T, int G, int VPT, bool VEC>
static void run_ln_fwd(const LnFwdArgs& a, cudaStream_t stream) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G;
  const unsigned grid = static_cast<unsigned>((a.rows + kGroups - 1) / kGroups);
  if (a.rng) ln_fwd_kernel<T, G, VPT, true, VEC><<<grid, kThreads, 0, stream>>>(a);
  else ln_fwd_kernel<T, G, VPT, false, VEC><<<grid, kThreads, 0, stream>>>(a);
}

// threads per row and pieces per thread by the row's width: the smallest group that holds it in at most 32 elements per thread
template <typename T, bool VEC>
static void pick_ln_fwd(const LnFwdArgs& a, cudaStream_t stream) {
  const int pieces = (a.cols + 7) / 8;
  if (pieces <= 32) run_ln_fwd<T, 32, 1, VEC>(a, stream);
  else if (pieces <= 64) run_ln_fwd<T, 32, 2, VEC>(a, stream);
  else if (pieces <= 96) run_ln_fwd<T, 32, 3, VEC>(a, stream);
  else if (pieces <= 128) run_ln_fwd<T, 32, 4, VEC>(a, stream);
  else if (pieces <= 256) run_ln_fwd<T, 128, 2, VEC>(a, stream);
  else if (pieces <= 512) run_ln_fwd<T, 128, 4, VEC>(a, stream);
  else if (pieces <= 1024) run_ln_fwd<T, 256, 4, VEC>(a, stream);
  else run_ln_fwd<T, 512, 4, VEC>(a, stream);
}

template <typename T>
static int launch_ln_fwd(const LnFwdArgs& a, cudaStream_t stream) {
  const uintptr_t es = sizeof(T);
  const bool vec = a.cols % 8 == 0 && rows_aligned(a.x, a.x_stride, es) && rows_aligned(a.residual, a.residual_stride, es) &&
                   aligned16(a.y) && aligned16(a.z) && aligned16(a.weight) && aligned16(a.bias);
  if (vec) pick_ln_fwd<T, true>(a, stream);
  else pick_ln_fwd<T, false>(a, stream);
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "ln_fwd_kernel");
}

template <typename T, int G, int VPT, bool DROP, bool VEC, bool SMEM>
static int run_ln_bwd(LnBwdArgs a, cudaStream_t stream) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G;
  auto kernel = ln_bwd_kernel<T, G, VPT, DROP, VEC, SMEM>;
  const uint32_t smem = SMEM ? kThreads * VPT * 8 * 8 : kGroups > 1 ? kThreads * 8 * 8 : 0;
  const int rc = set_smem(kernel, smem);
  if (rc) return rc;
  const long long batches = (a.rows + kGroups - 1) / kGroups;
  a.parts = resident_grid(kernel, kThreads, smem, static_cast<int>(batches < kLnMaxParts ? batches : kLnMaxParts));
  kernel<<<a.parts, kThreads, smem, stream>>>(a);
  HYC_LAUNCHED();
  if (a.partials) {
    ln_finish_kernel<<<(2 * a.cols + 31) / 32, 256, 0, stream>>>(a);
    HYC_LAUNCHED();
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "ln_bwd_kernel");
}

template <typename T, bool DROP, bool VEC>
static int pick_ln_bwd(const LnBwdArgs& a, cudaStream_t stream) {
  const int pieces = (a.cols + 7) / 8;
  if (pieces <= 32) return run_ln_bwd<T, 32, 1, DROP, VEC, false>(a, stream);
  if (pieces <= 64) return run_ln_bwd<T, 32, 2, DROP, VEC, false>(a, stream);
  if (pieces <= 96) return run_ln_bwd<T, 32, 3, DROP, VEC, false>(a, stream);
  if (pieces <= 128) return run_ln_bwd<T, 128, 1, DROP, VEC, false>(a, stream);
  if (pieces <= 256) return run_ln_bwd<T, 128, 2, DROP, VEC, false>(a, stream);
  if (pieces <= 512) return run_ln_bwd<T, 256, 2, DROP, VEC, false>(a, stream);
  if (pieces <= 1024) return run_ln_bwd<T, 512, 2, DROP, VEC, false>(a, stream);
  return run_ln_bwd<T, 512, 4, DROP, VEC, true>(a, stream);
}

template <typename T>
static int launch_ln_bwd(const LnBwdArgs& a, cudaStream_t stream) {
  const uintptr_t es = sizeof(T);
  const bool vec = a.cols % 8 == 0 && rows_aligned(a.dy, a.dy_stride, es) && rows_aligned(a.z, a.z_stride, es) &&
                   rows_aligned(a.dz, a.dz_stride, es) && aligned16(a.dresidual) && aligned16(a.dx) && aligned16(a.weight);
  if (vec) return a.rng ? pick_ln_bwd<T, true, true>(a, stream) : pick_ln_bwd<T, false, true>(a, stream);
  return a.rng ? pick_ln_bwd<T, true, false>(a, stream) : pick_ln_bwd<T, false, false>(a, stream);
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
  a.cols = q->cols; a.eps = q->eps; a.param_bf16 = q->param_dtype == HYC_BF16;
  a.rng = q->p > 0.0 ? reinterpret_cast<const long long*>(q->rng) : nullptr;
  a.rate = DropRate::make(q->p);
  return q->dtype == HYC_BF16 ? launch_ln_fwd<__nv_bfloat16>(a, stream) : launch_ln_fwd<float>(a, stream);
}

int64_t hyc_layer_norm_bwd_scratch_floats(int64_t rows, int32_t cols) {
  if (rows < 0 || cols < 1) return HYC_ERR_SHAPE;
  if (cols > kLnMaxCols || rows > 0x7fffffffLL) return HYC_ERR_CAPACITY;
  return 2LL * ln_max_parts(rows) * cols;
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
  a.partials = q->dweight || q->dbias ? q->partials : nullptr;
  a.rows = q->rows; a.dy_stride = q->dy_stride; a.z_stride = q->z_stride; a.dz_stride = q->dz_stride;
  a.cols = q->cols; a.parts = 0; a.param_bf16 = q->param_dtype == HYC_BF16;
  a.rng = q->p > 0.0 ? reinterpret_cast<const long long*>(q->rng) : nullptr;
  a.rate = DropRate::make(q->p);
  return q->dtype == HYC_BF16 ? launch_ln_bwd<__nv_bfloat16>(a, stream) : launch_ln_bwd<float>(a, stream);
}

}  // extern "C"
