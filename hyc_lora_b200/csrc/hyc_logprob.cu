// Log probabilities of given tokens under rows of logits, with the entropy of each row and its best alternatives, and the
// gradient of all three.  With m the largest logit of a row and S = sum over the row of exp(x - m):
//     log p_i = (x_i - m) - log S,   H = log S - (sum of exp(x - m) (x - m)) / S
//     d x_i = h_i - G p_i - dH p_i (log p_i + H),   h_i: what arrives for token i (target, alternatives), G: the sum of all h
// m's own terms are counted apart from the other sum r, so that log S = log1p(r) keeps its digits where one token has nearly
// all the weight, and 1 - p of a listed token is taken as -expm1(log p).  All of it is fp32.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hyc_host.cuh"

namespace hyc {

struct LogprobArgs {
  const void* logits;
  long long rows, row_stride, batch_stride, seq;
  int vocab, top;
  const long long* targets;
  long long ignore_index;
  float *logprob, *entropy, *stats, *top_logprob;
  long long* top_index;
};

struct LogprobBwdArgs {
  const void* logits;
  long long rows, row_stride, batch_stride, seq;
  int vocab, top;
  const long long* targets;
  long long ignore_index;
  const float *stats, *entropy, *d_logprob, *d_entropy, *d_top;
  const long long* top_index;
  void* grad;
};

__device__ __forceinline__ float lp_load(const float* p, long long i) { return p[i]; }
__device__ __forceinline__ float lp_load(const __nv_bfloat16* p, long long i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ void lp_store(float* p, long long i, float v) { p[i] = v; }
__device__ __forceinline__ void lp_store(__nv_bfloat16* p, long long i, float v) { p[i] = __float2bfloat16_rn(v); }

// Order of the alternatives as one integer: larger value first (-0 counts as +0, a NaN stands above +inf), lower index first
// among equals.
__device__ __forceinline__ unsigned long long lp_key(float v, uint32_t index) {
  uint32_t b = __float_as_uint(v + 0.f);
  b = v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(b) << 32 | (0xffffffffu - index);
}

struct OpMaxNan {
  __device__ __forceinline__ float operator()(float a, float b) const { return a != a ? a : b != b ? b : fmaxf(a, b); }
};

template <typename T>
__global__ void __launch_bounds__(512) logprob_kernel(const LogprobArgs a) {
  __shared__ float slot[3][32 * 3];
  __shared__ unsigned long long best[16];
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.logits) + (row / a.seq) * a.batch_stride + (row % a.seq) * a.row_stride;
    const long long target = a.targets ? a.targets[row] : 0;
    if (a.targets && target == a.ignore_index && !a.entropy && !a.top) {
      if (threadIdx.x == 0) {
        a.logprob[row] = 0.f;
        a.stats[2 * row] = -INFINITY;
        a.stats[2 * row + 1] = 0.f;
      }
      continue;
    }
    float m[1] = {-INFINITY};
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) m[0] = OpMaxNan()(m[0], lp_load(x, i));
    block_reduce<1>(m, slot[0], OpMaxNan());
    const float largest = m[0];
    const bool none = largest == -INFINITY;                      // no token is open
    float s[3] = {0.f, 0.f, 0.f};                                // how often m occurs, the other terms, sum of e (x - m)
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) {
      const float v = lp_load(x, i);
      if (v == largest) {
        s[0] += 1.f;
      } else {
        const float d = v - largest, e = expf(d);
        s[1] += e;
        s[2] += e == 0.f ? 0.f : e * d;
      }
    }
    block_reduce<3>(s, slot[1], OpSum());
    float logz = s[0] == 1.f ? log1pf(s[1]) : logf(s[0] + s[1]);
    if (none) logz = 0.f;
    if (!(largest < INFINITY)) logz = NAN;
    if (threadIdx.x == 0) {
      a.stats[2 * row] = largest;
      a.stats[2 * row + 1] = logz;
      if (a.entropy) a.entropy[row] = none ? 0.f : logz - s[2] / (s[0] + s[1]);
      if (a.targets) {
        float lp = NAN;                                          // a target outside the vocabulary
        if (target == a.ignore_index) lp = 0.f;
        else if (target >= 0 && target < a.vocab) lp = none ? -INFINITY : lp_load(x, target) - largest - logz;
        a.logprob[row] = lp;
      }
    }
    unsigned long long before = ~0ull;
    for (int k = 0; k < a.top; ++k) {
      unsigned long long key = 0;
      for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) {
        const unsigned long long q = lp_key(lp_load(x, i), i);
        if (q < before && q > key) key = q;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long q = __shfl_xor_sync(0xffffffffu, key, o);
        key = q > key ? q : key;
      }
      __syncthreads();
      if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = key;
      __syncthreads();
      for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) key = best[w] > key ? best[w] : key;
      if (threadIdx.x == 0) {
        const uint32_t i = 0xffffffffu - static_cast<uint32_t>(key);
        a.top_index[row * a.top + k] = i;
        a.top_logprob[row * a.top + k] = none ? -INFINITY : lp_load(x, i) - largest - logz;
      }
      before = key;
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(256) logprob_bwd_kernel(const LogprobBwdArgs a) {
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.logits) + (row / a.seq) * a.batch_stride + (row % a.seq) * a.row_stride;
    T* out = static_cast<T*>(a.grad) + row * a.vocab;
    const float m = a.stats[2 * row], logz = a.stats[2 * row + 1];
    const bool none = m == -INFINITY;
    long long target = a.targets ? a.targets[row] : a.ignore_index;
    float dt = a.d_logprob ? a.d_logprob[row] : 0.f;
    const bool counted = a.targets && a.d_logprob && target != a.ignore_index;
    if (!counted) dt = 0.f;
    if (counted && (target < 0 || target >= a.vocab)) dt = NAN;
    float whole = dt;
    for (int j = 0; a.d_top && j < a.top; ++j) whole += a.d_top[row * a.top + j];
    const float dh = a.d_entropy ? a.d_entropy[row] : 0.f, h = a.d_entropy ? a.entropy[row] : 0.f;
    for (int i = threadIdx.x; i < a.vocab; i += blockDim.x) {
      if (none) {
        lp_store(out, i, whole == whole ? 0.f : NAN);
        continue;
      }
      const float lp = lp_load(x, i) - m - logz, p = expf(lp);
      float share = counted && i == target ? dt : 0.f;
      for (int j = 0; a.d_top && j < a.top; ++j)
        if (a.top_index[row * a.top + j] == i) share += a.d_top[row * a.top + j];
      float g = share != 0.f ? (share - whole) * p - share * expm1f(lp) : -whole * p;
      if (a.d_entropy && p != 0.f) g -= dh * p * (lp + h);
      lp_store(out, i, g);
    }
  }
}

constexpr int kLpMaxVocab = 262144, kLpMaxTop = 32;

static int check_logprob(int64_t rows, int32_t vocab, int32_t dtype, int64_t seq, int64_t row_stride, int64_t batch_stride, int32_t top) {
  if (rows < 0 || vocab < 1 || seq < 1 || row_stride < 0 || batch_stride < 0) return HYC_ERR_SHAPE;
  if (top < 0 || top > vocab) return HYC_ERR_SHAPE;
  if (vocab > kLpMaxVocab || top > kLpMaxTop || rows > 0x7fffffffLL) return HYC_ERR_CAPACITY;
  if (dtype != HYC_F32 && dtype != HYC_BF16) return HYC_ERR_DTYPE;
  return HYC_OK;
}

static bool lp_misaligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

}  // namespace hyc

using namespace hyc;

extern "C" {

int hyc_token_logprobs(const hyc_logprob_args* q, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!q) return HYC_ERR_NULL;
  const int rc = check_logprob(q->rows, q->vocab, q->dtype, q->seq, q->row_stride, q->batch_stride, q->top);
  if (rc) return rc;
  if (q->rows == 0) return HYC_OK;
  if (!q->logits || !q->stats || (q->targets && !q->logprob) || (q->top && (!q->top_index || !q->top_logprob))) return HYC_ERR_NULL;
  if (lp_misaligned(q->logits, q->dtype == HYC_BF16 ? 2 : 4) || lp_misaligned(q->targets, 8) || lp_misaligned(q->logprob, 4) ||
      lp_misaligned(q->entropy, 4) || lp_misaligned(q->stats, 8) || lp_misaligned(q->top_logprob, 4) || lp_misaligned(q->top_index, 8))
    return HYC_ERR_ALIGN;
  LogprobArgs a;
  a.logits = q->logits; a.rows = q->rows; a.row_stride = q->row_stride; a.batch_stride = q->batch_stride; a.seq = q->seq;
  a.vocab = q->vocab; a.top = q->top; a.targets = reinterpret_cast<const long long*>(q->targets); a.ignore_index = q->ignore_index;
  a.logprob = q->logprob; a.entropy = q->entropy; a.stats = q->stats; a.top_logprob = q->top_logprob;
  a.top_index = reinterpret_cast<long long*>(q->top_index);
  const int grid = static_cast<int>(a.rows < 148 * 4 ? a.rows : 148 * 4);
  if (q->dtype == HYC_BF16)
    logprob_kernel<__nv_bfloat16><<<grid, 512, 0, stream>>>(a);
  else
    logprob_kernel<float><<<grid, 512, 0, stream>>>(a);
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "logprob_kernel");
}

int hyc_token_logprobs_bwd(const hyc_logprob_bwd_args* q, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!q) return HYC_ERR_NULL;
  const int rc = check_logprob(q->rows, q->vocab, q->dtype, q->seq, q->row_stride, q->batch_stride, q->top);
  if (rc) return rc;
  if (q->rows == 0) return HYC_OK;
  if (!q->logits || !q->stats || !q->grad || (q->d_logprob && !q->targets) || (q->d_entropy && !q->entropy) ||
      (q->d_top && !q->top_index))
    return HYC_ERR_NULL;
  const uintptr_t es = q->dtype == HYC_BF16 ? 2 : 4;
  if (lp_misaligned(q->logits, es) || lp_misaligned(q->grad, es) || lp_misaligned(q->targets, 8) || lp_misaligned(q->stats, 8) ||
      lp_misaligned(q->entropy, 4) || lp_misaligned(q->d_logprob, 4) || lp_misaligned(q->d_entropy, 4) || lp_misaligned(q->d_top, 4) ||
      lp_misaligned(q->top_index, 8))
    return HYC_ERR_ALIGN;
  LogprobBwdArgs a;
  a.logits = q->logits; a.rows = q->rows; a.row_stride = q->row_stride; a.batch_stride = q->batch_stride; a.seq = q->seq;
  a.vocab = q->vocab; a.top = q->d_top ? q->top : 0; a.targets = reinterpret_cast<const long long*>(q->targets);
  a.ignore_index = q->ignore_index; a.stats = q->stats; a.entropy = q->entropy; a.d_logprob = q->d_logprob;
  a.d_entropy = q->d_entropy; a.d_top = q->d_top; a.top_index = reinterpret_cast<const long long*>(q->top_index); a.grad = q->grad;
  const int grid = static_cast<int>(a.rows < 148 * 8 ? a.rows : 148 * 8);
  if (q->dtype == HYC_BF16)
    logprob_bwd_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else
    logprob_bwd_kernel<float><<<grid, 256, 0, stream>>>(a);
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "logprob_bwd_kernel");
}

}  // extern "C"
