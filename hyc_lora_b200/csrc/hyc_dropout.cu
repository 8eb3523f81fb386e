// Dropout with the mask drawn from a counter (hyc_philox.cuh), with or without the add of a residual:
//     y = residual + (keep ? x / (1 - p) : 0)
// The kept value x * scale, scale = 1 / (1 - p) in fp32, is rounded to fp32 before it is added: that rounding takes back what
// the rounding of scale brought in wherever x / (1 - p) has few digits (x = 9 k, p = 0.1).  Fused, scale's error went on into
// the sum: exact zeros came out as 1e-8 and ties of the output's rounding fell to one side.  The sum is rounded to fp32 and
// then once to the output's type.  What is dropped is selected away, not multiplied by zero: an infinity or a NaN in a
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

// product and sum each rounded (never contracted)
template <bool RES>
__device__ __forceinline__ float kept_sum(float x, float scale, float base) {
  const float kept = __fmul_rn(x, scale);
  return RES ? __fadd_rn(kept, base) : kept;
}

// Any addresses and strides.  One thread: the four elements of one counter block.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_any_kernel(const DropoutArgs a) {
  Philox gen = Philox::load(a.rng);
  const long long n = a.rows * a.cols, blocks = (n + 3) >> 2;
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  for (long long b = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; b < blocks;
       b += static_cast<long long>(gridDim.x) * blockDim.x) {
    const uint4 w4 = gen.at(static_cast<unsigned long long>(b));
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
    long long row = 4 * b / a.cols, col = 4 * b - row * a.cols;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (4 * b + e >= n) break;
      const float base = RES ? to_float<T>(res[row * a.residual_stride + col]) : 0.f;
      const float v = a.rate.none ? 0.f : to_float<T>(x[row * a.x_stride + col]);
      y[4 * b + e] = T(a.rate.keep(w[e]) ? kept_sum<RES>(v, a.rate.scale, base) : base);
      if (++col == a.cols) { col = 0; ++row; }
    }
  }
}

// One flat run of elements at 16-byte aligned addresses.  Persistent: a CTA takes tiles of U * NT pieces of 16 bytes and has the
// next tile's loads in flight while it draws this tile's words.  Without a residual and in bf16 it stands between two
// bounds that overlap in part, DRAM and the generator's products (see hyc_philox.cuh; their pipe is busy for 67 % of the time),
// else at DRAM's.  Many words per thread keep the multiplier fed: 16384 x 11008 bf16 takes 141 us (DRAM alone: 112; the
// products alone: 97) with U = 8 and 256 threads, 143 with 384, 160 with 512; at 8192 x 11008 U = 8 takes 74 us,
// U = 4 80, U = 2 83.  With a residual 384 threads of U = 4 take 69 us at 16384 x 4096 (DRAM: 62), 256 threads 75.

// eight bf16 values as fp32; both halves by byte permutes and masks, which leave the multiplier's pipe to the generator
__device__ __forceinline__ void piece_to_floats(const uint4& w, float (&f)[8]) {
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(__byte_perm(q[i], 0, 0x1044));
    f[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void piece_to_floats(const uint4& w, float (&f)[4]) {
  f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ uint4 floats_to_piece(const float (&f)[8]) { return pack_bf16x8(f); }
__device__ __forceinline__ uint4 floats_to_piece(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

template <typename T, bool RES, int U, int NT>
struct DropTile {
  static constexpr int kPiece = 16 / sizeof(T), kBlocks = kPiece / 4;
  uint4 x[U], r[U];

  __device__ __forceinline__ void load(const DropoutArgs& a, long long first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = load16_stream(static_cast<const uint4*>(a.x) + first + u * NT);
      if (RES) r[u] = load16_stream(static_cast<const uint4*>(a.residual) + first + u * NT);
    }
  }
  __device__ __forceinline__ static uint4 piece(const DropoutArgs& a, const Philox& gen, const uint4& xp, const uint4& rp, uint32_t block) {
    float f[kPiece], base[kPiece];
    piece_to_floats(xp, f);
    if (RES) piece_to_floats(rp, base);
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) {
      const uint4 w = gen.block(block + q);
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float b = RES ? base[4 * q + e] : 0.f;
        f[4 * q + e] = a.rate.keep(words[e]) ? kept_sum<RES>(f[4 * q + e], a.rate.scale, b) : b;
      }
    }
    return floats_to_piece(f);
  }
  __device__ __forceinline__ void finish(const DropoutArgs& a, Philox& gen, long long first) const {
    const unsigned long long block = static_cast<unsigned long long>(first) * kBlocks;
    if (static_cast<uint32_t>(block >> 32) != gen.upper) gen.prepare(static_cast<uint32_t>(block >> 32));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned long long at = block + u * NT * kBlocks;
      // tiles of a power of two never run across a change of the upper half
      if ((U * NT & (U * NT - 1)) != 0 && static_cast<uint32_t>(at >> 32) != gen.upper) gen.prepare(static_cast<uint32_t>(at >> 32));
      static_cast<uint4*>(a.y)[first + u * NT] = piece(a, gen, x[u], r[u], static_cast<uint32_t>(at));
    }
  }
};

template <typename T, bool RES, int U, int NT>
__global__ void __launch_bounds__(NT, 1) dropout_flat_kernel(const DropoutArgs a) {
  using Tile = DropTile<T, RES, U, NT>;
  constexpr int kTile = NT * U, kBlocks = Tile::kBlocks;
  Philox gen = Philox::load(a.rng);
  const long long pieces = a.cols / Tile::kPiece, tiles = pieces / kTile;
  if (!a.rate.none) {
    Tile one, two;
    long long tile = blockIdx.x;
    if (tile < tiles) one.load(a, tile * kTile + threadIdx.x);
    while (tile < tiles) {
      long long next = tile + gridDim.x;
      if (next < tiles) two.load(a, next * kTile + threadIdx.x);
      one.finish(a, gen, tile * kTile + threadIdx.x);
      if (next >= tiles) break;
      tile = next;
      next += gridDim.x;
      if (next < tiles) one.load(a, next * kTile + threadIdx.x);
      two.finish(a, gen, tile * kTile + threadIdx.x);
      tile = next;
    }
  } else {
    for (long long p = static_cast<long long>(blockIdx.x) * NT + threadIdx.x; p < tiles * kTile; p += static_cast<long long>(gridDim.x) * NT)
      static_cast<uint4*>(a.y)[p] = RES ? static_cast<const uint4*>(a.residual)[p] : make_uint4(0, 0, 0, 0);
  }
  // the pieces behind the last whole tile, and the elements behind the last piece
  if (blockIdx.x != tiles % gridDim.x) return;
  for (long long p = tiles * kTile + threadIdx.x; p < pieces; p += NT) {
    const unsigned long long block = static_cast<unsigned long long>(p) * kBlocks;
    if (static_cast<uint32_t>(block >> 32) != gen.upper) gen.prepare(static_cast<uint32_t>(block >> 32));
    const uint4 zero = make_uint4(0, 0, 0, 0);
    static_cast<uint4*>(a.y)[p] = Tile::piece(a, gen, a.rate.none ? zero : static_cast<const uint4*>(a.x)[p],
                                              RES ? static_cast<const uint4*>(a.residual)[p] : zero, static_cast<uint32_t>(block));
  }
  const long long e = pieces * Tile::kPiece + threadIdx.x;
  if (e < a.cols) {
    const uint4 w = gen.at(static_cast<unsigned long long>(e >> 2));
    const int lane = static_cast<int>(e & 3);
    const float base = RES ? to_float<T>(static_cast<const T*>(a.residual)[e]) : 0.f;
    const bool keep = a.rate.keep(lane == 0 ? w.x : lane == 1 ? w.y : lane == 2 ? w.z : w.w);
    const float last = a.rate.none ? 0.f : to_float<T>(static_cast<const T*>(a.x)[e]);
    static_cast<T*>(a.y)[e] = T(keep ? kept_sum<RES>(last, a.rate.scale, base) : base);
  }
}

__global__ void rng_take_kernel(unsigned long long* state, long long* used) {
  used[0] = static_cast<long long>(state[0]);
  used[1] = static_cast<long long>(atomicAdd(state + 1, 1ull));
}

template <typename T, bool RES, int U, int NT>
static void run_dropout_flat(const DropoutArgs& a, cudaStream_t stream) {
  auto kernel = dropout_flat_kernel<T, RES, U, NT>;
  const long long blocks = a.cols / (NT * U * (16 / sizeof(T))) + 1;
  static PerDevice resident;
  const int held = resident.get([&] { return held_at_once(kernel, NT, 0); });
  const long long most = held ? held : sm_count();
  kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), NT, 0, stream>>>(a);
}

template <typename T>
static int launch_dropout(const DropoutArgs& a, cudaStream_t stream) {
  const bool flat = a.rows == 1 && aligned16(a.x) && aligned16(a.y) && aligned16(a.residual);
  if (flat) {
    // One piece per thread, on as many SMs as there are, for small tensors.  Measured, us, one piece / many per thread: fp32 of
    // 6 MB 4.2 / 6.4; bf16 of 18 MB 12.4 / 10.3, of 36 MB 22.3 / 18.5; with a residual of 18 MB 12.4 / 13.5, of 36 MB 24.8 / 22.9.
    const bool large = a.cols * static_cast<long long>(sizeof(T)) >= 16LL * 256 * 8 * (a.residual ? 4 : 2) * sm_count();
    if (a.residual) {
      if (large) run_dropout_flat<T, true, 4, 384>(a, stream);
      else run_dropout_flat<T, true, 1, 256>(a, stream);
    } else {
      if (large) run_dropout_flat<T, false, 8, 256>(a, stream);
      else run_dropout_flat<T, false, 1, 256>(a, stream);
    }
  } else {
    const long long blocks = (a.rows * a.cols + 1023) / 1024;
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
  if (a.x_stride == a.cols && (!a.residual || a.residual_stride == a.cols)) {      // rows without gaps: one flat run
    a.cols *= a.rows;
    a.rows = 1;
  }
  return args->dtype == HYC_BF16 ? launch_dropout<__nv_bfloat16>(a, static_cast<cudaStream_t>(stream))
                                 : launch_dropout<float>(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
