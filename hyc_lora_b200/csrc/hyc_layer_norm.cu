// Layer norm of a residual sum, forward and backward, with dropout on the branch that joins the residual:
//     z = residual + dropout(x),  y = (z - mean(z)) * rstd(z) * weight + bias
//     with u = (z - mean) * rstd and g = dy * weight:
//     dz = (g - mean(g) - u * mean(g * u)) * rstd [+ the gradient that reaches z from elsewhere]
//     dx = keep ? dz / (1 - p) : 0, dresidual = dz, dweight = sum over rows of dy * u, dbias = sum over rows of dy
// Statistics, sums and gradients are held in fp32; every output is rounded once.  What the dropout keeps is rounded to fp32
// before the residual is added, as in hyc_dropout.cu.  The forward pass normalises the unrounded sum; the backward pass starts
// from z as it was stored.
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
// of the row, statistics in two exact passes over registers, one write.  A thread has VPT slots of eight elements.
//   VEC 1  16-byte pieces (8 bf16 or 4 fp32): thread t owns the pieces t, t + G, ...; every address of every row is 16-byte
//          aligned and a row is a multiple of eight elements;
//   VEC 2  the same where the row fills its threads' slots exactly: no bounds are left to test;
//   VEC 0  single elements, for odd widths and unaligned tensors: a warp's chunks of 128 consecutive ones, four sweeps of its
//          lanes each, a chunk per half slot.

// single elements, by the read-only path: no store in between holds the loads back
__device__ __forceinline__ float ln_one(const float* p) { return __ldg(p); }
__device__ __forceinline__ float ln_one(const __nv_bfloat16* p) {
  return __uint_as_float(static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(p))) << 16);
}

template <int VEC>
__device__ __forceinline__ bool ln_in(int c, int cols) { return VEC == 2 || c < cols; }

template <typename T, int G, int VEC>
__device__ __forceinline__ int ln_col(int t, int v, int j) {
  if (!VEC) return ((2 * v + (j >> 2)) * G + (t & ~31)) * 4 + (j & 3) * 32 + (t & 31);
  return sizeof(T) == 2 ? (v * G + t) * 8 + j : ((2 * v + (j >> 2)) * G + t) * 4 + (j & 3);
}

// Single elements: whether any thread of the warp has one of the row in slot v; else the warp passes over it.  The backward pass
// does so for the words alone: with branches around its loads 16384 x 1003 takes 94 us, not 82.  The forward pass gains by them
// (8192 x 4099: 219 us, not 322).
template <typename T, int G, int VEC>
__device__ __forceinline__ bool ln_any(int t, int v, int cols) { return VEC != 0 || ln_col<T, G, VEC>(t & ~31, v, 0) < cols; }

// a 16-byte piece as fp32 pairs, at f
__device__ __forceinline__ void ln_unpack(const uint4& w, __nv_bfloat16, f32x2* f) {
  // byte permutes and masks: the multiplier's pipe is left to the generator's products
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f2_make(__uint_as_float(__byte_perm(q[i], 0, 0x1044)), __uint_as_float(q[i] & 0xffff0000u));
}
__device__ __forceinline__ void ln_unpack(const uint4& w, float, f32x2* f) {
  f[0] = f2_make(__uint_as_float(w.x), __uint_as_float(w.y));
  f[1] = f2_make(__uint_as_float(w.z), __uint_as_float(w.w));
}
// A packed add takes both halves of the fp32 pipe, one of which also multiplies integers; two single ones can keep to the other.
// Beside the generator that is worth the issue slots in the rows of several warps (65536 x 4096 backward with dropout: 468 us,
// not 486), in those of one warp it is not (65536 x 768: 84 us, not 82.5).
template <bool APART>
__device__ __forceinline__ f32x2 ln_add(f32x2 a, f32x2 b) {
  if (!APART) return f2_add(a, b);
  float a0, a1, b0, b1;
  f2_split(a, a0, a1);
  f2_split(b, b0, b1);
  return f2_make(a0 + b0, a1 + b1);
}
__device__ __forceinline__ f32x2 f2_both(float v) { return f2_make(v, v); }

// the eight elements of slot v of thread t as four pairs, zero beyond the row's end
template <typename T, int G, int VEC, bool SKIP = false>
__device__ __forceinline__ void ln_get(const void* row, int t, int v, int cols, f32x2 (&f)[4]) {
  if (SKIP && !ln_any<T, G, VEC>(t, v, cols)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = 0;
    return;
  }
  if (VEC) {
    constexpr int kPiece = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / kPiece; ++h) {
      const int c = ln_col<T, G, VEC>(t, v, h * kPiece);
      ln_unpack(ln_in<VEC>(c, cols) ? load16_stream(static_cast<const T*>(row) + c) : make_uint4(0, 0, 0, 0), T(0.f), f + h * (kPiece / 2));
    }
  } else {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = ln_col<T, G, VEC>(t, v, j);
      if (sizeof(T) == 2) {                   // 16-bit loads under a condition are branched around, one wait each: 103 us, not 68
        const float one = ln_one(static_cast<const T*>(row) + min(c, cols - 1));
        e[j] = c < cols ? one : 0.f;
      } else {
        e[j] = c < cols ? ln_one(static_cast<const T*>(row) + c) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = f2_make(e[2 * i], e[2 * i + 1]);
  }
}

template <typename T, int G, int VEC, bool SKIP = false>
__device__ __forceinline__ void ln_put(void* row, int t, int v, int cols, const f32x2 (&p)[4]) {
  if (SKIP && !ln_any<T, G, VEC>(t, v, cols)) return;
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_split(p[i], f[2 * i], f[2 * i + 1]);
  if (VEC) {
    constexpr int kPiece = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / kPiece; ++h) {
      const int c = ln_col<T, G, VEC>(t, v, h * kPiece);
      if (!ln_in<VEC>(c, cols)) continue;
      uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(row) + c);
      if (sizeof(T) == 2) *to = pack_bf16x8(f);
      else *to = make_uint4(__float_as_uint(f[4 * h]), __float_as_uint(f[4 * h + 1]), __float_as_uint(f[4 * h + 2]), __float_as_uint(f[4 * h + 3]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = ln_col<T, G, VEC>(t, v, j);
      if (c < cols) static_cast<T*>(row)[c] = T(f[j]);
    }
  }
}

// weight or bias: read again for every row (L1 keeps them), as fp32
template <typename T, int G, int VEC>
__device__ __forceinline__ void ln_param(const void* p, bool bf16, int t, int v, int cols, float fill, f32x2 (&f)[4]) {
  if (VEC != 2 || !p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = f2_both(fill);
    if (!p) return;
  }
  if (VEC) {
    constexpr int kRun = 16 / sizeof(T);                   // consecutive columns of a thread
#pragma unroll
    for (int h = 0; h < 8 / kRun; ++h) {
      const int c = ln_col<T, G, VEC>(t, v, h * kRun);
      if (!ln_in<VEC>(c, cols)) continue;
#pragma unroll
      for (int q = 0; q < kRun / 4; ++q) {
        f32x2* to = f + h * (kRun / 2) + q * 2;
        if (bf16) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + c + 4 * q));
          to[0] = f2_make(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u));
          to[1] = f2_make(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
        } else {
          const float4 w = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + c + 4 * q));
          to[0] = f2_make(w.x, w.y);
          to[1] = f2_make(w.z, w.w);
        }
      }
    }
  } else {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = fill;                           // beyond the end: any finite value
    if (bf16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = ln_one(static_cast<const __nv_bfloat16*>(p) + min(ln_col<T, G, VEC>(t, v, j), cols - 1));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = ln_col<T, G, VEC>(t, v, j);
        if (c < cols) e[j] = ln_one(static_cast<const float*>(p) + c);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = f2_make(e[2 * i], e[2 * i + 1]);
  }
}

// The same from a table in shared memory that a persistent CTA fills once: fp32, a thread's four columns of a half slot in
// one 16-byte piece and the pieces of consecutive threads side by side.  Read from L1 for every row instead, the parameters
// cost the forward pass 250 us against 203 and the backward pass 174 against 145 (32768 x 4096 bf16; half of those reads miss
// next to the streams).
template <typename T, int G>
__device__ __forceinline__ void ln_table_fill(float* table, const void* p, bool bf16, int cols, int slots, float fill) {
  for (int c = threadIdx.x; c < slots * 8 * G; c += blockDim.x) {
    float value = fill;
    if (p && c < cols) value = bf16 ? static_cast<float>(static_cast<const __nv_bfloat16*>(p)[c]) : static_cast<const float*>(p)[c];
    const int piece = c >> 3;
    table[sizeof(T) == 4 ? c : ((piece / G * 2 + (c >> 2 & 1)) * G + piece % G) * 4 + (c & 3)] = value;
  }
}
template <int G>
__device__ __forceinline__ void ln_table_get(const float* table, int t, int v, f32x2 (&f)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(table + ((2 * v + h) * G + t) * 4);
    f[2 * h] = w.x;
    f[2 * h + 1] = w.y;
  }
}

// base + (kept ? x * scale : 0) of a slot; `first` is the index of the row's first element in the tensor.  VEC: a thread draws
// the words of its own elements, whole counter blocks.  Else a chunk of 128 elements starts s = first % 4 elements into a
// block: lane l draws the chunk's block l, ballots tell every lane all 128 keep bits, and the 33rd block, which the chunk's
// last s elements are in, has been drawn for all chunks of the row at once (ln_ends: lane q holds its bits for chunk q).
template <int G, int VPT, int VEC>
__device__ __forceinline__ uint32_t ln_ends(Philox& gen, const DropRate& rate, unsigned long long first, int t) {
  if (VEC || (first & 3) == 0) return 0;
  const unsigned q = t & 31;
  const uint4 w = gen.at(((first + (static_cast<unsigned>(q % (2 * VPT)) * G + (t & ~31)) * 4) >> 2) + 32);
  return (rate.keep(w.x) ? 1u : 0u) | (rate.keep(w.y) ? 2u : 0u) | (rate.keep(w.z) ? 4u : 0u) | (rate.keep(w.w) ? 8u : 0u);
}

template <typename T, int G, int VEC, bool BASE>
__device__ __forceinline__ void ln_drop(Philox& gen, const DropRate& rate, unsigned long long first, uint32_t ends, int t, int v,
                                        f32x2 (&x)[4], const f32x2 (&base)[4]) {
  bool keep[8];
  if (VEC) {                                   // rows of a multiple of eight elements: two whole counter blocks
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // bf16: the second block follows the first, whose index is even: it has the same upper half
      const unsigned long long at = (first + static_cast<unsigned>(ln_col<T, G, VEC>(t, v, sizeof(T) == 2 ? 0 : 4 * h))) >> 2;
      if (sizeof(T) == 4 || h == 0) {
        if (static_cast<uint32_t>(at >> 32) != gen.upper) gen.prepare(static_cast<uint32_t>(at >> 32));
      }
      const uint4 q = gen.block(static_cast<uint32_t>(at) + (sizeof(T) == 2 ? h : 0));
      keep[4 * h] = rate.keep(q.x); keep[4 * h + 1] = rate.keep(q.y); keep[4 * h + 2] = rate.keep(q.z); keep[4 * h + 3] = rate.keep(q.w);
    }
  } else {
    const int lane = t & 31, s = static_cast<int>(first & 3), word = (s + lane) & 3, block = (s + lane) >> 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned long long chunk = first + static_cast<unsigned>(ln_col<T, G, VEC>(t & ~31, v, 4 * h));
      const uint4 q = gen.at((chunk >> 2) + lane);
      const uint32_t b0 = __ballot_sync(0xffffffffu, rate.keep(q.x)), b1 = __ballot_sync(0xffffffffu, rate.keep(q.y));
      const uint32_t b2 = __ballot_sync(0xffffffffu, rate.keep(q.z)), b3 = __ballot_sync(0xffffffffu, rate.keep(q.w));
      const uint32_t bits = word == 0 ? b0 : word == 1 ? b1 : word == 2 ? b2 : b3;
      const uint32_t end = __shfl_sync(0xffffffffu, ends, 2 * v + h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 8 * j + block;                    // 0 .. 32
        keep[4 * h + j] = j == 3 && at == 32 ? end >> word & 1 : bits >> (at & 31) & 1;
      }
    }
  }
  if (rate.none) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = f2_both(0.f);
  }
  const f32x2 scale = f2_both(rate.scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2_split(f2_mul(x[i], scale), lo, hi);
    x[i] = f2_make(keep[2 * i] ? lo : 0.f, keep[2 * i + 1] ? hi : 0.f);
    if (BASE) x[i] = f2_add(x[i], base[i]);            // behind the choice: next to each other the two packed ones become an FMA
  }
}

// The rows to come of a group, on their way into shared memory while this one is worked on.  Every thread copies the pieces
// that it will read itself, so the copies need no barrier: a thread waits for its own (cp.async.wait_group).  One commit per
// turn, also where there is nothing left to copy, keeps the count.
template <typename T, int G, int VPT, int VEC, int ARRAYS, int STAGES, int THREADS>
struct LnRing {
  static constexpr int kPieces = VPT * 8 * static_cast<int>(sizeof(T)) / 16;
  static constexpr uint32_t kStageBytes = ARRAYS * kPieces * THREADS * 16u, kBytes = STAGES * kStageBytes;
  unsigned char* own;

  __device__ __forceinline__ void init(unsigned char* smem) { own = smem + threadIdx.x * 16; }
  __device__ __forceinline__ unsigned char* slot(int stage, int array, int piece) const {
    return own + stage * kStageBytes + (array * kPieces + piece) * (THREADS * 16);
  }
  __device__ __forceinline__ void copy(int stage, int array, const void* row, int t, int cols) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int c = (i * G + t) * (16 / static_cast<int>(sizeof(T)));
      if (ln_in<VEC>(c, cols))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(slot(stage, array, i))),
                     "l"(__cvta_generic_to_global(static_cast<const T*>(row) + c))
                     : "memory");
    }
  }
  __device__ __forceinline__ void commit() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ __forceinline__ void wait() const { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }
  __device__ __forceinline__ void get(int stage, int array, int t, int v, int cols, f32x2 (&f)[4]) const {
    constexpr int kPiece = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / kPiece; ++h) {
      const int i = v * (8 / kPiece) + h;
      const bool in = ln_in<VEC>((i * G + t) * kPiece, cols);
      ln_unpack(in ? *reinterpret_cast<const uint4*>(slot(stage, array, i)) : make_uint4(0, 0, 0, 0), T(0.f), f + h * (kPiece / 2));
    }
  }
};

// A thread's place in its group, and its group's in the CTA -- the same in every thread of a warp, which a warp-wide
// reduction lets the compiler know, so that rows' addresses are worked out once per warp, off the multiplier's pipe.
template <int G, int GROUPS>
__device__ __forceinline__ int group_thread() { return GROUPS == 1 ? threadIdx.x : threadIdx.x % G; }
template <int G, int GROUPS>
__device__ __forceinline__ int group_index() {
  return GROUPS == 1 ? 0 : static_cast<int>(__reduce_max_sync(0xffffffffu, threadIdx.x / G));
}

template <int G>
__device__ __forceinline__ void group_sync() {
  if (G == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / G), "n"(G) : "memory");
}

// Sums over the G threads of a group, the same bits in every thread.  `slot` is the group's own (2 * G / 32 floats, 16-byte
// aligned) and is not used again before the group has met at another barrier.
template <int G>
__device__ __forceinline__ float group_sum(float v, float* slot) {
  static_assert(G == 32 || G % 128 == 0, "warps are read four at a time");
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (G == 32) return v;
  if ((threadIdx.x & 31) == 0) slot[(threadIdx.x % G) >> 5] = v;
  group_sync<G>();
  float r = 0.f;
#pragma unroll
  for (int w = 0; w < G / 128; ++w) {
    const float4 p = *reinterpret_cast<const float4*>(slot + 4 * w);
    r += (p.x + p.y) + (p.z + p.w);
  }
  return r;
}
// two at once: after the first exchange each half of a warp carries one of them
template <int G>
__device__ __forceinline__ float2 group_sum2(float v0, float v1, float* slot) {
  static_assert(G == 32 || G % 64 == 0, "warps are read two at a time");
  const bool upper = threadIdx.x & 16;
  float v = (upper ? v1 : v0) + __shfl_xor_sync(0xffffffffu, upper ? v0 : v1, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (G == 32) return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
  if ((threadIdx.x & 15) == 0) slot[((threadIdx.x % G) >> 5) * 2 + (upper ? 1 : 0)] = v;
  group_sync<G>();
  float2 r = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < G / 64; ++w) {
    const float4 p = *reinterpret_cast<const float4*>(slot + 4 * w);
    r.x += p.x + p.z;
    r.y += p.y + p.w;
  }
  return r;
}

// ---------------------------------------------------------------- forward

// z in registers (where the residual, if any, has been read into r) -> statistics, y, z
template <typename T, int G, int VPT, bool DROP, int VEC, bool TABLE>
__device__ __forceinline__ void ln_fwd_row(const LnFwdArgs& a, Philox& gen, long long row, int t, f32x2 (&z)[VPT][4], f32x2 (&r)[VPT][4],
                                           float* slot, const float* table) {
  f32x2 s2 = f2_both(0.f);
  const unsigned long long element = static_cast<unsigned long long>(row) * a.cols;
  uint32_t ends = 0;
  if (DROP) ends = ln_ends<G, VPT, VEC>(gen, a.rate, element, t);
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    if (DROP) {
      if (ln_any<T, G, VEC>(t, v, a.cols)) ln_drop<T, G, VEC, true>(gen, a.rate, element, ends, t, v, z[v], r[v]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) z[v][i] = f2_add(z[v][i], r[v][i]);
    }
    s2 = f2_add(s2, f2_add(f2_add(z[v][0], z[v][1]), f2_add(z[v][2], z[v][3])));      // zero beyond the row's end
  }
  float lo, hi;
  f2_split(s2, lo, hi);
  const float mean = group_sum<G>(lo + hi, slot) / a.cols;
  const f32x2 minus_mean = f2_both(-mean);
  f32x2 q2 = f2_both(0.f);
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 d = f2_add(z[v][i], minus_mean);
      if (VEC) {
        if (ln_in<VEC>(ln_col<T, G, VEC>(t, v, 2 * i), a.cols)) q2 = f2_fma(d, d, q2);   // a piece is in the row or is not
      } else {
        f2_split(d, lo, hi);
        if (ln_col<T, G, VEC>(t, v, 2 * i) >= a.cols) lo = 0.f;
        if (ln_col<T, G, VEC>(t, v, 2 * i + 1) >= a.cols) hi = 0.f;
        const f32x2 in = f2_make(lo, hi);
        q2 = f2_fma(in, in, q2);
      }
    }
  }
  f2_split(q2, lo, hi);
  const float rstd = rsqrtf(group_sum<G>(lo + hi, slot + 32) / a.cols + a.eps);
  if (t == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  void* y = static_cast<T*>(a.y) + row * a.cols;
  if (a.z) {
    void* zp = static_cast<T*>(a.z) + row * a.cols;
#pragma unroll
    for (int v = 0; v < VPT; ++v) ln_put<T, G, VEC, true>(zp, t, v, a.cols, z[v]);
  }
  const f32x2 rstd2 = f2_both(rstd);
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    f32x2 w[4], b[4];
    if (TABLE) {
      ln_table_get<G>(table, t, v, w);
      ln_table_get<G>(table + VPT * 8 * G, t, v, b);
    } else {
      ln_param<T, G, VEC>(a.weight, a.param_bf16, t, v, a.cols, 1.f, w);
      ln_param<T, G, VEC>(a.bias, a.param_bf16, t, v, a.cols, 0.f, b);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f2_fma(f2_mul(f2_add(z[v][i], minus_mean), rstd2), w[i], b[i]);
    ln_put<T, G, VEC, true>(y, t, v, a.cols, w);
  }
}

// Persistent groups of G threads, rows ahead in the ring (long inputs).
template <typename T, int G, int VPT, bool DROP, int VEC, int STAGES, bool TABLE>
__global__ void __launch_bounds__(G < 256 ? 256 : G, G == 512 ? 1 : VPT <= 2 ? 3 : 2) ln_fwd_ring_kernel(const LnFwdArgs a) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G;
  extern __shared__ __align__(16) unsigned char staged[];
  __shared__ __align__(16) float slots[kGroups][2][64];
  const int t = group_thread<G, kGroups>(), group = group_index<G, kGroups>();
  using Ring = LnRing<T, G, VPT, VEC, 2, STAGES, kThreads>;
  Ring ring;
  ring.init(staged);
  float* table = reinterpret_cast<float*>(staged + Ring::kBytes);
  if (TABLE) {
    ln_table_fill<T, G>(table, a.weight, a.param_bf16, a.cols, VPT, 1.f);
    ln_table_fill<T, G>(table + VPT * 8 * G, a.bias, a.param_bf16, a.cols, VPT, 0.f);
    __syncthreads();
  }
  Philox gen = {};
  if (DROP) gen = Philox::load(a.rng);
  const long long step = static_cast<long long>(gridDim.x) * kGroups;
  const long long first = static_cast<long long>(blockIdx.x) * kGroups + group;
  auto ahead = [&](int stage, long long row) {
    if (row < a.rows) {
      ring.copy(stage, 0, static_cast<const T*>(a.x) + row * a.x_stride, t, a.cols);
      if (a.residual) ring.copy(stage, 1, static_cast<const T*>(a.residual) + row * a.residual_stride, t, a.cols);
    }
    ring.commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s) ahead(s, first + s * step);
  int stage = 0, turn = 0;
  for (long long row = first; row < a.rows; row += step) {
    ring.wait();
    f32x2 z[VPT][4], r[VPT][4];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      ring.get(stage, 0, t, v, a.cols, z[v]);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[v][i] = 0;
      if (a.residual) ring.get(stage, 1, t, v, a.cols, r[v]);
    }
    ahead(stage, row + STAGES * step);
    if (++stage == STAGES) stage = 0;
    ln_fwd_row<T, G, VPT, DROP, VEC, TABLE>(a, gen, row, t, z, r, slots[group][turn], table);
    turn ^= 1;
  }
}

// One row per group (inputs of few rows, where a ring would only lengthen the way; rows without 16-byte alignment).  Three CTAs
// an SM: 4096 x 768 with dropout and residual is one wave, 8.4 us; with the registers of two 10.3.
template <typename T, int G, int VPT, bool DROP, int VEC>
__global__ void __launch_bounds__(G < 256 ? 256 : G, G == 512 ? 1 : 3) ln_fwd_kernel(const LnFwdArgs a) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G;
  __shared__ __align__(16) float slots[kGroups][64];
  const int t = group_thread<G, kGroups>(), group = group_index<G, kGroups>();
  const long long row = static_cast<long long>(blockIdx.x) * kGroups + group;
  if (row >= a.rows) return;
  const void* x = static_cast<const T*>(a.x) + row * a.x_stride;
  f32x2 z[VPT][4], r[VPT][4];
#pragma unroll
  for (int v = 0; v < VPT; ++v) ln_get<T, G, VEC, true>(x, t, v, a.cols, z[v]);
  if (a.residual) {
    const void* res = static_cast<const T*>(a.residual) + row * a.residual_stride;
#pragma unroll
    for (int v = 0; v < VPT; ++v) ln_get<T, G, VEC, true>(res, t, v, a.cols, r[v]);
  } else {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) r[v][i] = 0;
  }
  Philox gen = {};
  if (DROP) gen = Philox::load(a.rng);
  ln_fwd_row<T, G, VPT, DROP, VEC, false>(a, gen, row, t, z, r, slots[group], nullptr);
}

// ---------------------------------------------------------------- backward

// Where the parameter gradients of a thread's own columns add up over its rows: registers, or (rows so wide that they would
// not fit beside the row) shared memory, one conflict-free column of it per thread.  Pairs of columns.
template <int VPT, bool SMEM, int THREADS, bool APART>
struct LnAcc {
  f32x2 w[VPT][4], b[VPT][4];
  __device__ __forceinline__ void init(void*) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[v][i] = b[v][i] = 0;
  }
  __device__ __forceinline__ void add(int v, int i, f32x2 dy, f32x2 u) {
    w[v][i] = f2_fma(dy, u, w[v][i]);
    b[v][i] = ln_add<APART>(dy, b[v][i]);
  }
  __device__ __forceinline__ ulonglong2 get(int v, int i) const { return make_ulonglong2(w[v][i], b[v][i]); }
};
template <int VPT, int THREADS, bool APART>
struct LnAcc<VPT, true, THREADS, APART> {
  ulonglong2* own;
  __device__ __forceinline__ void init(void* smem) {
    own = static_cast<ulonglong2*>(smem) + threadIdx.x;
    for (int i = 0; i < VPT * 4; ++i) own[i * THREADS] = make_ulonglong2(0, 0);
  }
  __device__ __forceinline__ void add(int v, int i, f32x2 dy, f32x2 u) {
    ulonglong2 s = own[(v * 4 + i) * THREADS];
    s.x = f2_fma(dy, u, s.x);
    s.y = f2_add(dy, s.y);
    own[(v * 4 + i) * THREADS] = s;
  }
  __device__ __forceinline__ ulonglong2 get(int v, int i) const { return own[(v * 4 + i) * THREADS]; }
};

// Persistent groups: group g of CTA b takes the rows b * kGroups + g, + gridDim * kGroups, ...  A row is read once; its
// gradient is written while the columns' sums stay with their thread, and leave once per CTA as a row of partial sums.
// STAGES > 0: rows ahead in the ring (VEC only).  Beyond a row's end dy is zero, and with it all that is summed.
template <typename T, int G, int VPT, bool DROP, int VEC, bool SMEM, int STAGES>
__global__ void __launch_bounds__(G < 256 ? 256 : G, G == 512 || VPT > 2 ? 1 : 2) ln_bwd_kernel(const LnBwdArgs a) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G;
  extern __shared__ __align__(16) unsigned char staged[];
  __shared__ __align__(16) float slots[kGroups][2][32];
  const int t = group_thread<G, kGroups>(), group = group_index<G, kGroups>();
  constexpr bool kApart = DROP && G > 32;
  LnAcc<VPT, SMEM, kThreads, kApart> acc;
  acc.init(staged);
  Philox gen = {};
  if (DROP) gen = Philox::load(a.rng);
  constexpr int kStages = STAGES > 0 ? STAGES : 1;
  using Ring = LnRing<T, G, VPT, VEC, 2, kStages, kThreads>;
  Ring ring;
  ring.init(staged);
  float* table = reinterpret_cast<float*>(staged + Ring::kBytes);      // with the ring only
  if (STAGES > 0) {
    ln_table_fill<T, G>(table, a.weight, a.param_bf16, a.cols, VPT, 1.f);
    __syncthreads();
  }
  const long long step = static_cast<long long>(gridDim.x) * kGroups;
  const long long first = static_cast<long long>(blockIdx.x) * kGroups + group;
  auto ahead = [&](int stage, long long row) {
    if (row < a.rows) {
      ring.copy(stage, 0, static_cast<const T*>(a.dy) + row * a.dy_stride, t, a.cols);
      ring.copy(stage, 1, static_cast<const T*>(a.z) + row * a.z_stride, t, a.cols);
    }
    ring.commit();
  };
  if (STAGES > 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) ahead(s, first + s * step);
  }
  float mean = 0.f, rstd = 0.f;
  if (first < a.rows) { mean = a.mean[first]; rstd = a.rstd[first]; }
  const float per_col = 1.f / a.cols;
  int stage = 0, turn = 0;
  for (long long row = first; row < a.rows; row += step, turn ^= 1) {
    f32x2 g[VPT][4], u[VPT][4];
    if (STAGES > 0) {
      ring.wait();
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        ring.get(stage, 0, t, v, a.cols, g[v]);
        ring.get(stage, 1, t, v, a.cols, u[v]);
      }
      ahead(stage, row + kStages * step);
      if (++stage == kStages) stage = 0;
    } else {
      const void* dyp = static_cast<const T*>(a.dy) + row * a.dy_stride;
      const void* zp = static_cast<const T*>(a.z) + row * a.z_stride;
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        ln_get<T, G, VEC>(dyp, t, v, a.cols, g[v]);
        ln_get<T, G, VEC>(zp, t, v, a.cols, u[v]);
      }
    }
    const f32x2 minus_mean = f2_both(-mean), rstd2 = f2_both(rstd);
    if (row + step < a.rows) { mean = a.mean[row + step]; rstd = a.rstd[row + step]; }      // the next row's, ahead of their use
    f32x2 s0 = 0, s1 = 0;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      f32x2 w[4];
      if (STAGES > 0) ln_table_get<G>(table, t, v, w);
      else ln_param<T, G, VEC>(a.weight, a.param_bf16, t, v, a.cols, 1.f, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[v][i] = f2_mul(ln_add<kApart>(u[v][i], minus_mean), rstd2);
        acc.add(v, i, g[v][i], u[v][i]);
        g[v][i] = f2_mul(g[v][i], w[i]);
        s0 = ln_add<kApart>(s0, g[v][i]);
        s1 = f2_fma(g[v][i], u[v][i], s1);
      }
    }
    float a0, a1, b0, b1;
    f2_split(s0, a0, a1);
    f2_split(s1, b0, b1);
    const float2 s = group_sum2<G>(a0 + a1, b0 + b1, slots[group][turn]);
    const f32x2 minus_c2 = f2_both(-s.x * per_col), minus_c1 = f2_both(-s.y * per_col);
    uint32_t ends = 0;
    if (DROP) ends = ln_ends<G, VPT, VEC>(gen, a.rate, static_cast<unsigned long long>(row) * a.cols, t);
    void* out = static_cast<T*>(a.dresidual) + row * a.cols;
    void* dx = static_cast<T*>(a.dx) + row * a.cols;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      f32x2 d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = f2_mul(f2_fma(u[v][i], minus_c1, ln_add<kApart>(g[v][i], minus_c2)), rstd2);
      if (a.dz) {
        f32x2 e[4];
        ln_get<T, G, VEC>(static_cast<const T*>(a.dz) + row * a.dz_stride, t, v, a.cols, e);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = f2_add(d[i], e[i]);
      }
      ln_put<T, G, VEC>(out, t, v, a.cols, d);
      if (DROP && ln_any<T, G, VEC>(t, v, a.cols)) {
        ln_drop<T, G, VEC, false>(gen, a.rate, static_cast<unsigned long long>(row) * a.cols, ends, t, v, d, d);
        ln_put<T, G, VEC>(dx, t, v, a.cols, d);
      }
    }
  }
  if (!a.partials) return;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  float* part = a.partials + static_cast<long long>(blockIdx.x) * 2 * a.cols;
  auto leave = [&](int c0, int c1, const ulonglong2& p) {
    float lo, hi;
    f2_split(p.x, lo, hi);
    if (c0 < a.cols) part[c0] = lo;
    if (c1 < a.cols) part[c1] = hi;
    f2_split(p.y, lo, hi);
    if (c0 < a.cols) part[a.cols + c0] = lo;
    if (c1 < a.cols) part[a.cols + c1] = hi;
  };
  if (kGroups == 1) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) leave(ln_col<T, G, VEC>(t, v, 2 * i), ln_col<T, G, VEC>(t, v, 2 * i + 1), acc.get(v, i));
    return;
  }
  // The groups of a CTA, summed in their order through shared memory: [group][pair][thread].  Nothing of the ring is under way
  // any more (its last commits are of nothing), and the barrier is behind every thread's last read of it.
  ulonglong2* all = reinterpret_cast<ulonglong2*>(staged);
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) all[(group * 4 + i) * G + t] = acc.get(v, i);
    __syncthreads();
    for (int k = threadIdx.x; k < 4 * G; k += kThreads) {
      ulonglong2 sum = all[k];
      for (int o = 1; o < kGroups; ++o) {
        const ulonglong2 p = all[o * 4 * G + k];
        sum.x = f2_add(sum.x, p.x);
        sum.y = f2_add(sum.y, p.y);
      }
      leave(ln_col<T, G, VEC>(k % G, v, 2 * (k / G)), ln_col<T, G, VEC>(k % G, v, 2 * (k / G) + 1), sum);
    }
  }
}

// The partial rows, summed in a fixed order: 32 columns per CTA, 32 lanes of rows.  Launched while the kernel above runs out
// (programmatic dependent launch): it waits for that one's partial rows before it reads them.
__global__ void __launch_bounds__(1024) ln_finish_kernel(const LnBwdArgs a) {
  __shared__ float sums[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float s = 0.f;
  if (c < 2 * a.cols) {
#pragma unroll 8
    for (int part = lane; part < a.parts; part += 32) s += a.partials[static_cast<long long>(part) * 2 * a.cols + c];
  }
  sums[lane][threadIdx.x & 31] = s;
  __syncthreads();
  // warp w adds up column w: lane l holds partial sum l
  const int col = blockIdx.x * 32 + lane;
  float t = sums[threadIdx.x & 31][lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if ((threadIdx.x & 31) == 0 && col < 2 * a.cols) {
    void* out = col < a.cols ? a.dweight : a.dbias;
    const int at = col < a.cols ? col : col - a.cols;
    if (out) {
      if (a.param_bf16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(t);
      else static_cast<float*>(out)[at] = t;
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

// CTAs of a kernel that the device holds at once, with the shared memory it asks for allowed first (without the attribute the
// limit counts static shared memory too); 0: that was refused.  Worked out once per device and kernel.
template <typename K>
static int ln_resident(PerDevice& cache, K kernel, int threads, uint32_t smem) {
  bool allowed = true;
  const int held = cache.get([&] {
    allowed = smem <= 32 * 1024 || cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) == cudaSuccess;
    return allowed ? held_at_once(kernel, threads, smem) : 0;
  });
  return held || !allowed ? held : sm_count();
}

// Rows ahead by what shared memory holds beside `table` bytes: two CTAs of 256 threads an SM, or one of 512.  Fewer than
// two: no ring.
template <typename T, int VPT, int THREADS>
constexpr int ln_stages(int table, int most) {
  const int stage = 2 * VPT * 8 * static_cast<int>(sizeof(T)) * THREADS, fit = ((THREADS == 512 ? 220 : 110) * 1024 - table) / stage;
  return fit > most ? most : fit < 2 ? 0 : fit;
}

template <typename T, int G, int VPT, bool DROP, int VEC>
static int run_ln_fwd(const LnFwdArgs& a, cudaStream_t stream) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G, kTable = 2 * VPT * 8 * G * 4;
  constexpr bool kHasTable = kTable + 2 * 2 * VPT * 8 * static_cast<int>(sizeof(T)) * kThreads <= (kThreads == 512 ? 220 : 110) * 1024;
  constexpr int kStages = VEC ? ln_stages<T, VPT, kThreads>(kHasTable ? kTable : 0, 2) : 0;
  if constexpr (kStages > 0) {
    // from four rows per group and SM on: 65536 x 768 takes 77 us with the ring, 102 without; 4096 x 768 stays below it
    if (a.rows >= 4LL * kGroups * sm_count()) {
      auto kernel = ln_fwd_ring_kernel<T, G, VPT, DROP, VEC, kStages, kHasTable>;
      constexpr uint32_t smem = LnRing<T, G, VPT, VEC, 2, kStages, kThreads>::kBytes + (kHasTable ? kTable : 0);
      static PerDevice resident;
      const long long most = ln_resident(resident, kernel, kThreads, smem), batches = (a.rows + kGroups - 1) / kGroups;
      if (most < 1) return cuda_fail(cudaGetLastError(), "cudaFuncSetAttribute");
      kernel<<<static_cast<unsigned>(batches < most ? batches : most), kThreads, smem, stream>>>(a);
      return HYC_OK;
    }
  }
  const unsigned grid = static_cast<unsigned>((a.rows + kGroups - 1) / kGroups);
  ln_fwd_kernel<T, G, VPT, DROP, VEC><<<grid, kThreads, 0, stream>>>(a);
  return HYC_OK;
}

template <typename T, int G, int VPT>
static int pick_ln_fwd_kind(const LnFwdArgs& a, bool vec, cudaStream_t stream) {
  if (!vec) return a.rng ? run_ln_fwd<T, G, VPT, true, 0>(a, stream) : run_ln_fwd<T, G, VPT, false, 0>(a, stream);
  if (a.cols != G * VPT * 8) return a.rng ? run_ln_fwd<T, G, VPT, true, 1>(a, stream) : run_ln_fwd<T, G, VPT, false, 1>(a, stream);
  return a.rng ? run_ln_fwd<T, G, VPT, true, 2>(a, stream) : run_ln_fwd<T, G, VPT, false, 2>(a, stream);
}

// threads per row and pieces per thread by the row's width: the smallest group that holds it in at most 32 elements per thread
template <typename T>
static int pick_ln_fwd(const LnFwdArgs& a, bool vec, cudaStream_t stream) {
  const int slots = (a.cols + 7) / 8;
  if (slots <= 32) return pick_ln_fwd_kind<T, 32, 1>(a, vec, stream);
  if (slots <= 64) return pick_ln_fwd_kind<T, 32, 2>(a, vec, stream);
  if (slots <= 96) return pick_ln_fwd_kind<T, 32, 3>(a, vec, stream);
  if (slots <= 128) return pick_ln_fwd_kind<T, 32, 4>(a, vec, stream);
  if (slots <= 256) return pick_ln_fwd_kind<T, 128, 2>(a, vec, stream);
  if (slots <= 512) return pick_ln_fwd_kind<T, 256, 2>(a, vec, stream);
  if (slots <= 768) return pick_ln_fwd_kind<T, 256, 3>(a, vec, stream);
  if (slots <= 1024) return pick_ln_fwd_kind<T, 512, 2>(a, vec, stream);
  if (slots <= 1536) return pick_ln_fwd_kind<T, 512, 3>(a, vec, stream);
  return pick_ln_fwd_kind<T, 512, 4>(a, vec, stream);
}

template <typename T>
static int launch_ln_fwd(const LnFwdArgs& a, cudaStream_t stream) {
  const uintptr_t es = sizeof(T);
  const bool vec = a.cols % 8 == 0 && rows_aligned(a.x, a.x_stride, es) && rows_aligned(a.residual, a.residual_stride, es) &&
                   aligned16(a.y) && aligned16(a.z) && aligned16(a.weight) && aligned16(a.bias);
  const int rc = pick_ln_fwd<T>(a, vec, stream);
  if (rc) return rc;
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "ln_fwd_kernel");
}

template <typename T, int G, int VPT, bool DROP, int VEC, bool SMEM>
static int run_ln_bwd(LnBwdArgs a, cudaStream_t stream) {
  constexpr int kThreads = G < 256 ? 256 : G, kGroups = kThreads / G;
  constexpr int kTable = VPT * 8 * G * 4, kStages = VEC && !SMEM ? ln_stages<T, VPT, kThreads>(kTable, 2) : 0;
  auto kernel = ln_bwd_kernel<T, G, VPT, DROP, VEC, SMEM, kStages>;
  constexpr uint32_t sums = SMEM ? kThreads * VPT * 8 * 8 : kGroups > 1 ? kThreads * 8 * 8 : 0;
  constexpr uint32_t ahead = kStages ? LnRing<T, G, VPT, VEC, 2, kStages ? kStages : 1, kThreads>::kBytes + kTable : 0;
  constexpr uint32_t smem = sums > ahead ? sums : ahead;
  static PerDevice resident;
  const long long most = ln_resident(resident, kernel, kThreads, smem), batches = (a.rows + kGroups - 1) / kGroups;
  if (most < 1) return cuda_fail(cudaGetLastError(), "cudaFuncSetAttribute");
  a.parts = static_cast<int>(batches < most ? batches : most);
  if (a.parts > kLnMaxParts) a.parts = kLnMaxParts;
  kernel<<<a.parts, kThreads, smem, stream>>>(a);
  HYC_LAUNCHED();
  if (a.partials) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((2 * a.cols + 31) / 32); cfg.blockDim = dim3(1024); cfg.stream = stream; cfg.attrs = &attr; cfg.numAttrs = 1;
    const cudaError_t f = cudaLaunchKernelEx(&cfg, ln_finish_kernel, a);
    HYC_LAUNCHED();
    if (f != cudaSuccess) {
      cudaGetLastError();                  // a refused launch is this call's error, not also the next one's
      return cuda_fail(f, "ln_finish_kernel");
    }
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "ln_bwd_kernel");
}

template <typename T, int G, int VPT, bool SMEM>
static int pick_ln_bwd_kind(const LnBwdArgs& a, bool vec, cudaStream_t stream) {
  if (!vec) return a.rng ? run_ln_bwd<T, G, VPT, true, 0, SMEM>(a, stream) : run_ln_bwd<T, G, VPT, false, 0, SMEM>(a, stream);
  if (a.cols != G * VPT * 8) return a.rng ? run_ln_bwd<T, G, VPT, true, 1, SMEM>(a, stream) : run_ln_bwd<T, G, VPT, false, 1, SMEM>(a, stream);
  return a.rng ? run_ln_bwd<T, G, VPT, true, 2, SMEM>(a, stream) : run_ln_bwd<T, G, VPT, false, 2, SMEM>(a, stream);
}

template <typename T>
static int pick_ln_bwd(const LnBwdArgs& a, bool vec, cudaStream_t stream) {
  const int slots = (a.cols + 7) / 8;
  if (slots <= 32) return pick_ln_bwd_kind<T, 32, 1, false>(a, vec, stream);
  if (slots <= 64) return pick_ln_bwd_kind<T, 32, 2, false>(a, vec, stream);
  if (slots <= 96) return pick_ln_bwd_kind<T, 32, 3, false>(a, vec, stream);
  if (slots <= 128) {
    // bf16: two warps of two slots (65536 x 1024 with dropout 106 us, 127 as four of one); fp32 the other way round (81 / 99)
    if constexpr (sizeof(T) == 2) return pick_ln_bwd_kind<T, 64, 2, false>(a, vec, stream);
    else return pick_ln_bwd_kind<T, 128, 1, false>(a, vec, stream);
  }
  if (slots <= 256) return pick_ln_bwd_kind<T, 128, 2, false>(a, vec, stream);
  if (slots <= 512) return pick_ln_bwd_kind<T, 256, 2, false>(a, vec, stream);
  if (slots <= 1024) return pick_ln_bwd_kind<T, 512, 2, false>(a, vec, stream);
  if (slots <= 1536) return pick_ln_bwd_kind<T, 512, 3, true>(a, vec, stream);
  return pick_ln_bwd_kind<T, 512, 4, true>(a, vec, stream);
}

template <typename T>
static int launch_ln_bwd(const LnBwdArgs& a, cudaStream_t stream) {
  const uintptr_t es = sizeof(T);
  const bool vec = a.cols % 8 == 0 && rows_aligned(a.dy, a.dy_stride, es) && rows_aligned(a.z, a.z_stride, es) &&
                   rows_aligned(a.dz, a.dz_stride, es) && aligned16(a.dresidual) && aligned16(a.dx) && aligned16(a.weight);
  return pick_ln_bwd<T>(a, vec, stream);
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
