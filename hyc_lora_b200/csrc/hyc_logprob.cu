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

// Order of the alternatives as one integer: larger value first (-0 counts as +0, a NaN stands above +inf), lower index first
// among equals.  0 stands for none.
__device__ __forceinline__ unsigned long long lp_key(float v, uint32_t index) {
  uint32_t b = __float_as_uint(v + 0.f);
  b = v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(b) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float lp_key_value(unsigned long long key) {
  const uint32_t b = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint32_t lp_key_index(unsigned long long key) { return 0xffffffffu - static_cast<uint32_t>(key); }

// largest of two, a NaN if there is one
__device__ __forceinline__ float lp_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float lp_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = lp_max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// 2^x to about 2^-22, results below the normal numbers as zero
__device__ __forceinline__ float lp_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- forward

// A row (or, in a cluster, a CTA's slice of one) is held in registers, kPer 16-byte pieces per thread, and read once.
//   1. its largest value (packed maxima), over the CTA;
//   2. the sums of e = exp(x - m) and e (x - m), with what equals m counted apart -- only the warps that hold it test for it;
//      each piece's register takes the next row's piece as soon as it is spent, so that loads run through the reductions;
//   3. alternatives: the k-th largest of 64 groups' maxima is a bound that the k best reach and hardly anything else does.
//      The few values that reach it are collected, and each counts those before it.  Where too many reach it (rows of equal
//      values, or hardly anything open), or the row holds a NaN, the best are picked one after the other instead.
// The CTAs of a cluster work on slices with their own m; the first one joins sums and alternatives through distributed shared
// memory, in rank order: no atomics on results, no workspace, one launch.
constexpr int kLpCandidates = 256, kLpGroups = 64;

__host__ __device__ constexpr int lp_per(int threads) { return threads > 512 ? 16 : 8; }

struct LpSums {
  float m, count, rest, te;     // largest, how often, sum of the other e, sum of e (x - m)
};

template <typename T>
__device__ __forceinline__ float lp_piece_max(const uint4& w);
template <>
__device__ __forceinline__ float lp_piece_max<__nv_bfloat16>(const uint4& w) {
  const __nv_bfloat162 a = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w.x), *reinterpret_cast<const __nv_bfloat162*>(&w.y));
  const __nv_bfloat162 b = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w.z), *reinterpret_cast<const __nv_bfloat162*>(&w.w));
  const __nv_bfloat162 c = __hmax2_nan(a, b);
  return lp_max(__low2float(c), __high2float(c));
}
template <>
__device__ __forceinline__ float lp_piece_max<float>(const uint4& w) {
  return lp_max(lp_max(__uint_as_float(w.x), __uint_as_float(w.y)), lp_max(__uint_as_float(w.z), __uint_as_float(w.w)));
}

template <typename T>
__device__ __forceinline__ void lp_unpack(const uint4& w, float (&f)[16 / sizeof(T)]);
template <>
__device__ __forceinline__ void lp_unpack<__nv_bfloat16>(const uint4& w, float (&f)[8]) { unpack_bf16x8(w, f); }
template <>
__device__ __forceinline__ void lp_unpack<float>(const uint4& w, float (&f)[4]) {
  f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
}

// where a CTA's slice of a row lies: pieces of 16 bytes counted from the aligned address at or below the row's start
struct LpRow {
  const unsigned char* base;   // 16-byte aligned
  int lead;                    // elements of the first piece that belong to what is before the row
  int first, pieces;           // this CTA's pieces
};

template <typename T>
__device__ __forceinline__ LpRow lp_row(const void* logits, long long offset, int vocab, int rank, int ranks) {
  const unsigned char* p = static_cast<const unsigned char*>(logits) + offset * static_cast<long long>(sizeof(T));
  LpRow r;
  const int phase = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15u);
  r.base = p - phase;
  r.lead = phase / static_cast<int>(sizeof(T));
  const int all = (r.lead + vocab + 16 / static_cast<int>(sizeof(T)) - 1) / (16 / static_cast<int>(sizeof(T)));
  const int each = (all + ranks - 1) / ranks;
  r.first = rank * each;
  r.pieces = min(each, all - r.first);      // may be <= 0
  return r;
}

// piece `i` of the slice; what lies outside the row is not read and counts as -inf
template <typename T>
__device__ __forceinline__ uint4 lp_fetch(const LpRow& r, int vocab, int i) {
  constexpr int kPiece = 16 / sizeof(T);
  const uint32_t shut = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  uint4 w = make_uint4(shut, shut, shut, shut);
  if (i >= r.pieces) return w;
  const int piece = r.first + i, e0 = piece * kPiece - r.lead;
  const unsigned char* p = r.base + static_cast<long long>(piece) * 16;
  if (e0 >= 0 && e0 + kPiece <= vocab) return load16_stream(p);
  // a row's ragged end: element by element, shifted in from above
#pragma unroll 1
  for (int e = 0; e < kPiece; ++e) {
    const bool in = e0 + e >= 0 && e0 + e < vocab;
    if (sizeof(T) == 2) {
      const uint32_t bits = in ? reinterpret_cast<const uint16_t*>(p)[e] : shut & 0xffffu;
      w.x = w.x >> 16 | w.y << 16;
      w.y = w.y >> 16 | w.z << 16;
      w.z = w.z >> 16 | w.w << 16;
      w.w = w.w >> 16 | bits << 16;
    } else {
      w.x = w.y; w.y = w.z; w.z = w.w;
      w.w = in ? reinterpret_cast<const uint32_t*>(p)[e] : shut;
    }
  }
  return w;
}

// sums of one piece; APART: values equal to m are counted instead
template <typename T, bool ENT, bool APART>
__device__ __forceinline__ void lp_piece_sums(const uint4& w, float m, f32x2& rest, f32x2& te, float& count) {
  constexpr int kPiece = 16 / sizeof(T);
  float f[kPiece];
  lp_unpack<T>(w, f);
  const f32x2 minus_m = f2_make(-m, -m), log2e = f2_make(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < kPiece / 2; ++i) {
    float x0 = f[2 * i], x1 = f[2 * i + 1];
    if (APART) {
      if (x0 == m) { count += 1.f; x0 = -INFINITY; }
      if (x1 == m) { count += 1.f; x1 = -INFINITY; }
    }
    f32x2 d = f2_add(f2_make(x0, x1), minus_m);
    if (ENT) {
      // e is 0 long before; a finite difference keeps 0 * d at 0 (and max.NaN keeps a NaN)
      float d0, d1;
      f2_split(d, d0, d1);
      d = f2_make(lp_max(d0, -10000.f), lp_max(d1, -10000.f));
    }
    float u0, u1;
    f2_split(f2_mul(d, log2e), u0, u1);
    const f32x2 e = f2_make(lp_exp2(u0), lp_exp2(u1));
    rest = f2_add(rest, e);
    if (ENT) te = f2_fma(e, d, te);
  }
}

// the best `top` of this CTA's slice one after the other, from memory (rare: see above); keys in descending order to `out`
template <typename T>
__device__ __noinline__ void lp_pick_slowly(const LpRow r, int vocab, int top, unsigned long long* best, unsigned long long* out) {
  constexpr int kPiece = 16 / sizeof(T);
  unsigned long long before = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long key = 0;
    for (int i = threadIdx.x; i < r.pieces; i += blockDim.x) {
      const uint4 w = lp_fetch<T>(r, vocab, i);
      float f[kPiece];
      lp_unpack<T>(w, f);
      const int e0 = (r.first + i) * kPiece - r.lead;
#pragma unroll
      for (int e = 0; e < kPiece; ++e) {
        if (e0 + e < 0 || e0 + e >= vocab) continue;
        const unsigned long long q = lp_key(f[e], e0 + e);
        if (q < before && q > key) key = q;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long q = __shfl_xor_sync(0xffffffffu, key, o);
      key = q > key ? q : key;
    }
    __syncthreads();                       // the previous turn's `best` has been read
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = key;
    __syncthreads();
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) key = best[w] > key ? best[w] : key;
    if (threadIdx.x == 0) out[k] = key;
    before = key;
  }
  __syncthreads();
}

template <int THREADS>
struct LpShared {
  float4 wmax4[2][8];                      // [parity][warps], as float
  LpSums part[2][32];                      // [parity][warp]
  float group[kLpGroups];
  float bound;
  int found;
  unsigned long long keys[kLpCandidates];
  unsigned long long picked[32];
  unsigned long long best[32];
  float2 result;                           // m, log S of the row (one CTA per row)
  LpSums slice[2][8];                      // [parity][rank], in the first CTA of a cluster
  unsigned long long slice_keys[2][8][32];
};

__device__ __forceinline__ LpSums lp_join(const LpSums* s, int n) {
  float m = s[0].m;
  for (int i = 1; i < n; ++i) m = lp_max(m, s[i].m);
  LpSums r = {m, 0.f, 0.f, 0.f};
  for (int i = 0; i < n; ++i) {
    if (s[i].m == -INFINITY) continue;     // nothing open there
    if (s[i].m == m) {
      r.count += s[i].count;
      r.rest += s[i].rest;
      r.te += s[i].te;
    } else {
      const float d = s[i].m - m, f = expf(d), sum = s[i].count + s[i].rest;
      r.rest += sum * f;
      r.te += f == 0.f ? 0.f : f * (s[i].te + d * sum);
    }
  }
  return r;
}

// one thread: the row's results from its sums; returns (m, log S) with log S NaN where the row has a NaN or +inf
__device__ __forceinline__ float2 lp_finish(const LogprobArgs& a, long long row, const LpSums& s, long long target, float at_target) {
  const bool none = s.m == -INFINITY;
  float logz = s.count == 1.f ? log1pf(s.rest) : logf(s.count + s.rest);
  if (none) logz = 0.f;
  if (!(s.m < INFINITY)) logz = NAN;
  *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(s.m, logz);
  if (a.entropy) a.entropy[row] = none ? 0.f : logz - s.te / (s.count + s.rest);
  if (a.targets) {
    float lp = NAN;                                                  // a target outside the vocabulary
    if (target == a.ignore_index) lp = 0.f;
    else if (target >= 0 && target < a.vocab) lp = none ? -INFINITY : at_target - s.m - logz;
    a.logprob[row] = lp;
  }
  return make_float2(s.m, logz);
}

__device__ __forceinline__ void lp_put_top(const LogprobArgs& a, long long row, int rank, unsigned long long key, float2 mz) {
  a.top_index[row * a.top + rank] = lp_key_index(key);
  a.top_logprob[row * a.top + rank] = mz.x == -INFINITY ? -INFINITY : lp_key_value(key) - mz.x - mz.y;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of `p` (this CTA's shared memory) in the shared memory of CTA 0 of the cluster
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}

template <typename T, int THREADS, bool ENT, bool TOP, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, THREADS > 512 ? 1 : 1024 / THREADS) logprob_kernel(const LogprobArgs a) {
  constexpr int kPiece = 16 / sizeof(T), kPer = lp_per(THREADS), kWarps = THREADS / 32;
  constexpr int kPerGroup = THREADS <= kLpGroups ? 1 : THREADS > 512 ? 16 : THREADS / kLpGroups;   // lanes of a group, a power of two
  __shared__ LpShared<THREADS> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = CLUSTER ? static_cast<int>(cluster_rank()) : 0, ranks = CLUSTER ? static_cast<int>(cluster_size()) : 1;
  const long long step = gridDim.x / ranks;
  if (TOP && threadIdx.x == 0) sh.found = 0;
  auto at = [&](long long row) {
    const long long batch = row / a.seq;
    return batch * a.batch_stride + (row - batch * a.seq) * a.row_stride;
  };
  // rows without a target of which nothing else is asked are not read
  auto next = [&](long long row) {
    if (!ENT && !TOP && a.targets) {
      while (row < a.rows && a.targets[row] == a.ignore_index) {
        if (rank == 0 && threadIdx.x == 0) {
          a.logprob[row] = 0.f;
          *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(-INFINITY, 0.f);
        }
        row += step;
      }
    }
    return row;
  };
  uint4 raw[kPer];
  long long row = next(blockIdx.x / ranks);
  LpRow r = {};
  long long target = -1;
  float at_target = 0.f;
  auto head = [&](long long to) {            // what the first thread needs of a row, beside its pieces
    if (a.targets && rank == 0 && threadIdx.x == 0) {
      target = a.targets[to];
      if (target >= 0 && target < a.vocab) at_target = lp_load(static_cast<const T*>(a.logits), at(to) + target);
    }
  };
  if (row < a.rows) {
    r = lp_row<T>(a.logits, at(row), a.vocab, rank, ranks);
#pragma unroll
    for (int i = 0; i < kPer; ++i) raw[i] = lp_fetch<T>(r, a.vocab, i * THREADS + threadIdx.x);
    head(row);
  }
  int turn = 0;
  while (row < a.rows) {
    // 1. the largest
    float mine = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine = lp_max(mine, lp_piece_max<T>(raw[i]));
    float wmax = mine;
    if (TOP && kPerGroup <= 16) {
#pragma unroll
      for (int o = 1; o < kPerGroup; o <<= 1) wmax = lp_max(wmax, __shfl_xor_sync(0xffffffffu, wmax, o));
      if (threadIdx.x % kPerGroup == 0 && threadIdx.x / kPerGroup < kLpGroups) sh.group[threadIdx.x / kPerGroup] = wmax;
#pragma unroll
      for (int o = kPerGroup; o < 32; o <<= 1) wmax = lp_max(wmax, __shfl_xor_sync(0xffffffffu, wmax, o));
    } else {
      wmax = lp_warp_max(wmax);
    }
    float m = wmax;
    float* all = reinterpret_cast<float*>(sh.wmax4[turn]);
    if (kWarps > 1 || TOP) {
      if (lane == 0) all[warp] = wmax;
      __syncthreads();
      if (kWarps > 1) m = lp_warp_max(lane < kWarps ? all[lane] : -INFINITY);
    }
    // the bound of the alternatives, by the first warps
    constexpr int kGroups = THREADS / kPerGroup < kLpGroups ? THREADS / kPerGroup : kLpGroups;
    if (TOP && threadIdx.x < kGroups) {
      const float v = sh.group[threadIdx.x];
      int before = 0;
#pragma unroll 8
      for (int j = 0; j < kGroups; ++j) {
        const float o = sh.group[j];
        before += o > v || (o == v && j < static_cast<int>(threadIdx.x));
      }
      if (before == a.top - 1) sh.bound = v;
    }
    // 2. the sums
    const float base = m == -INFINITY ? 0.f : m;
    f32x2 rest2 = 0, te2 = 0;
    LpSums s = {m, 0.f, 0.f, 0.f};
    const long long upcoming = next(row + step);
    const LpRow now = r;
    if (upcoming < a.rows) r = lp_row<T>(a.logits, at(upcoming), a.vocab, rank, ranks);
    if (wmax == m) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        lp_piece_sums<T, ENT, true>(raw[i], base, rest2, te2, s.count);
        if (!TOP && upcoming < a.rows) raw[i] = lp_fetch<T>(r, a.vocab, i * THREADS + threadIdx.x);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        lp_piece_sums<T, ENT, false>(raw[i], base, rest2, te2, s.count);
        if (!TOP && upcoming < a.rows) raw[i] = lp_fetch<T>(r, a.vocab, i * THREADS + threadIdx.x);
      }
    }
    float lo, hi;
    f2_split(rest2, lo, hi);
    s.rest = lo + hi;
    f2_split(te2, lo, hi);
    s.te = lo + hi;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s.count += __shfl_xor_sync(0xffffffffu, s.count, o);
      s.rest += __shfl_xor_sync(0xffffffffu, s.rest, o);
      if (ENT) s.te += __shfl_xor_sync(0xffffffffu, s.te, o);
    }
    if (kWarps > 1 || TOP) {
      if (lane == 0) sh.part[turn][warp] = s;
      __syncthreads();
    }
    if (warp == 0 && kWarps > 1) {
      s.count = s.rest = s.te = 0.f;
      if (lane < kWarps) s = sh.part[turn][lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        s.count += __shfl_xor_sync(0xffffffffu, s.count, o);
        s.rest += __shfl_xor_sync(0xffffffffu, s.rest, o);
        if (ENT) s.te += __shfl_xor_sync(0xffffffffu, s.te, o);
      }
    }
    if (!CLUSTER && threadIdx.x == 0) {
      const float2 mz = lp_finish(a, row, s, target, at_target);
      if (TOP) sh.result = mz;
    }
    if (CLUSTER && threadIdx.x == 0) {
      const uint32_t to = in_first_cta(&sh.slice[turn][rank]);
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(s.m), "f"(s.count), "f"(s.rest), "f"(s.te) : "memory");
    }
    // 3. the alternatives
    if (TOP) {
      const float bound = sh.bound;
      if (mine >= bound) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (!(lp_piece_max<T>(raw[i]) >= bound)) continue;
          if (i * THREADS + static_cast<int>(threadIdx.x) >= now.pieces) continue;
          uint4 w = raw[i];
          const int e0 = (now.first + i * THREADS + static_cast<int>(threadIdx.x)) * kPiece - now.lead;
#pragma unroll 1
          for (int e = 0; e < kPiece; ++e) {                     // few pieces come here: element by element, shifted out below
            const float v = sizeof(T) == 2 ? __uint_as_float(w.x << 16) : __uint_as_float(w.x);
            if (v >= bound && e0 + e >= 0 && e0 + e < a.vocab) {
              const int k = atomicAdd(&sh.found, 1);
              if (k < kLpCandidates) sh.keys[k] = lp_key(v, e0 + e);
            }
            if (sizeof(T) == 2) {
              w.x = w.x >> 16 | w.y << 16;
              w.y = w.y >> 16 | w.z << 16;
              w.z = w.z >> 16 | w.w << 16;
              w.w >>= 16;
            } else {
              w.x = w.y; w.y = w.z; w.z = w.w;
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (upcoming < a.rows) raw[i] = lp_fetch<T>(r, a.vocab, i * THREADS + threadIdx.x);
      __syncthreads();
      const int found = sh.found;
      const bool slowly = found > kLpCandidates || m != m;
      if (slowly) {
        lp_pick_slowly<T>(now, a.vocab, a.top, sh.best, sh.picked);
      } else {
        if (threadIdx.x < 32) sh.picked[threadIdx.x] = 0;
        __syncthreads();
        for (int c = threadIdx.x; c < found; c += THREADS) {
          const unsigned long long key = sh.keys[c];
          int before = 0;
          for (int j = 0; j < found; ++j) before += sh.keys[j] > key;
          if (before < a.top) sh.picked[before] = key;
        }
        __syncthreads();
      }
      if (threadIdx.x == 0) sh.found = 0;
      if (static_cast<int>(threadIdx.x) < a.top) {
        const unsigned long long key = sh.picked[threadIdx.x];
        if (!CLUSTER) {
          lp_put_top(a, row, threadIdx.x, key, sh.result);
        } else {
          const uint32_t to = in_first_cta(&sh.slice_keys[turn][rank][threadIdx.x]);
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(key) : "memory");
        }
      }
    }
    if (CLUSTER) {
      // The first CTA reads row n's slices behind this barrier; the others write the same place again two rows on, behind the
      // barrier of the row between, at which the first CTA arrives only when it is done reading.
      __syncwarp();
      cluster_barrier();
      if (rank == 0) {
        if (!TOP) {
          if (threadIdx.x == 0) lp_finish(a, row, lp_join(sh.slice[turn], ranks), target, at_target);
        } else {
          if (threadIdx.x == 0) sh.result = lp_finish(a, row, lp_join(sh.slice[turn], ranks), target, at_target);
          __syncthreads();
          const float2 mz = sh.result;
          for (int c = threadIdx.x; c < ranks * a.top; c += THREADS) {
            const unsigned long long key = sh.slice_keys[turn][c / a.top][c % a.top];
            if (key == 0) continue;
            int before = 0;
            for (int q = 0; q < ranks; ++q)
              for (int j = 0; j < a.top; ++j) before += sh.slice_keys[turn][q][j] > key;
            if (before < a.top) lp_put_top(a, row, before, key, mz);
          }
        }
      }
    }
    if (upcoming < a.rows) head(upcoming);
    row = upcoming;
    turn ^= 1;
  }
  __syncwarp();
  if (CLUSTER) cluster_barrier();          // nobody leaves while the first CTA's shared memory may still be written
}

// ---------------------------------------------------------------- backward

// Elementwise over the logits with five numbers per row: a CTA (or, for short rows, a warp) takes a run of pieces of one row,
// kLpPieces per thread.  What arrives for single tokens is put right afterwards by the threads that hold those few, after a
// barrier that orders their stores behind the run's.
constexpr int kLpPieces = 4;

template <typename T>
__device__ __forceinline__ void lp_store_piece(void* p, const float (&f)[16 / sizeof(T)]);
template <>
__device__ __forceinline__ void lp_store_piece<__nv_bfloat16>(void* p, const float (&f)[8]) { *static_cast<uint4*>(p) = pack_bf16x8(f); }
template <>
__device__ __forceinline__ void lp_store_piece<float>(void* p, const float (&f)[4]) {
  *static_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
}

struct LpGrad {
  float m, logz, whole, dh, h;
  bool ent, none;
  // the gradient of a token for which nothing arrives on its own
  __device__ __forceinline__ float of(float x) const {
    const float lp = (x - m) - logz, p = lp_exp2(lp * kLog2e);
    const float g = -whole * p;
    return ent ? (p == 0.f ? g : g - dh * p * (lp + h)) : g;
  }
  // ... and of one for which `share` does
  __device__ __forceinline__ float of(float x, float share) const {
    const float lp = (x - m) - logz, p = expf(lp);
    const float g = (share - whole) * p - share * expm1f(lp);
    return ent && p != 0.f ? g - dh * p * (lp + h) : g;
  }
};

// WARP: a warp takes whole rows (they are at most 32 * kLpPieces pieces and a ragged end); else gridDim covers rows * runs.
template <typename T, bool WARP>
__global__ void __launch_bounds__(256) logprob_bwd_kernel(const LogprobBwdArgs a, int runs) {
  constexpr int kPiece = 16 / sizeof(T), kWidth = WARP ? 32 : 256;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const long long total = a.rows * runs, step = static_cast<long long>(gridDim.x) * (WARP ? 8 : 1);
  for (long long work = WARP ? static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x; work < total; work += step) {
    const long long row = WARP ? work : work / runs;
    const int run = WARP ? 0 : static_cast<int>(work - row * runs);
    const long long batch = row / a.seq;
    const T* x = static_cast<const T*>(a.logits) + batch * a.batch_stride + (row - batch * a.seq) * a.row_stride;
    T* out = static_cast<T*>(a.grad) + row * a.vocab;
    // the row's numbers; what arrives for the alternatives, one per lane
    const float2 st = *reinterpret_cast<const float2*>(a.stats + 2 * row);
    LpGrad g = {st.x, st.y, 0.f, 0.f, 0.f, a.d_entropy != nullptr, st.x == -INFINITY};
    if (a.d_entropy) { g.dh = a.d_entropy[row]; g.h = a.entropy[row]; }
    long long target = -1;
    float dt = 0.f;
    if (a.d_logprob) {
      target = a.targets[row];
      if (target == a.ignore_index) {
        target = -1;
      } else {
        dt = target >= 0 && target < a.vocab ? a.d_logprob[row] : NAN;
      }
    }
    const int lane = threadIdx.x & 31;
    float dk = 0.f;
    long long index = -1;
    if (lane < a.top) { dk = a.d_top[row * a.top + lane]; index = a.top_index[row * a.top + lane]; }
    g.whole = dk;
    if (a.top) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) g.whole += __shfl_xor_sync(0xffffffffu, g.whole, o);
    }
    g.whole += dt;
    const bool zero = g.none || (g.whole == 0.f && !a.top && !g.ent);        // nothing to read
    const float fill = g.whole == g.whole ? 0.f : NAN;
    // pieces counted from the aligned address at or below the row's start, if x and out lie alike
    const int phase = static_cast<int>(reinterpret_cast<uintptr_t>(out) & 15u), lead = phase / static_cast<int>(sizeof(T));
    const bool alike = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15u) == phase;
    const int pieces = (lead + a.vocab + kPiece - 1) / kPiece;
    const int first = run * (kWidth * kLpPieces), last = min(pieces, WARP ? pieces : first + kWidth * kLpPieces);
    for (int p0 = first; p0 < last; p0 += kWidth * kLpPieces) {
      uint4 raw[kLpPieces];
#pragma unroll
      for (int i = 0; i < kLpPieces; ++i) {
        const int piece = p0 + i * kWidth + t, e0 = piece * kPiece - lead;
        if (piece < last && alike && !zero && e0 >= 0 && e0 + kPiece <= a.vocab) raw[i] = load16_stream(x + e0);
      }
#pragma unroll
      for (int i = 0; i < kLpPieces; ++i) {
        const int piece = p0 + i * kWidth + t, e0 = piece * kPiece - lead;
        if (piece >= last) continue;
        if (e0 >= 0 && e0 + kPiece <= a.vocab) {
          float f[kPiece];
          if (zero) {
#pragma unroll
            for (int e = 0; e < kPiece; ++e) f[e] = fill;
          } else {
            if (alike) {
              lp_unpack<T>(raw[i], f);
            } else {
#pragma unroll
              for (int e = 0; e < kPiece; ++e) f[e] = lp_load(x, e0 + e);
            }
            const long long hot = target - e0;
            const bool has = !a.top && hot >= 0 && hot < kPiece;
            float there = 0.f;
            if (has) {
#pragma unroll
              for (int e = 0; e < kPiece; ++e) there = e == static_cast<int>(hot) ? f[e] : there;
              there = g.of(there, dt);
            }
#pragma unroll
            for (int e = 0; e < kPiece; ++e) f[e] = g.of(f[e]);
            if (has) {
#pragma unroll
              for (int e = 0; e < kPiece; ++e) f[e] = e == static_cast<int>(hot) ? there : f[e];
            }
          }
          lp_store_piece<T>(out + e0, f);
        } else {
#pragma unroll
          for (int e = 0; e < kPiece; ++e) {
            const int c = e0 + e;
            if (c < 0 || c >= a.vocab) continue;
            out[c] = T(zero ? fill : c == target && !a.top ? g.of(lp_load(x, c), dt) : g.of(lp_load(x, c)));
          }
        }
      }
    }
    if (a.top && !zero) {
      // the tokens for which something arrives: the alternatives, and the target behind them, one per lane and each by its
      // first mention; every warp of a CTA knows them, the first one writes those of the CTA's run
      if (WARP) __syncwarp();
      else __syncthreads();
      if (WARP || threadIdx.x < 32) {
        const int from = first * kPiece - lead, to = last * kPiece - lead;
        float share = 0.f, target_share = dt;
        bool seen = false, target_seen = false;
        for (int j = 0; j < a.top; ++j) {
          const long long o = __shfl_sync(0xffffffffu, index, j);
          const float d = __shfl_sync(0xffffffffu, dk, j);
          if (o == index) { share += d; seen |= j < lane; }
          if (o == target) { target_share += d; target_seen = true; }
        }
        if (index == target) share += dt;
        if (lane < a.top && !seen && index >= 0 && index < a.vocab && index >= from && index < to)
          out[index] = T(g.of(lp_load(x, index), share));
        if (lane == 0 && !target_seen && target >= 0 && target < a.vocab && target >= from && target < to)
          out[target] = T(g.of(lp_load(x, target), target_share));
      }
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

// clusters of `ranks` CTAs that the device holds at once
template <typename K>
static int resident_clusters(K kernel, int threads, int ranks) {
  if (ranks == 1) return resident_grid(kernel, threads, 0, 1 << 20);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(ranks); cfg.blockDim = dim3(threads); cfg.attrs = &attr; cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return sm_count() / ranks;
  }
  return n;
}

template <typename T, int THREADS, bool ENT, bool TOP, bool CLUSTER>
static int run_logprob(const LogprobArgs& a, int ranks, cudaStream_t stream) {
  auto kernel = logprob_kernel<T, THREADS, ENT, TOP, CLUSTER>;
  static PerDevice resident[4];            // by cluster size
  const long long most = resident[ranks == 8 ? 3 : ranks >> 1].get([&] { return resident_clusters(kernel, THREADS, ranks); }), clusters = a.rows < most ? a.rows : most;
  cudaError_t e;
  if (CLUSTER) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ranks; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * ranks)); cfg.blockDim = dim3(THREADS); cfg.stream = stream;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, a);
  } else {
    kernel<<<static_cast<unsigned>(clusters), THREADS, 0, stream>>>(a);
    e = cudaGetLastError();
  }
  HYC_LAUNCHED();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "logprob_kernel");
}

template <typename T, int THREADS, bool CLUSTER>
static int pick_logprob(const LogprobArgs& a, int ranks, cudaStream_t stream) {
  if (a.top) return a.entropy ? run_logprob<T, THREADS, true, true, CLUSTER>(a, ranks, stream) : run_logprob<T, THREADS, false, true, CLUSTER>(a, ranks, stream);
  return a.entropy ? run_logprob<T, THREADS, true, false, CLUSTER>(a, ranks, stream) : run_logprob<T, THREADS, false, false, CLUSTER>(a, ranks, stream);
}

// The smallest CTA, then the smallest cluster, whose registers hold a row (one piece more than its bytes, where it starts
// inside a piece).
template <typename T>
static int launch_logprob(const LogprobArgs& a, cudaStream_t stream) {
  const int pieces = static_cast<int>((static_cast<long long>(a.vocab) * sizeof(T) + 15) / 16) + 1;
  if (pieces <= 32 * 8) return pick_logprob<T, 32, false>(a, 1, stream);
  if (pieces <= 64 * 8) return pick_logprob<T, 64, false>(a, 1, stream);
  if (pieces <= 128 * 8) return pick_logprob<T, 128, false>(a, 1, stream);
  if (pieces <= 256 * 8) return pick_logprob<T, 256, false>(a, 1, stream);
  if (pieces <= 512 * 8) return pick_logprob<T, 512, false>(a, 1, stream);
  for (int ranks = 2; ranks <= 8; ranks *= 2)
    if (pieces <= ranks * 512 * 8) return pick_logprob<T, 512, true>(a, ranks, stream);
  return pick_logprob<T, 576, true>(a, 8, stream);
}

template <typename T>
static int launch_logprob_bwd(const LogprobBwdArgs& a, cudaStream_t stream) {
  const long long pieces = (static_cast<long long>(a.vocab) * sizeof(T) + 15) / 16 + 1;
  if (pieces <= 2 * 32 * kLpPieces) {
    const long long blocks = (a.rows + 7) / 8;
    logprob_bwd_kernel<T, true><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a, 1);
  } else {
    const int runs = static_cast<int>((pieces + 256 * kLpPieces - 1) / (256 * kLpPieces));
    const long long total = a.rows * runs;
    logprob_bwd_kernel<T, false><<<static_cast<unsigned>(total < 0x7fffffffLL ? total : 0x7fffffffLL), 256, 0, stream>>>(a, runs);
  }
  HYC_LAUNCHED();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HYC_OK : cuda_fail(e, "logprob_bwd_kernel");
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
  return q->dtype == HYC_BF16 ? launch_logprob<__nv_bfloat16>(a, stream) : launch_logprob<float>(a, stream);
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
  return q->dtype == HYC_BF16 ? launch_logprob_bwd<__nv_bfloat16>(a, stream) : launch_logprob_bwd<float>(a, stream);
}

}  // extern "C"
