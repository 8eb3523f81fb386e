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
  long long row_stride, batch_stride;
  int rows, seq, vocab, top;               // seq >= rows: one stride
  const long long* targets;
  long long ignore_index;
  float *logprob, *entropy, *stats, *top_logprob;
  long long* top_index;
};

struct LogprobBwdArgs {
  const void* logits;
  long long row_stride, batch_stride;
  int rows, seq, vocab, top;
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
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// 2^x to about 2^-22, results below the normal numbers as zero
__device__ __forceinline__ float lp_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- forward

// Persistent CTAs, a row at a time; a row is streamed once, in chunks of kLpChunk 16-byte pieces per thread, the next chunk (of
// this row or the next) in flight while one is worked on.  Within a row the warps go their own ways:
//   1. a warp keeps a largest value m of what it has seen, and the sums of e = exp(x - m) and e (x - m), with what equals m
//      counted apart.  A chunk whose own largest is below m is summed as it stands; else the sums so far are scaled to the new
//      m, and the values of the pieces that hold it are tested for it.  At the row's end the warps' sums are joined.
//   2. alternatives: every thread also knows the largest value it has seen.  The k-th largest of 64 groups' maxima is a bound
//      that the k best reach and hardly anything else does; the few threads that have seen something that reaches it have
//      their pieces read again (from L2) by their warp, what reaches the bound is collected, and each counts those before it.
//      Where too many reach it (equal values; fewer open tokens than alternatives), what stands above the bound is collected
//      and the first of its equals in index order with it; where the row holds a NaN, the best are picked one after the other.
// Few long rows are split over the CTAs of a cluster, which work on slices with their own m; the first one joins sums and
// alternatives through distributed shared memory, in rank order: no atomics on results, no workspace, one launch.
//
// Issue slots are as scarce as bytes here: bf16 leaves 11 of them per 32 elements at full bandwidth, and the exponentials take
// 8 of their unit's cycles.  Holding whole rows in registers instead, with a barrier behind the maximum and one behind the
// sums, took 122 us at 8192 x 32000 (512 threads of 8 pieces) or 186 (256 of 16), staging them in shared memory 151; this takes 104
// with 256 threads per row and 91 with 64 (see lp_threads).  With 256, chunks of 2 pieces take 107, of 6 113; two buffers that
// change places instead of a copy 114 (spills).
constexpr int kLpCandidates = 256, kLpGroups = 64, kLpChunk = 4;

struct alignas(16) LpSums {        // stored by 16 bytes into another CTA's shared memory
  float m, count, rest, te;     // largest, how often, sum of the other e, sum of e (x - m)
};

// elements between the first row's start and this one's
template <typename A>
__device__ __forceinline__ long long lp_offset(const A& a, int row) {
  if (a.seq >= a.rows) return row * a.row_stride;
  const unsigned batch = static_cast<unsigned>(row) / static_cast<unsigned>(a.seq);
  return batch * a.batch_stride + (row - static_cast<int>(batch) * a.seq) * a.row_stride;
}

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
  int first, pieces;           // this CTA's pieces; may be <= 0
  int from, whole;             // of those, [from, from + whole) lie wholly inside the row
};

template <typename T>
__device__ __forceinline__ LpRow lp_row(const void* logits, long long offset, int vocab, int rank, int ranks) {
  constexpr int kPiece = 16 / sizeof(T);
  const unsigned char* p = static_cast<const unsigned char*>(logits) + offset * static_cast<long long>(sizeof(T));
  LpRow r;
  const int phase = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15u);
  r.base = p - phase;
  r.lead = phase / static_cast<int>(sizeof(T));
  const int all = (r.lead + vocab + kPiece - 1) / kPiece;
  r.first = 0;
  r.pieces = all;
  if (ranks > 1) {
    const int each = (all + ranks - 1) / ranks;
    r.first = rank * each;
    r.pieces = min(each, all - r.first);
  }
  const int begin = r.lead ? 1 : 0, end = (r.lead + vocab) / kPiece;
  r.from = max(begin - r.first, 0);
  r.whole = max(min(end - r.first, r.pieces) - r.from, 0);
  return r;
}

// piece `i` of the slice, a ragged end of the row: element by element, shifted in from above; -inf outside the row
template <typename T>
__device__ __forceinline__ uint4 lp_ragged(const LpRow& r, int vocab, int i) {
  constexpr int kPiece = 16 / sizeof(T);
  const uint32_t shut = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  uint4 w = make_uint4(shut, shut, shut, shut);
  const int piece = r.first + i, e0 = piece * kPiece - r.lead;
  const unsigned char* p = r.base + static_cast<long long>(piece) * 16;
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

// piece `i` of the slice; what lies outside the row is not read and counts as -inf
template <typename T>
__device__ __forceinline__ uint4 lp_fetch(const LpRow& r, int vocab, int i) {
  if (static_cast<unsigned>(i - r.from) < static_cast<unsigned>(r.whole))
    return load16_stream(r.base + static_cast<long long>(r.first + i) * 16);
  if (i < r.pieces && i >= 0) return lp_ragged<T>(r, vocab, i);
  const uint32_t shut = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  return make_uint4(shut, shut, shut, shut);
}

// A thread's pieces t, t + THREADS, ...: chunk k is those of the sweeps 4 k .. 4 k + 3.  Chunks of whole pieces cost their
// loads and a uniform branch.
template <typename T, int THREADS>
struct LpSweep {
  LpRow r;
  const unsigned char* own;    // the thread's piece of sweep 0
  int begin, plain;            // chunks [begin, plain) are whole
  int chunks;
  __device__ __forceinline__ void start(const void* logits, long long offset, int vocab, int rank, int ranks) {
    r = lp_row<T>(logits, offset, vocab, rank, ranks);
    own = r.base + (static_cast<long long>(r.first) + threadIdx.x) * 16;
    begin = r.from > 0 ? 1 : 0;
    plain = (r.from + r.whole) / (THREADS * kLpChunk);
    chunks = r.pieces > 0 ? (r.pieces + THREADS * kLpChunk - 1) / (THREADS * kLpChunk) : 0;
  }
  __device__ __forceinline__ void load(int k, int vocab, uint4 (&w)[kLpChunk]) const {
    if (k >= begin && k < plain) {
      const unsigned char* p = own + static_cast<long long>(k) * (THREADS * kLpChunk * 16);
#pragma unroll
      for (int i = 0; i < kLpChunk; ++i) w[i] = load16_stream(p + i * (THREADS * 16));
    } else {
#pragma unroll
      for (int i = 0; i < kLpChunk; ++i) w[i] = lp_fetch<T>(r, vocab, (k * kLpChunk + i) * THREADS + static_cast<int>(threadIdx.x));
    }
  }
};

// Sums of one piece in base 2: with L = log2 e in fp32 and c = -m L rounded, u = x L + c in one rounding, e = 2^u; what c lost
// to its rounding is a common factor that the sums are given at the end (lp_lost).  APART: values equal to m are
// counted instead.
template <typename T, bool ENT, bool APART>
__device__ __forceinline__ void lp_piece_sums(const uint4& w, float m, f32x2 c, f32x2& rest, f32x2& te, float& count) {
  constexpr int kPiece = 16 / sizeof(T);
  float f[kPiece];
  lp_unpack<T>(w, f);
  const f32x2 log2e = f2_make(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < kPiece / 2; ++i) {
    float x0 = f[2 * i], x1 = f[2 * i + 1];
    if (APART) {
      if (x0 == m) { count += 1.f; x0 = -INFINITY; }
      if (x1 == m) { count += 1.f; x1 = -INFINITY; }
    }
    f32x2 u = f2_fma(f2_make(x0, x1), log2e, c);
    float u0, u1;
    f2_split(u, u0, u1);
    if (ENT) {
      // e is 0 long before; a finite u keeps 0 * u at 0 (and max.NaN keeps a NaN)
      u0 = lp_max(u0, -10000.f);
      u1 = lp_max(u1, -10000.f);
      u = f2_make(u0, u1);
    }
    const f32x2 e = f2_make(lp_exp2(u0), lp_exp2(u1));
    rest = f2_add(rest, e);
    if (ENT) te = f2_fma(e, u, te);
  }
}

// The same for an m so far from zero that c would lose too much: from the differences themselves, c = 0.
template <typename T>
__device__ __forceinline__ void lp_piece_sums_far(const uint4& w, float m, f32x2& rest, f32x2& te, float& count) {
  constexpr int kPiece = 16 / sizeof(T);
  float f[kPiece], r = 0.f, t = 0.f;
  lp_unpack<T>(w, f);
#pragma unroll 1
  for (int i = 0; i < kPiece; ++i) {
    float x = f[0];
#pragma unroll
    for (int e = 1; e < kPiece; ++e) x = e == i ? f[e] : x;
    if (x == m) {
      count += 1.f;
    } else {
      const float u = lp_max((x - m) * kLog2e, -10000.f), e = lp_exp2(u);
      r += e;
      t = fmaf(e, u, t);
    }
  }
  rest = f2_add(rest, f2_make(r, 0.f));
  te = f2_add(te, f2_make(t, 0.f));
}

// what c = -m L has lost to its rounding: exact
__device__ __forceinline__ float lp_lost(float m, float c, bool far) { return far ? 0.f : fmaf(-m, kLog2e, -c); }

// the best `top` of this CTA's slice one after the other, from memory (rare: see above); keys in descending order to `out`
template <typename T>
__device__ __noinline__ void lp_pick_slowly(const LpRow r, int vocab, int top, unsigned long long* best, unsigned long long* out) {
  constexpr int kPiece = 16 / sizeof(T);
  unsigned long long before = 0;            // the last turn's; the first has no upper bound (a NaN at index 0 has the largest key)
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
        if ((k == 0 || q < before) && q > key) key = q;
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

struct LpShared {
  LpSums part[2][8];                       // [parity][warp]
  int ties[8];                             // [warp]
  float4 group[kLpGroups / 4];
  int found;
  unsigned long long keys[kLpCandidates];
  unsigned long long picked[32];
  unsigned long long best[8];
  float2 result;                           // m, log S of the row
  LpSums slice[2][8];                      // [parity][rank], in the first CTA of a cluster
  unsigned long long slice_keys[2][8][32];
};

// Candidates of a row in which very many equal the bound: all that is above it, and as many of its equals, lowest index first,
// as are still wanted.  Returns how many there are (more than kLpCandidates: too many above).  All threads of the CTA.
template <typename T, int THREADS>
__device__ __noinline__ int lp_collect_ties(const LpRow r, int vocab, int top, float bound, LpShared* sh) {
  constexpr int kPiece = 16 / sizeof(T);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (threadIdx.x == 0) sh->found = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < r.pieces; i += THREADS) {
    const uint4 w = lp_fetch<T>(r, vocab, i);
    if (!(lp_piece_max<T>(w) > bound)) continue;
    float f[kPiece];
    lp_unpack<T>(w, f);
    const int e0 = (r.first + i) * kPiece - r.lead;
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
      if (!(f[e] > bound)) continue;                               // beyond the row: -inf, above nothing
      const int at = atomicAdd(&sh->found, 1);
      if (at < kLpCandidates) sh->keys[at] = lp_key(f[e], e0 + e);
    }
  }
  __syncthreads();
  int wanted = top - sh->found;
  if (wanted > 0 && sh->found + wanted > kLpCandidates) return kLpCandidates + 1;
  for (int first = 0; first < r.pieces && wanted > 0; first += THREADS) {
    const int i = first + threadIdx.x;
    const uint4 w = lp_fetch<T>(r, vocab, i);
    float f[kPiece];
    lp_unpack<T>(w, f);
    const int e0 = (r.first + i) * kPiece - r.lead;
    uint32_t equal = 0;
#pragma unroll
    for (int e = 0; e < kPiece; ++e) equal |= i < r.pieces && f[e] == bound && e0 + e >= 0 && e0 + e < vocab ? 1u << e : 0u;
    int before = __popc(equal);                                    // inclusive over the lanes, then over the warps
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int lower = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += lower;
    }
    if (lane == 31) sh->ties[warp] = before;
    before -= __popc(equal);
    __syncthreads();
    int all = 0;
    for (int v = 0; v < THREADS / 32; ++v) {
      if (v == warp) before += all;
      all += sh->ties[v];
    }
    for (; equal && before < wanted; equal &= equal - 1, ++before) sh->keys[atomicAdd(&sh->found, 1)] = lp_key(bound, e0 + __ffs(equal) - 1);
    wanted -= all;
    __syncthreads();
  }
  return sh->found;
}

// sums of up to eight parts, one per lane; complete in the first eight lanes
__device__ __forceinline__ LpSums lp_join(LpSums s, bool have) {
  if (!have) s.m = -INFINITY;
  const float m = lp_warp_max(s.m);
  LpSums r = {m, 0.f, 0.f, 0.f};
  if (s.m == -INFINITY) {
    // nothing open there
  } else if (s.m == m) {
    r = s;
  } else {
    const float d = s.m - m, f = expf(d), sum = s.count + s.rest;
    r.rest = sum * f;
    r.te = f == 0.f ? 0.f : f * (s.te + d * sum);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    r.count += __shfl_xor_sync(0xffffffffu, r.count, o);
    r.rest += __shfl_xor_sync(0xffffffffu, r.rest, o);
    r.te += __shfl_xor_sync(0xffffffffu, r.te, o);
  }
  return r;
}

// one thread: the row's results from its sums; returns (m, log S) with log S NaN where the row has a NaN or +inf
__device__ __forceinline__ float2 lp_finish(const LogprobArgs& a, int row, const LpSums& s, long long target, float at_target) {
  const bool none = s.m == -INFINITY;
  float logz = s.count == 1.f ? log1pf(s.rest) : logf(s.count + s.rest);
  if (none) logz = 0.f;
  if (!(s.m < INFINITY)) logz = NAN;
  *reinterpret_cast<float2*>(a.stats + 2LL * row) = make_float2(s.m, logz);
  if (a.entropy) a.entropy[row] = none ? 0.f : logz - s.te / (s.count + s.rest);
  if (a.targets) {
    float lp = NAN;                                                  // a target outside the vocabulary
    if (target == a.ignore_index) lp = 0.f;
    else if (target >= 0 && target < a.vocab) lp = none ? -INFINITY : at_target - s.m - logz;
    a.logprob[row] = lp;
  }
  return make_float2(s.m, logz);
}

__device__ __forceinline__ void lp_put_top(const LogprobArgs& a, int row, int rank, unsigned long long key, float2 mz) {
  a.top_index[static_cast<long long>(row) * a.top + rank] = lp_key_index(key);
  a.top_logprob[static_cast<long long>(row) * a.top + rank] = mz.x == -INFINITY ? -INFINITY : lp_key_value(key) - mz.x - mz.y;
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
// the two halves of a barrier that passes no data on
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// address of `p` (this CTA's shared memory) in the shared memory of CTA 0 of the cluster
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}

// a warp's running sums (per lane) over the chunks of a row
template <typename T, bool ENT>
struct LpRunning {
  float m, c, count;             // m and c = -m log2(e) of the warp
  f32x2 rest, te;
  bool far;                      // |m| of 2^20 or more, where c would lose over a tenth to its rounding

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    c = count = 0.f;
    rest = te = 0;
    far = true;
  }
  // the sums so far, taken to a larger m: out of the old frame (what c lost, what equalled m), down by the difference, into the new
  __device__ __forceinline__ void raise(float largest) {
    const float old_m = m, lost = lp_lost(m, c, far);
    m = lp_max(m, largest);
    far = !(fabsf(m) < 1048576.f);
    c = far ? 0.f : -m * kLog2e;
    float r0, r1, t0, t1;
    f2_split(rest, r0, r1);
    f2_split(te, t0, t1);
    const float down = (old_m - m) * kLog2e;
    if (old_m == -INFINITY || !(down > -300.f)) {
      r0 = r1 = t0 = t1 = 0.f;
    } else {
      const float out = lp_exp2(lost), f = lp_exp2(down), now = lp_lost(m, c, far), in = lp_exp2(-now);
      t0 = (t0 + lost * r0) * out;
      t1 = (t1 + lost * r1) * out;
      r0 = r0 * out + count;
      r1 *= out;
      t0 = f * (t0 + down * r0);
      t1 = f * (t1 + down * r1);
      r0 *= f;
      r1 *= f;
      t0 = in * (t0 - now * r0);
      t1 = in * (t1 - now * r1);
      r0 *= in;
      r1 *= in;
    }
    rest = f2_make(r0, r1);
    te = f2_make(t0, t1);
    count = 0.f;
  }
  // a chunk, the thread's largest value of each piece and the warp's of all
  __device__ __forceinline__ void add(const uint4 (&w)[kLpChunk], const float (&most)[kLpChunk], float largest) {
    const bool above = !(largest < m);                   // or a NaN
    if (above && largest != m) raise(largest);
    if (far) {
      if (m == -INFINITY) return;                        // nothing open yet
#pragma unroll
      for (int i = 0; i < kLpChunk; ++i) lp_piece_sums_far<T>(w[i], m, rest, te, count);
      return;
    }
    const f32x2 c2 = f2_make(c, c);
    if (above) {
#pragma unroll
      for (int i = 0; i < kLpChunk; ++i) {
        if (__any_sync(0xffffffffu, !(most[i] < m))) lp_piece_sums<T, ENT, true>(w[i], m, c2, rest, te, count);
        else lp_piece_sums<T, ENT, false>(w[i], m, c2, rest, te, count);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLpChunk; ++i) lp_piece_sums<T, ENT, false>(w[i], m, c2, rest, te, count);
    }
  }
  __device__ __forceinline__ LpSums warp_sums() const {
    float lo, hi;
    LpSums s = {m, count, 0.f, 0.f};
    f2_split(rest, lo, hi);
    s.rest = lo + hi;
    f2_split(te, lo, hi);
    s.te = lo + hi;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s.count += __shfl_xor_sync(0xffffffffu, s.count, o);
      s.rest += __shfl_xor_sync(0xffffffffu, s.rest, o);
      if (ENT) s.te += __shfl_xor_sync(0xffffffffu, s.te, o);
    }
    const float lost = lp_lost(m, c, far), out = exp2f(lost);
    s.te = (s.te + lost * s.rest) * out * 0.6931471805599453f;
    s.rest *= out;
    return s;
  }
};

template <typename T, int THREADS, bool ENT, bool TOP, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 768 / THREADS > 24 ? 24 : 768 / THREADS) logprob_kernel(const LogprobArgs a) {
  constexpr int kPiece = 16 / sizeof(T), kWarps = THREADS / 32;
  constexpr int kPerGroup = THREADS <= kLpGroups ? 1 : THREADS / kLpGroups, kGroups = THREADS / kPerGroup;   // lanes of a group: 1, 2 or 4
  __shared__ LpShared sh;
  if (CLUSTER) cluster_arrive();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = CLUSTER ? static_cast<int>(cluster_rank()) : 0, ranks = CLUSTER ? static_cast<int>(cluster_size()) : 1;
  const int step = static_cast<int>(gridDim.x) / ranks;
  // rows without a target of which nothing else is asked are not read
  auto next = [&](int row) {
    if (!ENT && !TOP && a.targets) {
      while (row < a.rows && a.targets[row] == a.ignore_index) {
        if (rank == 0 && threadIdx.x == 0) {
          a.logprob[row] = 0.f;
          *reinterpret_cast<float2*>(a.stats + 2LL * row) = make_float2(-INFINITY, 0.f);
        }
        if (row >= a.rows - step) return a.rows;
        row += step;
      }
    }
    return row;
  };
  int row = next(static_cast<int>(blockIdx.x) / ranks);
  LpSweep<T, THREADS> sweep;
  uint4 cur[kLpChunk];
  if (row < a.rows) {
    sweep.start(a.logits, lp_offset(a, row), a.vocab, rank, ranks);
    sweep.load(0, a.vocab, cur);
  }
  if (CLUSTER) {
    // The first CTA's shared memory may be written once that CTA is known to have started.  The wait passes under the first
    // loads, and CTAs without a row take part.
    __syncwarp();
    cluster_wait();
  }
  int turn = 0;
  while (row < a.rows) {
    // what the first thread needs of the row beside its pieces
    long long target = -1;
    float at_target = 0.f;
    if (a.targets && rank == 0 && threadIdx.x == 0) {
      target = a.targets[row];
      if (target >= 0 && target < a.vocab) at_target = lp_load(static_cast<const T*>(a.logits), lp_offset(a, row) + target);
    }
    const int upcoming = row >= a.rows - step ? a.rows : next(row + step);
    // 1. the sums
    LpRunning<T, ENT> sums;
    sums.clear();
    float mine = -INFINITY;
    const int chunks = max(sweep.chunks, 1);             // an empty slice of a cluster still hands its loads on
    auto chunk = [&](int k, const uint4 (&w)[kLpChunk], uint4 (&to_come)[kLpChunk]) {
      if (k + 1 < chunks) {
        sweep.load(k + 1, a.vocab, to_come);
      } else if (upcoming < a.rows) {
        sweep.start(a.logits, lp_offset(a, upcoming), a.vocab, rank, ranks);
        sweep.load(0, a.vocab, to_come);
      }
      float most[kLpChunk];
#pragma unroll
      for (int i = 0; i < kLpChunk; ++i) most[i] = lp_piece_max<T>(w[i]);
      float largest = most[0];
#pragma unroll
      for (int i = 1; i < kLpChunk; ++i) largest = lp_max(largest, most[i]);
      if (TOP) mine = lp_max(mine, largest);
      sums.add(w, most, lp_warp_max(largest));
    };
    for (int k = 0; k < chunks; ++k) {
      uint4 w[kLpChunk];
#pragma unroll
      for (int i = 0; i < kLpChunk; ++i) w[i] = cur[i];
      chunk(k, w, cur);
    }
    LpSums s = sums.warp_sums();
    if (TOP) {
      float group = mine;
#pragma unroll
      for (int o = 1; o < kPerGroup; o <<= 1) group = lp_max(group, __shfl_xor_sync(0xffffffffu, group, o));
      if (threadIdx.x % kPerGroup == 0) reinterpret_cast<float*>(sh.group)[threadIdx.x / kPerGroup] = group;
    }
    if (kWarps > 1 || TOP) {
      if (lane == 0) sh.part[turn][warp] = s;
      if (TOP && threadIdx.x == 0) sh.found = 0;         // the last row's has been read by everybody, a barrier ago
      __syncthreads();
    }
    if (warp == 0) {
      if (kWarps > 1) s = lp_join(sh.part[turn][lane < kWarps ? lane : 0], lane < kWarps);
      if (!CLUSTER && lane == 0) {
        const float2 mz = lp_finish(a, row, s, target, at_target);
        if (TOP) sh.result = mz;
      }
      if (CLUSTER && lane == 0) {
        const uint32_t to = in_first_cta(&sh.slice[turn][rank]);
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(s.m), "f"(s.count), "f"(s.rest), "f"(s.te) : "memory");
      }
    }
    // 2. the alternatives
    if (TOP) {
      bool slow_nan;
      const LpRow r = lp_row<T>(a.logits, lp_offset(a, row), a.vocab, rank, ranks);
      // The bound, by every warp for itself: the largest group maximum, taken away top - 1 times.
      float g0 = reinterpret_cast<const float*>(sh.group)[lane], g1 = -INFINITY;
      if (kGroups > 32) g1 = reinterpret_cast<const float*>(sh.group)[lane + 32];
      slow_nan = __any_sync(0xffffffffu, g0 != g0 || g1 != g1);
      float bound = lp_warp_max(lp_max(g0, g1));
      for (int k = 1; k < a.top && bound != -INFINITY && !slow_nan; ++k) {
        const uint32_t b0 = __ballot_sync(0xffffffffu, g0 == bound), b1 = __ballot_sync(0xffffffffu, g1 == bound);
        if (b0) {
          if (lane == __ffs(b0) - 1) g0 = -INFINITY;
        } else if (lane == __ffs(b1) - 1) {
          g1 = -INFINITY;
        }
        bound = lp_warp_max(lp_max(g0, g1));
      }
      // a warp's threads that have seen something that reaches it: their pieces again, two threads' at a time
      uint32_t hot = slow_nan || bound == -INFINITY ? 0u : __ballot_sync(0xffffffffu, mine >= bound);
      const int sweeps = r.pieces > 0 ? (r.pieces + THREADS - 1) / THREADS : 0;
      while (hot) {
        // more than can be kept: equal values, see below
        if (__shfl_sync(0xffffffffu, *const_cast<volatile int*>(&sh.found), 0) > kLpCandidates) break;
        const int h0 = __ffs(hot) - 1;
        hot &= hot - 1;
        const int h1 = hot ? __ffs(hot) - 1 : -1;
        hot &= hot - 1;                                          // of 0: 0
        const int h = lane < 16 ? h0 : h1;
        for (int k = h >= 0 ? lane & 15 : sweeps; k < sweeps; k += 16) {
          const int piece = warp * 32 + h + k * THREADS;
          if (piece >= r.pieces) continue;
          const uint4 w = lp_fetch<T>(r, a.vocab, piece);
          if (!(lp_piece_max<T>(w) >= bound)) continue;
          float f[kPiece];
          lp_unpack<T>(w, f);
          uint32_t reach = 0;
#pragma unroll
          for (int e = 0; e < kPiece; ++e) reach |= f[e] >= bound ? 1u << e : 0u;
          const int e0 = (r.first + piece) * kPiece - r.lead;
          while (reach) {                                        // hardly ever more than one
            const int e = __ffs(reach) - 1;
            reach &= reach - 1;
            if (e0 + e < 0 || e0 + e >= a.vocab) continue;
            const int word = sizeof(T) == 2 ? e >> 1 : e;
            const uint32_t bits = word == 0 ? w.x : word == 1 ? w.y : word == 2 ? w.z : w.w;
            const float x = __uint_as_float(sizeof(T) == 4 ? bits : e & 1 ? bits & 0xffff0000u : bits << 16);
            const int at = atomicAdd(&sh.found, 1);
            if (at < kLpCandidates) sh.keys[at] = lp_key(x, e0 + e);
          }
        }
        __syncwarp();
      }
      __syncthreads();
      int found = sh.found;
      if (found > kLpCandidates || (bound == -INFINITY && !slow_nan)) found = lp_collect_ties<T, THREADS>(r, a.vocab, a.top, bound, &sh);
      auto put = [&](int place, unsigned long long key) {
        if (!CLUSTER) {
          sh.picked[place] = key;
        } else {
          const uint32_t to = in_first_cta(&sh.slice_keys[turn][rank][place]);
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(key) : "memory");
        }
      };
      if (found > kLpCandidates || slow_nan) {
        lp_pick_slowly<T>(r, a.vocab, a.top, sh.best, sh.picked);
        if (CLUSTER && static_cast<int>(threadIdx.x) < a.top) put(threadIdx.x, sh.picked[threadIdx.x]);
      } else {
        // eight threads per candidate count the ones before it
        for (int c0 = 0; c0 < found; c0 += THREADS / 8) {
          const int c = c0 + threadIdx.x / 8;
          const unsigned long long key = c < found ? sh.keys[c] : 0;
          int before = 0;
          for (int j = threadIdx.x % 8; j < found; j += 8) before += sh.keys[j] > key;
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
          if (threadIdx.x % 8 == 0 && c < found && before < a.top) put(before, key);
        }
        if (CLUSTER && static_cast<int>(threadIdx.x) >= found && static_cast<int>(threadIdx.x) < a.top) put(threadIdx.x, 0);
      }
      if (!CLUSTER) {
        __syncthreads();                     // the places, and the first thread's result
        if (static_cast<int>(threadIdx.x) < a.top) lp_put_top(a, row, threadIdx.x, sh.picked[threadIdx.x], sh.result);
      }
    }
    if (CLUSTER) {
      // The first CTA reads row n's slices behind this barrier; the others write the same place again two rows on, behind the
      // barrier of the row between, at which the first CTA arrives only when it is done reading.
      __syncwarp();
      cluster_barrier();
      if (rank == 0) {
        if (warp == 0) {
          const LpSums all = lp_join(sh.slice[turn][lane < ranks ? lane : 0], lane < ranks);
          if (lane == 0) {
            const float2 mz = lp_finish(a, row, all, target, at_target);
            if (TOP) sh.result = mz;
          }
        }
        if (TOP) {
          __syncthreads();
          const float2 mz = sh.result;
          const int all = ranks * a.top;
          for (int c0 = 0; c0 < all; c0 += THREADS / 8) {
            const int c = c0 + threadIdx.x / 8, q = threadIdx.x % 8;
            const unsigned long long key = c < all ? sh.slice_keys[turn][c / a.top][c % a.top] : 0;
            int before = 0;
            if (key != 0 && q < ranks) {
              // a slice's keys descend: the ones before this one are its first ones
              int end = a.top;
              while (before < end) {
                const int mid = (before + end) >> 1;
                if (sh.slice_keys[turn][q][mid] > key) before = mid + 1;
                else end = mid;
              }
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
            if (q == 0 && key != 0 && before < a.top) lp_put_top(a, row, before, key, mz);
          }
        }
      }
    }
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
constexpr int kLpWarpPieces = 4, kLpPieces = 8;

template <typename T>
__device__ __forceinline__ void lp_store_piece(void* p, const float (&f)[16 / sizeof(T)]);
template <>
__device__ __forceinline__ void lp_store_piece<__nv_bfloat16>(void* p, const float (&f)[8]) { *static_cast<uint4*>(p) = pack_bf16x8(f); }
template <>
__device__ __forceinline__ void lp_store_piece<float>(void* p, const float (&f)[4]) {
  *static_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
}

// what a row's gradient is made of
struct LpGrad {
  float m, logz, whole, dh, h, dt;
  int target;                    // -1: nothing arrives for it
  float dk;                      // per lane: what arrives for its alternative
  int index;                     // that alternative, -1 outside the vocabulary
  bool zero;                     // nothing to read: the row is `fill`
  float fill;

  __device__ __forceinline__ void load(const LogprobBwdArgs& a, int row) {
    const float2 st = *reinterpret_cast<const float2*>(a.stats + 2LL * row);
    m = st.x;
    logz = st.y;
    dh = h = dt = dk = 0.f;
    if (a.d_entropy) { dh = a.d_entropy[row]; h = a.entropy[row]; }
    target = index = -1;
    if (a.d_logprob) {
      const long long t = a.targets[row];
      const float d = a.d_logprob[row];
      if (t != a.ignore_index) {
        const bool in = t >= 0 && t < a.vocab;
        target = in ? static_cast<int>(t) : -1;
        dt = in ? d : NAN;
      }
    }
    const int lane = threadIdx.x & 31;
    if (lane < a.top) {
      dk = a.d_top[static_cast<long long>(row) * a.top + lane];
      const long long t = a.top_index[static_cast<long long>(row) * a.top + lane];
      index = t >= 0 && t < a.vocab ? static_cast<int>(t) : -1;
    }
  }
  // once the loads are in; all threads of a warp
  __device__ __forceinline__ void ready(const LogprobBwdArgs& a) {
    whole = dk;
    if (a.top) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) whole += __shfl_xor_sync(0xffffffffu, whole, o);
    }
    whole += dt;
    zero = m == -INFINITY || (whole == 0.f && !a.top && !a.d_entropy);
    fill = whole == whole ? 0.f : NAN;
  }
  // the gradient of two tokens for which nothing arrives on its own
  template <bool ENT>
  __device__ __forceinline__ f32x2 of(f32x2 x) const {
    const f32x2 d = f2_add(x, f2_make(-m, -m));
    f32x2 lp = 0;
    float u0, u1;
    if (ENT) {
      lp = f2_add(d, f2_make(-logz, -logz));
      f2_split(f2_mul(lp, f2_make(kLog2e, kLog2e)), u0, u1);
    } else {
      f2_split(f2_fma(d, f2_make(kLog2e, kLog2e), f2_make(-logz * kLog2e, -logz * kLog2e)), u0, u1);
    }
    const f32x2 p = f2_make(lp_exp2(u0), lp_exp2(u1));
    if (!ENT) return f2_mul(p, f2_make(-whole, -whole));
    // p (-whole - dh (lp + h)): p is 0 long before lp is -10000: the bracket stays finite, a NaN stays one
    float l0, l1;
    f2_split(lp, l0, l1);
    lp = f2_make(lp_max(l0, -10000.f), lp_max(l1, -10000.f));
    return f2_mul(p, f2_fma(f2_add(lp, f2_make(h, h)), f2_make(-dh, -dh), f2_make(-whole, -whole)));
  }
  template <bool ENT>
  __device__ __forceinline__ float of(float x) const {
    float lo, hi;
    f2_split(of<ENT>(f2_make(x, x)), lo, hi);
    return lo;
  }
  // ... and of one for which `share` does
  template <bool ENT>
  __device__ __forceinline__ float of(float x, float share) const {
    const float lp = (x - m) - logz, p = expf(lp);
    const float g = (share - whole) * p - share * expm1f(lp);
    return ENT && p != 0.f ? g - dh * p * (lp + h) : g;
  }
};

// A warp takes a whole short row (WARP), a CTA one run of kWidth * kLpPieces pieces of a longer one.
template <typename T, bool WARP, bool ENT>
__global__ void __launch_bounds__(256) logprob_bwd_kernel(const LogprobBwdArgs a) {
  constexpr int kPiece = 16 / sizeof(T), kWidth = WARP ? 32 : 256, kPer = WARP ? kLpWarpPieces : kLpPieces;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int row = WARP ? static_cast<int>(blockIdx.x * 8 + (threadIdx.x >> 5)) : static_cast<int>(blockIdx.x), run = WARP ? 0 : blockIdx.y;
  if (WARP && (row >= a.rows || row < 0)) return;
  const T* x = static_cast<const T*>(a.logits) + lp_offset(a, row);
  T* out = static_cast<T*>(a.grad) + static_cast<long long>(row) * a.vocab;
  LpGrad g;
  g.load(a, row);
  // pieces counted from the aligned address at or below the row's start, if x and out lie alike
  const int phase = static_cast<int>(reinterpret_cast<uintptr_t>(out) & 15u), lead = phase / static_cast<int>(sizeof(T));
  const bool alike = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15u) == phase;
  const int first = run * (kWidth * kPer), last = min((lead + a.vocab + kPiece - 1) / kPiece, first + kWidth * kPer);
  g.ready(a);
  uint4 raw[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int piece = first + i * kWidth + t, e0 = piece * kPiece - lead;
    if (piece < last && alike && !g.zero && e0 >= 0 && e0 + kPiece <= a.vocab) raw[i] = load16_stream(x + e0);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int piece = first + i * kWidth + t, e0 = piece * kPiece - lead;
    if (piece >= last) continue;
    if (alike && e0 >= 0 && e0 + kPiece <= a.vocab) {
      float f[kPiece];
      if (g.zero) {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) f[e] = g.fill;
      } else {
        lp_unpack<T>(raw[i], f);
        const int hot = g.target - e0;
        const bool has = !a.top && hot >= 0 && hot < kPiece;
        float there = 0.f;
        if (has) {
#pragma unroll
          for (int e = 0; e < kPiece; ++e) there = e == hot ? f[e] : there;
          there = g.of<ENT>(there, g.dt);
        }
#pragma unroll
        for (int e = 0; e < kPiece; e += 2) f2_split(g.of<ENT>(f2_make(f[e], f[e + 1])), f[e], f[e + 1]);
        if (has) {
#pragma unroll
          for (int e = 0; e < kPiece; ++e) f[e] = e == hot ? there : f[e];
        }
      }
      lp_store_piece<T>(out + e0, f);
    } else {
      // a row's ragged end, or rows of x and out that lie differently
#pragma unroll 1
      for (int e = 0; e < kPiece; ++e) {
        const int c = e0 + e;
        if (c < 0 || c >= a.vocab) continue;
        float v = g.fill;
        if (!g.zero) v = c == g.target && !a.top ? g.of<ENT>(lp_load(x, c), g.dt) : g.of<ENT>(lp_load(x, c));
        out[c] = T(v);
      }
    }
  }
  if (a.top && !g.zero) {
    // the tokens for which something arrives: the alternatives, and the target behind them, one per lane and each by its
    // first mention; every warp of a CTA knows them, the first one writes those of the CTA's run
    if (WARP) __syncwarp();
    else __syncthreads();
    if (WARP || threadIdx.x < 32) {
      const int lane = threadIdx.x & 31, from = first * kPiece - lead, to = last * kPiece - lead;
      float share = 0.f, target_share = g.dt;
      bool seen = false, target_seen = false;
      for (int j = 0; j < a.top; ++j) {
        const int o = __shfl_sync(0xffffffffu, g.index, j);
        const float d = __shfl_sync(0xffffffffu, g.dk, j);
        if (o == g.index) { share += d; seen |= j < lane; }
        if (o == g.target) { target_share += d; target_seen = true; }
      }
      if (g.index == g.target) share += g.dt;
      if (lane < a.top && !seen && g.index >= 0 && g.index >= from && g.index < to) out[g.index] = T(g.of<ENT>(lp_load(x, g.index), share));
      if (lane == 0 && !target_seen && g.target >= 0 && g.target >= from && g.target < to)
        out[g.target] = T(g.of<ENT>(lp_load(x, g.target), target_share));
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

// clusters of `ranks` CTAs that the device holds at once; 0 where the query fails
template <typename K>
static int resident_clusters(K kernel, int threads, int ranks) {
  if (ranks == 1) return held_at_once(kernel, threads, 0);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(ranks); cfg.blockDim = dim3(threads); cfg.attrs = &attr; cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return 0;
  }
  return n;
}

template <typename T, int THREADS, bool ENT, bool TOP, bool CLUSTER>
static int run_logprob(const LogprobArgs& a, int ranks, cudaStream_t stream) {
  auto kernel = logprob_kernel<T, THREADS, ENT, TOP, CLUSTER>;
  static PerDevice resident[4];            // by cluster size
  const int held = resident[ranks == 8 ? 3 : ranks >> 1].get([&] { return resident_clusters(kernel, THREADS, ranks); });
  const long long most = held ? held : sm_count() / ranks;
  const long long clusters = a.rows < most ? a.rows : most;
  cudaError_t e;
  if (CLUSTER) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ranks; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * ranks)); cfg.blockDim = dim3(THREADS);
    cfg.stream = stream; cfg.attrs = &attr; cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) cudaGetLastError();                    // a refused launch is this call's error, not also the next one's
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

// What `rows` rows take on CTAs of which the device holds `places` at once, relative to their bytes: whole rounds, a last one
// that is not full but takes a third of a round at least, and what `extra` percent a row costs on such CTAs beside its bytes.
static double lp_cost(long long rows, long long places, int extra) {
  const long long whole = rows / places, rest = rows % places;
  const double rounds = static_cast<double>(whole) + (rest ? 0.35 + 0.65 * static_cast<double>(rest) / static_cast<double>(places) : 0.0);
  return rounds * static_cast<double>(places) * (100 + extra);
}

// Threads per row.  A row's end (joining the sums, finding the alternatives) is a chain of latencies that only other CTAs of
// the SM fill, so small CTAs -- more of them, each with more of a row per thread -- do better; large ones do where there are too
// few rows for all places, or where they leave a fuller last round.  Measured, us, with 256 / 128 / 64 threads (bf16, 32000
// tokens): with five alternatives and entropy 8192 rows 146 / 126 / 126, 4096 rows 76 / 65 / 71, 1000 rows 24 / 24 / 23, 300
// rows 10 / 12 / 16; log probabilities only 8192 rows 106 / 96 / 91, 4096 rows 55 / 50 / 50, 300 rows 9 / 10 / 12; fp32, 1024
// rows of 50265 with entropy 41 / 44 / 39.  The percentages below are these, less the rounds: shares of the bytes of such rows,
// by which the choice is within 2 % of the best of the three there.  A row's end does not grow with the vocabulary, so
// elsewhere it is further off.  With alternatives: 8200 tokens, 4096 rows 53 / 36 / 28 (128 are taken; 35 % off at worst);
// 131072 tokens, 1000 rows 61 / 78 / 90 (128, 27 %), 4096 rows 214 / 233 / 285 (128, 9 %); fp32, 32000 tokens, 1000 rows 33 /
// 41 / 45 (128, 23 %).  Log probabilities only: 8200 tokens, 4096 rows 33 / 24 / 19 (128, 25 %), 131072 tokens, 1000 rows 50 /
// 58 / 52 (64, 5 %).  Rows of fewer than two chunks take fewer threads in any case.
template <typename T>
static int lp_threads(const LogprobArgs& a, long long pieces) {
  if (pieces <= 2 * 32 * kLpChunk) return 32;
  if (pieces > 2 * 128 * kLpChunk && a.rows <= sm_count() * 3) return 256;          // every row has a place of its own
  const int most = pieces <= 2 * 64 * kLpChunk ? 64 : pieces <= 2 * 128 * kLpChunk ? 128 : 256;
  int best = 64;
  double least = lp_cost(a.rows, sm_count() * 12, a.top ? 55 : 9);
  if (most >= 128) {
    const double cost = lp_cost(a.rows, sm_count() * 6, a.top ? 53 : 16);
    if (cost < least) { best = 128; least = cost; }
  }
  if (most >= 256 && lp_cost(a.rows, sm_count() * 3, a.top ? 78 : 28) < least) best = 256;
  return best;
}

// Few long rows are spread over clusters, as far as a slice keeps 512 pieces (two per thread, half a chunk: all of them are then
// fetched under bounds) and four CTAs per SM go.
template <typename T>
static int launch_logprob(const LogprobArgs& a, cudaStream_t stream) {
  const long long pieces = (static_cast<long long>(a.vocab) * sizeof(T) + 15) / 16 + 1;
  int ranks = 1;
  while (ranks < 8 && static_cast<long long>(a.rows) * ranks * 2 <= sm_count() * 4 && pieces / (ranks * 2) >= 512) ranks *= 2;
  if (ranks > 1) return pick_logprob<T, 256, true>(a, ranks, stream);
  switch (lp_threads<T>(a, pieces)) {
    case 32: return pick_logprob<T, 32, false>(a, 1, stream);
    case 64: return pick_logprob<T, 64, false>(a, 1, stream);
    case 128: return pick_logprob<T, 128, false>(a, 1, stream);
    default: return pick_logprob<T, 256, false>(a, 1, stream);
  }
}

template <typename T, bool WARP, bool ENT>
static void run_logprob_bwd(const LogprobBwdArgs& a, int runs, cudaStream_t stream) {
  if (WARP) logprob_bwd_kernel<T, WARP, ENT><<<static_cast<unsigned>((a.rows + 7LL) / 8), 256, 0, stream>>>(a);
  else logprob_bwd_kernel<T, WARP, ENT><<<dim3(a.rows, runs), 256, 0, stream>>>(a);
}

template <typename T>
static int launch_logprob_bwd(const LogprobBwdArgs& a, cudaStream_t stream) {
  const long long pieces = (static_cast<long long>(a.vocab) * sizeof(T) + 15) / 16 + 1;
  const bool warp = pieces <= 32 * kLpWarpPieces;                       // short rows: a warp each
  const int width = warp ? 32 * kLpWarpPieces : 256 * kLpPieces, runs = static_cast<int>((pieces + width - 1) / width);
  if (warp) a.d_entropy ? run_logprob_bwd<T, true, true>(a, runs, stream) : run_logprob_bwd<T, true, false>(a, runs, stream);
  else a.d_entropy ? run_logprob_bwd<T, false, true>(a, runs, stream) : run_logprob_bwd<T, false, false>(a, runs, stream);
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
  a.logits = q->logits; a.row_stride = q->row_stride; a.batch_stride = q->batch_stride;
  a.rows = static_cast<int>(q->rows); a.seq = static_cast<int>(q->seq < 0x7fffffffLL ? q->seq : 0x7fffffffLL);
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
  a.logits = q->logits; a.row_stride = q->row_stride; a.batch_stride = q->batch_stride;
  a.rows = static_cast<int>(q->rows); a.seq = static_cast<int>(q->seq < 0x7fffffffLL ? q->seq : 0x7fffffffLL);
  a.vocab = q->vocab; a.top = q->d_top ? q->top : 0; a.targets = reinterpret_cast<const long long*>(q->targets);
  a.ignore_index = q->ignore_index; a.stats = q->stats; a.entropy = q->entropy; a.d_logprob = q->d_logprob;
  a.d_entropy = q->d_entropy; a.d_top = q->d_top; a.top_index = reinterpret_cast<const long long*>(q->top_index); a.grad = q->grad;
  return q->dtype == HYC_BF16 ? launch_logprob_bwd<__nv_bfloat16>(a, stream) : launch_logprob_bwd<float>(a, stream);
}

}  // extern "C"
