// Counter-based random words for the dropout kernels: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011).  Element i of the tensor of call c under the seed s takes word i % 4 of the block
// with counter (i / 4, c) and key s, so the mask of a call is a function of (seed, call, element index) alone: the
// backward pass draws it again in whatever order its threads run, and no mask is ever written to memory.
#pragma once

#include <math.h>
#include <stdint.h>

namespace hyc {

// The multiplications bound it: a 32 x 32 -> 64 bit product takes four issue cycles of a scheduler (measured), 18 of them are
// 72 cycles per 128 words, 18 cycles per 32 elements against the 22 in which a bf16 dropout's traffic passes.  So the round
// keys, the same in every thread, are kept in uniform registers (a warp-wide reduction tells the compiler that they are), and
// what the first two rounds make of the call number and of the upper half of the index, which hardly ever changes, is made
// once per thread: 2 of their 4 products.
__device__ __forceinline__ void philox_product(uint32_t a, uint32_t factor, uint32_t& hi, uint32_t& lo) {
  asm("{\n\t.reg .b64 p;\n\tmul.wide.u32 p, %2, %3;\n\tmov.b64 {%1, %0}, p;\n\t}" : "=r"(hi), "=r"(lo) : "r"(a), "r"(factor));
}

struct Philox {
  uint32_t k0, k1;         // seed, warp-uniform
  uint32_t c2, c3;         // call number, warp-uniform
  uint32_t upper;          // upper half of the index that the following are for
  uint32_t e, f, g, h;

  // all threads of the warp
  __device__ __forceinline__ static Philox load(const long long* seed_call) {
    const unsigned long long s = static_cast<unsigned long long>(__ldg(seed_call)), c = static_cast<unsigned long long>(__ldg(seed_call + 1));
    Philox p;
    p.k0 = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(s));
    p.k1 = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(s >> 32));
    p.c2 = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(c));
    p.c3 = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(c >> 32));
    p.prepare(0);
    return p;
  }

  __device__ __forceinline__ void prepare(uint32_t index_upper) {
    upper = index_upper;
    const unsigned long long first = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
    const unsigned long long second = static_cast<unsigned long long>(static_cast<uint32_t>(first >> 32) ^ index_upper ^ k0) * 0xD2511F53u;
    e = c3 ^ k1;
    f = static_cast<uint32_t>(first) ^ (k0 + 0x9E3779B9u);
    g = static_cast<uint32_t>(second >> 32) ^ (k1 + 0xBB67AE85u);
    h = static_cast<uint32_t>(second);
  }

  // the block of an index whose upper half is the prepared one
  __device__ __forceinline__ uint4 block(uint32_t index) const {
    uint32_t hi, lo, x0, x1, x2, x3;
    // rounds 0 and 1
    philox_product(index, 0xD2511F53u, hi, lo);
    x2 = lo ^ g;
    philox_product(hi ^ e, 0xCD9E8D57u, hi, x1);
    x0 = hi ^ f;
    x3 = h;
    uint32_t a = k0 + 2u * 0x9E3779B9u, b = k1 + 2u * 0xBB67AE85u;
#pragma unroll
    for (int round = 2; round < 10; ++round) {
      uint32_t hi0, lo0, hi1, lo1;
      philox_product(x0, 0xD2511F53u, hi0, lo0);
      philox_product(x2, 0xCD9E8D57u, hi1, lo1);
      x0 = hi1 ^ x1 ^ a;
      x1 = lo1;
      x2 = hi0 ^ x3 ^ b;
      x3 = lo0;
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(x0, x1, x2, x3);
  }

  // any index
  __device__ __forceinline__ uint4 at(unsigned long long index) {
    if (static_cast<uint32_t>(index >> 32) != upper) prepare(static_cast<uint32_t>(index >> 32));
    return block(static_cast<uint32_t>(index));
  }
};

// What a dropout rate becomes on the device: an element is kept where its word is at least `border`, p in 32 bits, and is
// then multiplied by 1 / (1 - p), rounded once to fp32.  A rate that rounds to 1 keeps nothing (`none`): no 32-bit border says
// that, so the kernels take what is to be dropped as zeros then, and scale is 0.
struct DropRate {
  uint32_t border;
  float scale;
  int none;

  static DropRate make(double p) {
    const double words = rint(p * 4294967296.0);
    DropRate r;
    r.none = words >= 4294967296.0;
    r.border = r.none ? 0xffffffffu : static_cast<uint32_t>(words);
    r.scale = r.none ? 0.f : static_cast<float>(1.0 / (1.0 - p));
    return r;
  }
  __device__ __forceinline__ bool keep(uint32_t word) const { return word >= border; }
};

}  // namespace hyc
