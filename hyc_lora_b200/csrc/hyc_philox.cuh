// Counter-based random words for the dropout kernels: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011).  Element i of the tensor of call c under the seed s takes word i % 4 of the block
// with counter (i / 4, c) and key s, so the mask of a call is a function of (seed, call, element index) alone: the
// backward pass draws it again in whatever order its threads run, and no mask is ever written to memory.
#pragma once

#include <math.h>
#include <stdint.h>

namespace hyc {

struct Philox {
  uint32_t k0, k1;   // seed
  uint32_t c2, c3;   // call number

  __device__ __forceinline__ static Philox load(const long long* seed_call) {
    const unsigned long long s = static_cast<unsigned long long>(seed_call[0]), c = static_cast<unsigned long long>(seed_call[1]);
    return {static_cast<uint32_t>(s), static_cast<uint32_t>(s >> 32), static_cast<uint32_t>(c), static_cast<uint32_t>(c >> 32)};
  }

  __device__ __forceinline__ uint4 block(unsigned long long index) const {
    uint32_t x0 = static_cast<uint32_t>(index), x1 = static_cast<uint32_t>(index >> 32), x2 = c2, x3 = c3, a = k0, b = k1;
#pragma unroll
    for (int round = 0; round < 10; ++round) {
      const unsigned long long p0 = static_cast<unsigned long long>(x0) * 0xD2511F53u;
      const unsigned long long p1 = static_cast<unsigned long long>(x2) * 0xCD9E8D57u;
      x0 = static_cast<uint32_t>(p1 >> 32) ^ x1 ^ a;
      x1 = static_cast<uint32_t>(p1);
      x2 = static_cast<uint32_t>(p0 >> 32) ^ x3 ^ b;
      x3 = static_cast<uint32_t>(p0);
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(x0, x1, x2, x3);
  }
};

// What a dropout rate becomes on the device: an element is kept where its word is at least `border`, p in 32 bits;
// a rate that rounds to 1 keeps nothing.  Kept values are multiplied by 1 / (1 - p), rounded once to fp32.
struct DropRate {
  uint32_t border;
  float scale;
  int none;          // keep nothing

  static DropRate make(double p) {
    const double words = rint(p * 4294967296.0);
    DropRate r;
    r.none = words >= 4294967296.0;
    r.border = r.none ? 0xffffffffu : static_cast<uint32_t>(words);
    r.scale = r.none ? 0.f : static_cast<float>(1.0 / (1.0 - p));
    return r;
  }
  __device__ __forceinline__ bool keep(uint32_t word) const { return word >= border && !none; }
};

}  // namespace hyc
