// Random bits from a counter: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011).
//
// Four 32-bit words for every 128-bit counter under a 64-bit key.  A round multiplies two of the words by constants and swaps the halves of the
// products, with the other two words and the round's key added without carry; the key grows by two constants from round to round.  Here the
// counter is the number of a block of four neighbouring elements and the key is the seed of the call, so an element's bits depend on its place and the
// seed alone, whoever asks for them and whenever: a mask is drawn again instead of being stored.
//
// The element stays where its bits reach p 2^32, to the nearest whole number, and is then multiplied by the fp32 number next to 1 / (1 - p).
#pragma once

#include <math.h>
#include <stdint.h>

namespace pamk {

struct Dropping {
    const int64_t* seed_at;               // on the device, or null: `seed`
    int64_t seed;
    uint32_t below;                       // elements whose bits are below this are dropped
    float scale;
};

// For 0 < p < 1 (a p within 2^-33 of one drops all but one of 2^32).
inline Dropping dropping(double p, const int64_t* seed_at, int64_t seed) {
    const double below = nearbyint(p * 4294967296.0);
    return {seed_at, seed, below >= 4294967295.0 ? 0xffffffffu : (uint32_t)below, (float)(1.0 / (1.0 - p))};
}

#if defined(__CUDACC__)
__device__ __forceinline__ uint2 key_of(const Dropping& d) {
    const int64_t s = d.seed_at ? __ldg(reinterpret_cast<const long long*>(d.seed_at)) : d.seed;
    return make_uint2((uint32_t)s, (uint32_t)((uint64_t)s >> 32));
}

__device__ __forceinline__ uint4 philox(uint64_t block, uint2 key) {
    uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), c = 0u, d = 0u;
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t left = (uint64_t)a * 0xd2511f53u, right = (uint64_t)c * 0xcd9e8d57u;
        a = (uint32_t)(right >> 32) ^ b ^ (key.x + round * 0x9e3779b9u);
        c = (uint32_t)(left >> 32) ^ d ^ (key.y + round * 0xbb67ae85u);
        b = (uint32_t)right;
        d = (uint32_t)left;
    }
    return make_uint4(a, b, c, d);
}
#endif

}  // namespace pamk
