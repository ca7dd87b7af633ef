// PAM products of many elements by one number.
//
// pam(x, s) is the sum of two patterns and a constant where |x s| lies within the range rule's bounds, and the rule costs more than the sum: a product, two comparisons
// and two selections.  Where |x| itself lies in a band that keeps |x s| between 2^-118 and 2^119, nothing is cut off, and one comparison of the largest of four
// neighbours shows that for all of them.  (A PAM product is at most an eighth below the true one.)
#pragma once

#include "pam_scalar.cuh"

namespace pamk {

struct Times {
    float s;
    int32_t off, add;
    uint32_t low, span;                   // twice the pattern of the least |x| of the band, and how far the greatest is from there

    Times() = default;
    Times(float by, int32_t offset) : s(by), off(offset), add(iadd(isub(f2i(by), kBias), offset)), low(0), span(0) {
        const int64_t size = f2i(by) & 0x7fffffff, one = kBias;
        if (size < (1 << 23) || size >= 0x7f800000) return;                           // (zero, denormal, not finite: no band)
        const int64_t least = one - ((int64_t)118 << 23) - (size - one), most = one + ((int64_t)118 << 23) - (size - one);
        const int64_t from = least > (1 << 23) ? least : (1 << 23), to = most < 0x7f7fffff ? most : 0x7f7fffff;
        if (to <= from) return;
        low = 2u * (uint32_t)from;
        span = 2u * (uint32_t)(to - from);
    }
#if defined(__CUDACC__)
    __device__ __forceinline__ uint32_t beyond(float x) const { return 2u * (uint32_t)f2i(x) - low; }                  // below `span` in the band
    __device__ __forceinline__ bool plain(const float4& x) const { return max(max(beyond(x.x), beyond(x.y)), max(beyond(x.z), beyond(x.w))) < span; }
    __device__ __forceinline__ float one(float x) const { return mul(x, s, off); }
    __device__ __forceinline__ float4 of(const float4& x) const {
        if (plain(x)) return make_float4(i2f(iadd(f2i(x.x), add)), i2f(iadd(f2i(x.y), add)), i2f(iadd(f2i(x.z), add)), i2f(iadd(f2i(x.w), add)));
        return make_float4(one(x.x), one(x.y), one(x.z), one(x.w));
    }
#endif
};

}  // namespace pamk
