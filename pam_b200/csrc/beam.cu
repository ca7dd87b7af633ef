// Beam search: the best continuations of every group of beams from their logits, and the beams' states moved to where they go on.
//
// Selection.  A candidate is a beam and a token; its value is the beam's score plus the PAM log-softmax of the beam's logits
// (pam/pam_ops.py:331-347):
//     t_j = pam(x_j, log2 e)    m = floor(max_j t_j)    S = sum_j 2^(floor(t_j) - m) (1 + (t_j - floor(t_j)))
//     value_j = (x_j - pad(m + log2(S), log2 e)) + score           log2(2^i (1 + f)) = i + f
// t and the terms of S are fp32 values, exact or rounded once (1 + fraction; scaling by a power of two is exact); S, the logarithm, the quotient and the value
// are 64-bit ones, so that candidates of different beams are told apart where fp32 could not.  Within a beam the larger logit comes
// first, whatever the value's rounding.
//
// The logits are read once.  A first kernel takes up to 4092 of a beam's logits into the registers of a CTA and leaves
// their maximum, their sum and the best k of them: where each of W warps has k / W logits of at least some value, the k-th largest of all is no
// smaller, so the least of the warps' (k / W)-th largest thread maxima leaves a few dozen candidates, and each of those counts how many are
// larger.  Keys (logit, then lower token) are all different, so a candidate's rank is its place, and no order of atomics shows.  A
// second kernel joins the parts of each beam and picks the k best of the group from the lists in the same way.
// (A closer bound, the k-th largest of all that the warps give, leaves a dozen candidates and costs more than they do: 128 x 5 beams 24 -> 26 us.)
#include <type_traits>

#include "common.cuh"
#include "pam_scalar.cuh"

namespace pamk {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kThreads = 256, kEach = 16, kMostLogits = kThreads * kEach;
constexpr int kMostPicked = 64;                       // k
constexpr int kMostLists = 4096;
constexpr float kMasked = -1e30f;                     // a logit as low as this is masked
constexpr uint32_t kMaskedKey = 1u;                   // masked or banned; 0: no logit at all

struct Select {
    const float *logits, *scores;                     // scores [groups, rows]
    const unsigned char* banned;                      // or null
    int64_t x_group, x_row, ban_group, ban_row;
    int rows, vocab, k, parts, part;                  // a beam's logits in `parts` ranges of `part`
    double* sums;                                     // [groups * rows, parts]
    float* shifts;
    unsigned long long* lists;                        // [groups * rows, parts, k], largest first, 0 where there are fewer
    float* out_scores;
    int64_t *out_beams, *out_tokens;
};

__device__ __forceinline__ bool dead(float score) { return !(score > -INFINITY); }        // -inf or NaN

// Larger for larger x (no NaN); -0 as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
    const int32_t b = f2i(fadd(x, 0.0f));
    return (uint32_t)b ^ (b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_ordered(uint32_t u) { return i2f((int32_t)(u ^ (u & 0x80000000u ? 0x80000000u : 0xffffffffu))); }
__device__ __forceinline__ unsigned long long ordered(double x) {
    const long long b = __double_as_longlong(x + 0.0);
    return (unsigned long long)b ^ (b < 0 ? 0xffffffffffffffffull : 0x8000000000000000ull);
}

__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    return s;
}

// 2^e for whole e from -127 (there 0) to 127: e + 127 are the low bits of the sum
__device__ __forceinline__ float power_of(float e) { return i2f(f2i(fadd(e, 8388608.0f + 127.0f)) << 23); }

// s 2^e for whole e <= 0 (-inf and NaN among them: 0, unless s is NaN)
__device__ __forceinline__ double rescaled(double s, float e) {
    return e >= -1000.0f ? s * __longlong_as_double((long long)((int)e + 1023) << 52) : s == s ? 0.0 : s;
}

// A term of the sum: t = pam(x, log2 e) as 1 + fraction, times a power of two.
__device__ __forceinline__ double term(float t, float shift) {
    const float whole = floorf(t), lin = fadd(1.0f, fadd(t, -whole));
    return (double)fmul(lin, power_of(fmaxf(fadd(whole, -shift), -127.0f)));
}

// Below kBand where the exponent field lies in [66, 187]: the product with log2 e passes the range rule, and such a logit is not masked (|x| < 2^61, and
// -1e30 is beyond it).
__device__ __forceinline__ uint32_t beyond(float x) { return 2u * (uint32_t)f2i(x) - 2u * (66u << 23); }
constexpr uint32_t kBand = 2u * ((188u - 66u) << 23);

// Below kNear where |x| lies in [2^-61, 64): t 2^23 and the pattern of a term are then within 32 bits.
constexpr uint32_t kNear = 2u * ((133u - 66u) << 23);

constexpr int kWarps = kThreads / 32, kQuads = kEach / 4;
static_assert(kWarps == 8 && kQuads == 4);
constexpr int kMany = 512;                            // so many candidates are narrowed down by their full keys first

// Bound by instructions and the barriers between them: 740 per warp and 512 logits, the sum's terms the smaller part of them, issued in 71 % of the cycles; 155 MB of logits and 39 of
// flags in 78 us with a cold cache, 2.5 TB/s.
// (Five CTAs on an SM in 48 registers: 64 x 4 beams of 151643 words 91 -> 81 us; six spill, 90.)
__global__ void __launch_bounds__(kThreads, 5) pick_kernel(const Select a) {
    __shared__ unsigned long long found[kMostLogits];
    __shared__ double warp_total[kWarps];
    __shared__ float warp_shift[kWarps];
    __shared__ float bounds[kWarps];
    __shared__ unsigned long long warp_key[kWarps];
    __shared__ int count, live;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const unsigned beam = blockIdx.x, group = beam / (unsigned)a.rows, row = beam - group * a.rows;
    after_previous();
    const int begin = (int)blockIdx.y * a.part, end = min(begin + a.part, a.vocab);
    const float score = a.scores[beam];
    const float* x = a.logits + group * a.x_group + row * a.x_row;
    const unsigned char* banned = a.banned ? a.banned + group * a.ban_group + row * a.ban_row : nullptr;
    if (dead(score)) return;                                                      // (its logits are not looked at)
    // vectors start at addresses that are multiples of 16 bytes: the first one may begin before the range
    const int first = begin - (int)((reinterpret_cast<uintptr_t>(x + begin) >> 2) & 3);
    float4 v[kQuads];
    uint32_t flags[kQuads];                                                       // a byte for each of the four: banned
    const auto start = [&](int i) { return first + (i * kThreads + t) * 4; };
    const auto whole = [&](int i) { return (i > 0 || start(i) >= begin) && start(i) <= end - 4; };
    const bool by_four = banned && (reinterpret_cast<uintptr_t>(banned + first) & 3) == 0;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
        const int j = start(i);
        v[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);           // (masked, where there is nothing)
        flags[i] = 0u;
        if (whole(i)) v[i] = __ldcs(reinterpret_cast<const float4*>(x + j));
    }
    if (by_four)
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
            if (whole(i)) flags[i] = *reinterpret_cast<const uint32_t*>(banned + start(i));
    // the two vectors that the range may cut
    const auto cut = [&](int i) {
        const int j = start(i);
        if (j >= begin && j < end) v[i].x = x[j];
        if (j + 1 >= begin && j + 1 < end) v[i].y = x[j + 1];
        if (j + 2 >= begin && j + 2 < end) v[i].z = x[j + 2];
        if (j + 3 >= begin && j + 3 < end) v[i].w = x[j + 3];
    };
    const int last = (end - first) / 4;
    const bool cuts_first = t == 0 && first < begin, cuts_last = ((end - first) & 3) != 0 && t == last % kThreads;
    if (cuts_first) cut(0);
    if (cuts_last)
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
            if (i == last / kThreads) cut(i);
    if (banned && (!by_four || cuts_first || cuts_last))
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            const int j = start(i);
            if (j < end && !(by_four && whole(i)))
#pragma unroll 1
                for (int e = 0; e < 4; ++e)
                    if (j + e >= begin && j + e < end && banned[j + e]) flags[i] |= 1u << (8 * e);
        }
    if (t == 0) count = live = 0;
    const auto value = [&](int i, int e) { return e == 0 ? v[i].x : e == 1 ? v[i].y : e == 2 ? v[i].z : v[i].w; };
    const auto flag = [&](int i, int e) { return (flags[i] >> (8 * e) & 0xffu) != 0u; };
    // maxima: of all (for the shift), and of what may be chosen, by quads
    float best[kQuads];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) best[i] = fmaxf(fmaxf(v[i].x, v[i].y), fmaxf(v[i].z, v[i].w));
    const float all = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
    if ((flags[0] | flags[1] | flags[2] | flags[3]) != 0u)
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            best[i] = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e) best[i] = flag(i, e) ? best[i] : fmaxf(best[i], value(i, e));
        }
    const float most = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
    // the n-th largest distinct thread maximum, n = k / W rounded up, of the W warps that have one in each lane
    const int full = min(max((end - first) / 128, 1), kWarps), need = (a.k + full - 1) / full;
    const uint32_t masked = ordered(kMasked);
    uint32_t left = max(ordered(most), masked), least = masked;
    for (int i = 0; i < need; ++i) {
        least = __reduce_max_sync(0xffffffffu, left);
        left = left == least ? masked : left;
    }
    if (lane == 0) bounds[warp] = least == masked ? -INFINITY : of_ordered(least);
    const float top = of_ordered(__reduce_max_sync(0xffffffffu, ordered(all)));
    // the sum, shifted by the warp's own maximum
    const float shift = top > kMasked ? floorf(mul(top, kLog2e, 0)) : -INFINITY;
    const int32_t by = isub(f2i(kLog2e), kBias);
    double total = 0.0;
    uint32_t far[kQuads];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) far[i] = max(max(beyond(v[i].x), beyond(v[i].y)), max(beyond(v[i].z), beyond(v[i].w)));
    if (__all_sync(0xffffffffu, max(max(far[0], far[1]), max(far[2], far[3])) < kNear)) {
        // (a term's exponent is the whole part of t - shift, its mantissa the fraction, rounded once; what is below 2^-126 is as good as nothing)
        const int32_t least_exponent = isub(kBias, (int)shift << 23);
        const auto near_term = [&](float y) { return (double)i2f(__viaddmax_s32(__float2int_rn(i2f(iadd(f2i(y), by + (23 << 23)))), least_exponent, 0)); };
#pragma unroll
        for (int i = 0; i < kQuads; ++i) total += (near_term(v[i].x) + near_term(v[i].y)) + (near_term(v[i].z) + near_term(v[i].w));
    } else {
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            if (start(i) >= end) continue;
            if (far[i] < kBand) {
                const double s01 = term(i2f(iadd(f2i(v[i].x), by)), shift) + term(i2f(iadd(f2i(v[i].y), by)), shift);
                total += s01 + (term(i2f(iadd(f2i(v[i].z), by)), shift) + term(i2f(iadd(f2i(v[i].w), by)), shift));
            } else {
#pragma unroll 1
                for (int e = 0; e < 4; ++e) {
                    const float y = value(i, e);
                    if (!(y <= kMasked)) {
                        const float s = mul(y, kLog2e, 0);
                        total += s == s && shift > -INFINITY ? term(s, shift) : (double)quiet_nan();       // (NaN, or too large)
                    }
                }
            }
        }
    }
    total = warp_sum(total);
    if (lane == 0) {
        warp_total[warp] = total;
        warp_shift[warp] = shift;
    }
    __syncthreads();
    const auto key = [&](int i, int e) {                                          // 0 outside the range
        const int j = start(i) + e;
        if (j < begin || j >= end) return 0ull;
        const float y = value(i, e);
        return (unsigned long long)(y > kMasked && !flag(i, e) ? ordered(y) : kMaskedKey) << 32 | (uint32_t)~j;
    };
    const auto push = [&](unsigned long long full) { found[atomicAdd(&count, 1)] = full; };
    float bound = bounds[min(lane & 7, full - 1)];
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) bound = fminf(bound, __shfl_xor_sync(0xffffffffu, bound, d));
    if (bound > kMasked) {
        if (most >= bound)
#pragma unroll
            for (int i = 0; i < kQuads; ++i)
                if (best[i] >= bound)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (value(i, e) >= bound && !flag(i, e)) push((unsigned long long)ordered(value(i, e)) << 32 | (uint32_t)~(start(i) + e));
    } else {
        // too few to choose from for a bound: all of them, and masked ones from the first on, of which as many are needed at most
        int mine = 0;
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) mine += value(i, e) > kMasked && !flag(i, e);
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0 && mine) atomicAdd(&live, mine);
        __syncthreads();
        const int before = begin + a.k + live;
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned long long here = key(i, e);
                if (here && ((uint32_t)(here >> 32) != kMaskedKey || start(i) + e < before)) push(here);
            }
    }
    __syncthreads();
    const int at_first = count;
    __syncthreads();
    if (at_first > kMany) {
        // many equal ones: the k-th largest full key of a warp's threads is a bound that they do not share, or the least of two warps' (k / 2)-th largest where k
        // is more than a warp has (four have one in each thread where so many were found)
        unsigned long long first_key = 0ull;
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) first_key = max(first_key, key(i, e));
        const int of_each = a.k > 32 ? (a.k + 1) / 2 : a.k;
        int rank = 0;
#pragma unroll 8
        for (int l = 0; l < 32; ++l) rank += __shfl_sync(0xffffffffu, first_key, l) > first_key;
        const unsigned who = __ballot_sync(0xffffffffu, rank == of_each - 1 && first_key != 0ull);
        const unsigned long long mine = who ? __shfl_sync(0xffffffffu, first_key, __ffs(who) - 1) : 1ull;
        if (lane == 0) warp_key[warp] = mine;
        if (t == 0) count = 0;
        __syncthreads();
        unsigned long long from = 1ull, second = 1ull;
        for (int w = 0; w < kWarps; ++w) {
            second = max(second, min(from, warp_key[w]));
            from = max(from, warp_key[w]);
        }
        if (a.k > 32) from = second;
#pragma unroll
        for (int i = 0; i < kQuads; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (key(i, e) >= from) push(key(i, e));
        __syncthreads();
    }
    const int64_t list = (int64_t)beam * a.parts + blockIdx.y;
    if (t == 0) {
        float m = warp_shift[0];
        for (int w = 1; w < kWarps; ++w) m = fmaxf(m, warp_shift[w]);
        double sum = 0.0;
        for (int w = 0; w < kWarps; ++w) sum += rescaled(warp_total[w], fadd(warp_shift[w], -m));
        a.sums[list] = sum;
        a.shifts[list] = m;
    }
    unsigned long long* to = a.lists + list * a.k;
    const int n = count;
    for (int i = t; i < n; i += kThreads) {
        const unsigned long long mine = found[i];
        int r = 0;
        for (int o = 0; o < n; ++o) r += found[o] > mine;
        if (r < a.k) to[r] = mine;
    }
    for (int i = n + t; i < a.k; i += kThreads) to[i] = 0ull;
}

// pad(a, b) in 64 bits for b = log2 e: pam/pam_ops.py:342, cuda_kernels.cu:60-83 on patterns of 64 bits
__device__ __forceinline__ double over_log2e(double x) {
    const long long by = __double_as_longlong((double)kLog2e), one = __double_as_longlong(1.0);
    if (!(fabs(x) < 1e37)) return (double)quiet_nan();                             // (also NaN)
    if (x == 0.0) return 0.0;                                                      // (a whole number plus a logarithm is nothing else below 1e-37)
    return __longlong_as_double(__double_as_longlong(x) - by + one);
}

// log2 of a positive normal number
__device__ __forceinline__ double affine_log2(double x) {
    const long long b = __double_as_longlong(x);
    const double fraction = __longlong_as_double((b & 0xfffffffffffffll) | 0x3ff0000000000000ll) - 1.0;
    return (double)((int)(b >> 52) - 1023) + fraction;
}

struct Candidate {
    unsigned long long value, key;                    // value: 0 for none
    int beam;
    __device__ __forceinline__ bool before(const Candidate& o) const {
        if (value != o.value) return value > o.value;
        if (beam != o.beam) return beam < o.beam;
        return key > o.key;
    }
};

// i / n for 0 <= i <= 8192, given 1 / n: (i + 1/2) / n is 1 / 2n from a whole number at least, and the roundings reach less than (i + 1/2) / n 2^-22
__device__ __forceinline__ int quotient(int i, float one_over_n) { return (int)fmul(fadd((float)i, 0.5f), one_over_n); }

// `KEPT`: the lists have been copied to shared memory.  A chain of five barriers between short loops, one CTA for a group: bound by latency, 11 us for 15 lists of 10 each in 128
// groups, alone with a cold cache.
template <bool KEPT>
__global__ void __launch_bounds__(kThreads) merge_kernel(const Select a) {
    extern __shared__ __align__(16) unsigned char shared[];
    __shared__ Candidate least;
    __shared__ int count;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int lists = a.rows * a.parts, entries = lists * a.k;
    double* lse = reinterpret_cast<double*>(shared);                              // [rows], NaN for a beam without finite sum
    double* score = lse + a.rows;                                                 // [rows]
    unsigned long long* heads = reinterpret_cast<unsigned long long*>(score + a.rows);   // [lists]
    unsigned long long* kept = heads + lists;                                     // [lists, k]
    Candidate* found = reinterpret_cast<Candidate*>(kept + (KEPT ? entries : 0));
    const int64_t first_beam = (int64_t)blockIdx.x * a.rows;
    const unsigned long long* from = a.lists + first_beam * a.parts * a.k;
    for (int r = t; r < a.rows; r += kThreads) score[r] = (double)a.scores[first_beam + r];
    after_previous();
    if (KEPT)
        for (int i = t; i < entries; i += kThreads) kept[i] = __ldcg(from + i);   // (of a beam that is not continued: anything)
    for (int r = warp; r < a.rows; r += kThreads / 32) {
        double value = (double)quiet_nan();
        if (!dead(a.scores[first_beam + r])) {
            const int64_t at = (first_beam + r) * a.parts;
            float m = -INFINITY;
            double sum = 0.0;
            for (int c = lane; c < a.parts; c += 32) m = fmaxf(m, __ldcg(a.shifts + at + c));
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            for (int c = lane; c < a.parts; c += 32) sum += rescaled(__ldcg(a.sums + at + c), fadd(__ldcg(a.shifts + at + c), -m));
            sum = warp_sum(sum);
            if (sum > 0.0 && sum < 1e300) value = over_log2e((double)m + affine_log2(sum));
        }
        if (lane == 0) lse[r] = value;
    }
    if (t == 0) {
        count = 0;
        least.value = 0ull;                           // (fewer than k lists have entries: no bound)
        least.key = 0ull;
        least.beam = a.rows;
    }
    __syncthreads();
    const float one_over_parts = 1.0f / (float)a.parts;
    const auto beam_of = [&](int list) { return quotient(list, one_over_parts); };
    // entry i of a list as a candidate; a beam without finite sum has its first tokens at -inf
    const auto candidate = [&](int beam, int list, int i) {
        Candidate c;
        c.beam = beam;
        const double by = lse[c.beam];
        if (by != by) {
            c.key = list == beam * a.parts && i < a.vocab ? (unsigned long long)kMaskedKey << 32 | (uint32_t)~i : 0ull;
            c.value = c.key ? ordered((double)-INFINITY) : 0ull;
            return c;
        }
        c.key = KEPT ? kept[list * a.k + i] : __ldcg(from + (int64_t)list * a.k + i);
        const uint32_t x = (uint32_t)(c.key >> 32);
        c.value = c.key == 0ull ? 0ull
                                : ordered(x == kMaskedKey ? (double)-INFINITY : ((double)of_ordered(x) - by) + score[c.beam]);
        return c;
    };
    // The k-th best head of a list bounds the k-th best candidate: only k lists reach it.
    const bool bounded = lists >= a.k;
    if (bounded) {
        for (int i = t; i < lists; i += kThreads) heads[i] = candidate(beam_of(i), i, 0).value;
        __syncthreads();
        for (int i = t; i < lists; i += kThreads) {
            const unsigned long long mine = heads[i];
            if (mine == 0ull) continue;
            int r = 0, same = 0;
#pragma unroll 4
            for (int o = 0; o < lists; ++o) {
                r += heads[o] > mine;
                same += heads[o] == mine;
            }
            if (r >= a.k || r + same < a.k) continue;
            const Candidate full = candidate(beam_of(i), i, 0);
            if (same > 1)
                for (int o = 0; o < lists; ++o) r += heads[o] == mine && o != i && candidate(beam_of(o), o, 0).before(full);
            if (r == a.k - 1) least = full;
        }
        __syncthreads();
    }
    if (KEPT) {
        const float one_over_k = 1.0f / (float)a.k;
        for (int i = t; i < entries; i += kThreads) {
            const int list = quotient(i, one_over_k);
            const Candidate c = candidate(beam_of(list), list, i - list * a.k);
            if (c.value != 0ull && !(bounded && least.before(c))) found[atomicAdd(&count, 1)] = c;
        }
    } else {
        for (int i = t; i < lists; i += kThreads)
            for (int e = 0; e < a.k; ++e) {
                const Candidate c = candidate(beam_of(i), i, e);
                if (c.value == 0ull || (bounded && least.before(c))) break;
                found[atomicAdd(&count, 1)] = c;
            }
    }
    __syncthreads();
    const int n = count;
    for (int i = t; i < n; i += kThreads) {
        const Candidate mine = found[i];
        int r = 0;
        for (int o = 0; o < n; ++o) r += found[o].before(mine);
        if (r < a.k) {
            const int64_t to = (int64_t)blockIdx.x * a.k + r;
            const uint32_t x = (uint32_t)(mine.key >> 32);
            a.out_scores[to] = x == kMaskedKey ? -INFINITY : (float)(((double)of_ordered(x) - lse[mine.beam]) + score[mine.beam]);
            a.out_beams[to] = mine.beam;
            a.out_tokens[to] = (int64_t)(uint32_t)~(uint32_t)mine.key;
        }
    }
}

size_t aligned(size_t n) { return (n + 255) / 256 * 256; }

// (a range may begin inside a vector of four)
constexpr int kMostPart = kMostLogits - 4;
int parts_of(int64_t vocab) { return (int)((vocab + kMostPart - 1) / kMostPart); }

// The shared memory of the second kernel: at most k lists of k entries reach the bound, fewer lists than k are taken whole.  Lists that are kept there
// are read at once; beyond 8192 entries each is read as far as the bound.
constexpr int64_t kMostKept = 8192;
size_t merge_bytes(int64_t rows, int64_t parts, int64_t k) {
    const int64_t lists = rows * parts, reach = (lists < k ? lists : k) * k;
    return (size_t)(rows * 16 + lists * 8 + (lists * k <= kMostKept ? lists * k * 8 : 0) + reach * (int64_t)sizeof(Candidate));
}

// (what the kernel may ask for, whatever a call needs: calls of two threads set the same)
constexpr int kMostMemory = 200 * 1024;
static_assert(64 * 16 + kMostLists * 8 + kMostKept * 8 + kMostPicked * kMostPicked * sizeof(Candidate) <= kMostMemory);

int launch_merge(void (*kernel)(const Select), int64_t groups, size_t bytes, const Select& a, cudaStream_t st) {
    if (bytes > 40 * 1024) {                                                      // (48 KB with what the kernel declares)
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostMemory);
        if (err != cudaSuccess) return record_cuda_error(err);
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;                // (set up behind the first kernel)
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)groups);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = bytes;
    config.stream = st;
    config.attrs = &attr;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, a);
    count_launch();
    return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
}

// ---- reordering ------------------------------------------------------------------------------------------------

constexpr int kStatesPerLaunch = 256;

struct States {
    char* base[kStatesPerLaunch];
    int64_t group[kStatesPerLaunch], row[kStatesPerLaunch], bytes[kStatesPerLaunch], unit[kStatesPerLaunch];   // strides, a row's and a position's bytes
    unsigned first[kStatesPerLaunch + 1];             // blocks [first[k], first[k + 1]) move tensor k
    int used;
};

// A thread takes pieces of a row's bytes in every row of a group: all rows that something is taken from are read before the first
// is written, so the move needs no second copy of the states.  A thread has ROWS pieces on their way at once, of as many columns as the rows that move leave room for:
// 64 groups of 5 beams of which 2 move, 302 MB, 67 us with one column and 48 so, 0.96 of the copy rate.
constexpr int kColumns = 4;                           // of a block: so many times 256 pieces of a row

template <class T, int ROWS>
__global__ void __launch_bounds__(kThreads) reorder_kernel(const States s, const int64_t* parents, const int64_t* positions, int rows) {
    __shared__ int to[ROWS], from[ROWS];
    __shared__ int moving;
    int lo = 0, hi = s.used - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (s.first[mid] <= blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    after_previous();
    int64_t bytes = s.bytes[lo];
    constexpr int64_t kBlock = (int64_t)kThreads * kColumns * (int64_t)sizeof(T);
    const unsigned blocks = (unsigned)((bytes + kBlock - 1) / kBlock), block = blockIdx.x - s.first[lo], group = block / blocks;
    if (positions) {
        const int64_t n = *positions, most = bytes / s.unit[lo];
        bytes = (n < 0 ? 0 : n < most ? n : most) * s.unit[lo];
    }
    if (threadIdx.x == 0) moving = 0;
    __syncthreads();
    if (threadIdx.x < rows) {
        const int64_t p = parents[(int64_t)group * rows + threadIdx.x];
        if (p >= 0 && p < rows && p != threadIdx.x) {                             // (a parent that does not exist leaves the row as it is)
            const int at = atomicAdd(&moving, 1);
            to[at] = threadIdx.x;
            from[at] = (int)p;
        }
    }
    __syncthreads();
    const int n = moving;
    if (n == 0) return;
    int per = 1, shift = 0;                                                       // a column's pieces, to a power of two
    while (per < n) {
        per *= 2;
        ++shift;
    }
    const int columns = min(ROWS >> shift, kColumns);
    char* base = s.base[lo] + (int64_t)group * s.group[lo];
    const int64_t row = s.row[lo];
    for (int c0 = 0; c0 < kColumns; c0 += columns) {
        const int64_t at = (block - group * blocks) * kBlock + (int64_t)(c0 * kThreads + threadIdx.x) * (int64_t)sizeof(T);
        if (at >= bytes) return;
        T x[ROWS];
        const auto each = [&](auto&& one) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const int m = i & (per - 1), c = i >> shift;
                const int64_t here = at + (int64_t)c * (kThreads * (int)sizeof(T));
                if (m < n && c < columns && here < bytes) one(x[i], m, here);
            }
        };
        each([&](T& y, int m, int64_t here) { y = *reinterpret_cast<const T*>(base + from[m] * row + here); });
        each([&](T& y, int m, int64_t here) { *reinterpret_cast<T*>(base + to[m] * row + here) = y; });
    }
}

template <class T>
int launch_reorder(const States& s, unsigned blocks, const int64_t* parents, const int64_t* positions, int rows, cudaStream_t st) {
    const auto launch = [&](void (*kernel)(const States, const int64_t*, const int64_t*, int)) {
        return launch_behind(kernel, dim3(blocks), kThreads, st, s, parents, positions, rows);
    };
    if (rows <= 8) return launch(reorder_kernel<T, 8>);
    if (rows <= 16) return launch(reorder_kernel<T, 16>);
    return launch(reorder_kernel<std::conditional_t<sizeof(T) == 16, uint32_t, T>, 64>);
}

}  // namespace
}  // namespace pamk

extern "C" {

size_t pamk_beam_select_workspace_bytes(int64_t groups, int64_t rows, int64_t vocab, int64_t k) {
    using namespace pamk;
    if (groups <= 0 || rows <= 0 || vocab <= 0 || vocab > INT32_MAX - 2 * kMostLogits || k <= 0 || k > kMostPicked) return 0;
    const size_t lists = (size_t)(groups * rows) * parts_of(vocab);
    return aligned(lists * 8) + aligned(lists * 4) + aligned(lists * k * 8);
}

int pamk_beam_select(const float* logits, const float* scores, const unsigned char* banned, float* out_scores, int64_t* out_beams,
                     int64_t* out_tokens, int64_t groups, int64_t rows, int64_t vocab, int64_t k, int64_t logits_group, int64_t logits_row,
                     int64_t banned_group, int64_t banned_row, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace pamk;
    if (groups < 0 || rows < 1 || vocab < 1 || k < 1) return PAMK_ERR_ARG;
    if (rows > kMostPicked || k > kMostPicked || vocab > INT32_MAX - 2 * kMostLogits || k > rows * vocab) return PAMK_ERR_SIZE;
    if (groups == 0) return PAMK_OK;
    if (!logits || !scores || !out_scores || !out_beams || !out_tokens) return PAMK_ERR_ARG;
    const int64_t parts = parts_of(vocab), lists = rows * parts;
    if (lists > kMostLists || groups > INT32_MAX / lists) return PAMK_ERR_SIZE;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < pamk_beam_select_workspace_bytes(groups, rows, vocab, k))
        return PAMK_ERR_WORKSPACE;
    cudaStream_t st = (cudaStream_t)stream;
    Select a{};
    a.logits = logits; a.scores = scores; a.banned = banned;
    a.x_group = logits_group; a.x_row = logits_row; a.ban_group = banned_group; a.ban_row = banned_row;
    a.rows = (int)rows; a.vocab = (int)vocab; a.k = (int)k; a.parts = (int)parts;
    a.part = (int)(((vocab + parts - 1) / parts + 3) / 4 * 4);
    char* ws = static_cast<char*>(workspace);
    a.sums = reinterpret_cast<double*>(ws);
    ws += aligned((size_t)(groups * lists) * 8);
    a.shifts = reinterpret_cast<float*>(ws);
    ws += aligned((size_t)(groups * lists) * 4);
    a.lists = reinterpret_cast<unsigned long long*>(ws);
    a.out_scores = out_scores; a.out_beams = out_beams; a.out_tokens = out_tokens;
    const int status = launch_behind(pick_kernel, dim3((unsigned)(groups * rows), (unsigned)parts), kThreads, st, a);
    if (status != PAMK_OK) return status;
    return lists * k <= kMostKept ? launch_merge(merge_kernel<true>, groups, merge_bytes(rows, parts, k), a, st)
                                  : launch_merge(merge_kernel<false>, groups, merge_bytes(rows, parts, k), a, st);
}

int pamk_reorder_states(void* const* states, const int64_t* group_bytes, const int64_t* row_bytes, const int64_t* moved_bytes,
                        const int64_t* position_bytes, int count, const int64_t* parents, const int64_t* positions, int64_t groups, int64_t rows,
                        void* stream) {
    using namespace pamk;
    if (count < 0 || groups < 0 || rows < 1) return PAMK_ERR_ARG;
    if (count == 0 || groups == 0) return PAMK_OK;
    if (!states || !group_bytes || !row_bytes || !moved_bytes || !position_bytes || !parents) return PAMK_ERR_ARG;
    if (rows > kMostPicked) return PAMK_ERR_SIZE;
    for (int i = 0; i < count; ++i)
        if (moved_bytes[i] < 0 || (moved_bytes[i] && !states[i]) || position_bytes[i] < 1) return PAMK_ERR_ARG;
    // per kind of piece (16 bytes, 4, 1): the tensors whose rows consist of such pieces
    // (beyond 16 rows a thread holds no 16 bytes of each)
    for (int kind = rows > 16 ? 1 : 0; kind < 3; ++kind) {
        const int64_t piece = kind == 0 ? 16 : kind == 1 ? 4 : 1;
        const auto divides = [&](int i, int64_t by) {
            return (reinterpret_cast<uintptr_t>(states[i]) % by == 0 && group_bytes[i] % by == 0 && row_bytes[i] % by == 0 && moved_bytes[i] % by == 0 &&
                    position_bytes[i] % by == 0);
        };
        int i = 0;
        while (i < count) {
            States s{};
            uint64_t blocks = 0;
            for (; i < count && s.used < kStatesPerLaunch; ++i) {
                if (!moved_bytes[i] || (kind > 0 && rows <= 16 && divides(i, 16)) || (kind > 1 && divides(i, 4)) || !divides(i, piece)) continue;
                const int64_t block = (int64_t)kThreads * kColumns * piece;
                const uint64_t more = (uint64_t)((moved_bytes[i] + block - 1) / block) * (uint64_t)groups;
                if (more > INT32_MAX) return PAMK_ERR_SIZE;
                if (blocks + more > INT32_MAX) break;
                const int n = s.used++;
                s.base[n] = static_cast<char*>(states[i]);
                s.group[n] = group_bytes[i]; s.row[n] = row_bytes[i]; s.bytes[n] = moved_bytes[i]; s.unit[n] = position_bytes[i];
                s.first[n] = (unsigned)blocks;
                blocks += more;
                s.first[n + 1] = (unsigned)blocks;
            }
            if (!s.used) continue;
            cudaStream_t st = (cudaStream_t)stream;
            const int status = kind == 0   ? launch_reorder<uint4>(s, (unsigned)blocks, parents, positions, (int)rows, st)
                               : kind == 1 ? launch_reorder<uint32_t>(s, (unsigned)blocks, parents, positions, (int)rows, st)
                                           : launch_reorder<unsigned char>(s, (unsigned)blocks, parents, positions, (int)rows, st);
            if (status != PAMK_OK) return status;
        }
    }
    return PAMK_OK;
}

}
