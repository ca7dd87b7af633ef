// Sampling: one token of every row of logits, drawn by a uniform number that the caller gives.
//
//     x_j = pad(logit_j, temperature)    t_j = pam(x_j, log2 e) = i_j + f_j  (i whole, 0 <= f < 1)
//     w_j = floor(2^(44 - d_j) (1 + f'_j))     d_j = max i - i_j,   f' = f rounded down to steps of 2^-23
// The weights w are the PAM exponentials in units of 2^-44 of the row's greatest power of two, as whole numbers: their sums are exact in any order, so that
// what is drawn follows from the logits alone and no rounding, split or order of atomics shows.  (2^18 of them stay below 2^63.)
// Tokens are ordered by 2^-d (1 + f'), equal ones by their number.  In that order stay
//     the first top_k;  of these, those before which less than top_p of their weights lies;  of these, those of at least min_p times the first one's weight;
// and the token is the first in the vocabulary whose weights up to and with it exceed u times all that stay.  (These shares are ordinary products of whole
// numbers: a PAM product would favour some tokens.)  Its score is x - pad(M + log2(S), log2 e), the PAM log-softmax over all of the row's tokens (pam/pam_ops.py:331-347),
// from a sum S of all bits of the exponentials down to 2^-62 and a logarithm and a quotient in 64 bits.
//
// An exponential is kept as the pattern of the float e = 2^-d (1 + f'), taken from that of the largest: a key that is smaller for larger weights, so that
// "in order" is the order of (key, number).  Sums of weights are sums of e in doubles that start at 2^8 and are rounded down: there a unit is 2^-44, and adding e
// adds floor(2^44 e) units, without an error, until they reach 2^8.
//
// A row belongs to a cluster of up to eight CTAs, each of which keeps its part in shared memory: the t of its tokens, then their keys.  A warp has neighbouring
// tokens, of which a thread has the same four at a time from loading to drawing.  The logits are read once.  What stays is cut off at one token, found as follows:
//   top-k   each warp's q-th best of its lanes' best tokens, where q of each of w warps are k at least, bounds the k-th best of all; the few tokens as good as the
//           bound go to a list in the first CTA, where each counts those before it and their weights, and which draws from them;
//   top-p   each warp sets aside its tokens that are not too light to matter (most often few), whose weights go into a histogram of as many parts as a CTA has
//           threads; the few tokens of the part that holds the cut go to the list.  (More than a list holds: the part is divided again.)
// Bound by the row's few common numbers, each of which is a barrier of the cluster, and by instructions (52 per token without a cut): 256 rows of 151643 tokens 124 us,
// of which 53 for loading alone in this form, 23 for the largest t, 27 for keys and sums; top-k 183, top-p 250.  640 rows of 10000: 22, 37, 37; one row of 10000: 8, 12, 14.
#include <cooperative_groups.h>

#include "common.cuh"
#include "pam_scalar.cuh"

namespace pamk {
namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMasked = -1e30f;                     // a logit as low as this is masked
constexpr int kMostCtas = 8, kMostKeys = 32768;       // of a cluster; of a CTA
constexpr uint32_t kOut = 0xffffffffu;                // the key of a token without weight
constexpr uint32_t kTop = 0x3fffffffu;                // key + pattern
constexpr uint32_t kEnd = 45u << 23;                  // keys with a weight are below
constexpr int kNumberBits = 18;
static_assert(kMostCtas * kMostKeys == 1 << kNumberBits);
typedef unsigned long long u64;

struct Sample {
    const float *logits, *uniform;
    const unsigned char* banned;                      // or null
    int64_t x_row, ban_row;
    const float *temperatures, *top_ps, *min_ps;      // one for each row, or null: the same for all
    const int64_t* top_ks;
    float temperature, top_p, min_p;
    int64_t top_k;
    int vocab, part;                                  // a CTA's tokens
    int vocab_bits;                                   // of the power of two next to the vocabulary from above
    int64_t* tokens;
    float* scores;
};

constexpr int kListed = 256;

template <int THREADS>
struct Shared {
    static constexpr int kWarps = THREADS / 32, kFew = THREADS;
    union {
        struct { u64 list[kListed], weights[kListed]; };
        struct { uint32_t count[THREADS], low[THREADS], high[THREADS]; };             // of each part: keys, and the sum of their weights' digits by 12 bits
    };
    uint16_t few[kWarps][kFew];                       // slots of a warp's keys in the range of a search
    // what the other CTAs of the cluster read
    float all, ok;
    int bad;
    double sums[kWarps], banned_sums[kWarps];
    u64 parts[kWarps], staying[2][kWarps];            // weights of the warps: of all, of what stays
    uint32_t live[kWarps], bounds[kWarps], ties[kWarps];
    uint32_t listed;
    u64 cut, kept;
    // within the CTA
    float warp_all[kWarps], warp_ok[kWarps];
    u64 every[kWarps * kMostCtas];                    // all warps' of the cluster
    double every_sum[kWarps * kMostCtas];
    uint32_t every_bound[kWarps * kMostCtas], bound;
    u64 scan[kWarps];
    uint32_t scan_count[kWarps];
    uint32_t part, part_count, less_count;            // what a histogram gave
    u64 less_weight;
};

// Where the threads of a cluster wait for one another.
struct Team {
    cg::cluster_group cluster;
    int ctas;
    __device__ void wait() {
        if (ctas == 1) __syncthreads(); else cluster.sync();
    }
    // In two halves: this CTA reads no more of the others; none reads of this one.
    __device__ void done() {
        if (ctas > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");
    }
    __device__ void all_done() {
        if (ctas > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
    }
    template <class S>
    __device__ S& of(S& sh, int c) { return ctas == 1 ? sh : *cluster.map_shared_rank(&sh, c); }
};

// A normal float >= 0 of this pattern as a double (the conversion instruction has a quarter of the rate).
__device__ __forceinline__ double widened(uint32_t bits) { return __hiloint2double((int)((bits >> 3) + (896u << 20)), (int)(bits << 29)); }
__device__ __forceinline__ double value_of(uint32_t key) { return widened(kTop - key); }

__device__ __forceinline__ u64 weight_of(uint32_t key) {
    const uint32_t d = key >> 23, m = 0x800000u | (~key & 0x7fffffu);
    return d <= 21u ? (u64)m << (21u - d) : (u64)(m >> min(d - 21u, 31u));
}

// The digits of a key's weight without its shift, which is the same for all keys of an octave.
__device__ __forceinline__ uint32_t digits(uint32_t key) {
    const uint32_t d = key >> 23, m = 0x800000u | (~key & 0x7fffffu);
    return d <= 21u ? m : m >> (d - 21u);
}

// Sums of weights.
struct Units {
    double sum = 256.0;
    __device__ void add(double e) { sum = __dadd_rd(sum, e); }
    __device__ u64 get() const { return (u64)__double_as_longlong(sum) & 0xfffffffffffffull; }
};

// floor and the rest of fraction 2^-24 total
struct Share { u64 whole; bool rest; };
__device__ __forceinline__ Share share(uint32_t fraction, u64 total) {
    const u64 low = total * fraction;
    return {__umul64hi(total, fraction) << 40 | low >> 24, (low & 0xffffffu) != 0};
}
__device__ __forceinline__ u64 share_up(uint32_t fraction, u64 total) {
    const Share s = share(fraction, total);
    return s.whole + s.rest;
}
// A fraction in steps of 2^-24, NaN as 0.
__device__ __forceinline__ uint32_t steps(float f, uint32_t most) { return f > 0.0f ? min((uint32_t)fminf(f * 16777216.0f, 16777216.0f), most) : 0u; }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {      // by 22 bits, whose sums have 27
    const u64 low = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x3fffffu), mid = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 22) & 0x3fffffu);
    return low + (mid << 22) + ((u64)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 44)) << 44);
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
__device__ __forceinline__ u64 warp_upto(u64 v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const u64 w = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += w;
    }
    return v;
}

// pad(M + log2(S), log2 e) in 64 bits, log2(2^i (1 + f)) = i + f, S >= 1
__device__ double log_sum(double shift, double total) {
    const long long bits = __double_as_longlong(total);
    const double fraction = __longlong_as_double((bits & 0xfffffffffffffll) | 0x3ff0000000000000ll) - 1.0;
    const double log2 = shift + ((double)((bits >> 52) - 1023) + fraction), by = (double)kLog2e;
    if (log2 == 0.0) return 0.0;                      // (the range rule's only case: any other is 2^-53 at least)
    return __longlong_as_double(__double_as_longlong(log2) - __double_as_longlong(by) + 0x3ff0000000000000ll);
}

// 2^e for whole e <= 1 (0 far below)
__device__ __forceinline__ double power_of(float e) { return e >= -1000.0f ? __longlong_as_double((long long)((int)e + 1023) << 52) : 0.0; }

// t = pam(pad(x, temperature), log2 e): one sum of patterns where x lies far from what the range rule cuts off, in which case no value in between does either.
struct Scaling {
    float temperature;
    uint32_t low, span;                               // twice the pattern of the least such |x|, and how far the greatest is from there
    int32_t shift;
    __device__ explicit Scaling(float t) : temperature(t) {
        // |x| / temperature from 2^-100 to 2^100, |x| normal and below what is masked
        const int32_t bits = f2i(t);
        const uint32_t least = (uint32_t)max(bits - (100 << 23), 1 << 23), most = (uint32_t)min((int64_t)bits + (100 << 23), (int64_t)f2i(-kMasked) - 1);
        low = 2u * least;
        span = most > least ? 2u * (most - least) : 0u;
        shift = f2i(kLog2e) - bits;
    }
    __device__ __forceinline__ uint32_t beyond(float x) const { return 2u * (uint32_t)f2i(x) - low; }              // below `span` there
    __device__ __forceinline__ float plainly(float x) const { return i2f(iadd(f2i(x), shift)); }
    __device__ __noinline__ float any(float x) const { return x <= kMasked ? -INFINITY : mul(div(x, temperature, 0), kLog2e, 0); }
};

// What is asked of a row.
struct Wanted { float top_p; uint32_t min_p, uniform; };

// A search for the token at which a count or a weight is reached, in the order of (key, number).
template <int THREADS>
struct Search {
    static constexpr int kWarps = THREADS / 32;
    typedef Shared<THREADS> Sh;
    Sh& sh;
    Team& team;
    const uint32_t* keys;                             // of the CTA's slots
    int first, last, lane, warp;                      // the warp's quads; the lane's are every 32nd
    int begin, rank;                                  // the number of slot 0 (it may be before the part); the CTA's rank
    int few = -1;                                     // how many of its keys the warp has set aside

    __device__ __forceinline__ uint4 quad(int q) const { return q < last ? reinterpret_cast<const uint4*>(keys)[q] : make_uint4(kOut, kOut, kOut, kOut); }

    template <class F>
    __device__ __forceinline__ void each(F&& f) const {               // f(key, slot) for all
        for (int q = first + lane; q < last; q += 32) {
            const uint4 k = reinterpret_cast<const uint4*>(keys)[q];
            f(k.x, q * 4);
            f(k.y, q * 4 + 1);
            f(k.z, q * 4 + 2);
            f(k.w, q * 4 + 3);
        }
    }
    template <class F>
    __device__ __forceinline__ void each_aside(F&& f) const {         // f(key, slot) for those set aside
        for (int i = lane; i < few; i += 32) {
            const int slot = sh.few[warp][i];
            f(keys[slot], slot);
        }
    }
    __device__ __forceinline__ u64 composite(uint32_t key, int slot) const { return (u64)key << kNumberBits | (uint32_t)(begin + slot); }

    // The sum of a value of all warps of the cluster, and of those before this one.  There is a barrier within.
    template <class F>
    __device__ u64 total_of(F&& of, u64* before) {
        const int warps = team.ctas * kWarps, t = threadIdx.x;
        if (t < warps) sh.every[t] = of(t / kWarps, t % kWarps);
        __syncthreads();
        u64 total = 0ull, less = 0ull;
        for (int w = lane; w < warps; w += 32) {
            total += sh.every[w];
            if (w < rank * kWarps + warp) less += sh.every[w];
        }
        *before = warp_sum(less);
        return warp_sum(total);
    }

    // The weight of all tokens up to `cut`; `own` is this warp's and `before` that of the warps before.  `turn` alternates from call to call.
    __device__ u64 weigh(u64 cut, int turn, u64* own, u64* before) {
        Units stay;
        if (few >= 0) {                               // (all up to a cut by weight)
            each_aside([&](uint32_t key, int slot) {
                if (composite(key, slot) <= cut) stay.add(value_of(key));
            });
        } else {
            const uint32_t cut_key = (uint32_t)(cut >> kNumberBits);
            const int cut_slot = (int)((uint32_t)cut & ((1u << kNumberBits) - 1u)) - begin;
            each([&](uint32_t key, int slot) {
                if (key < cut_key || (key == cut_key && slot <= cut_slot)) stay.add(value_of(key));
            });
        }
        *own = warp_sum(stay.get());
        if (lane == 0) sh.staying[turn][warp] = *own;
        team.wait();
        return total_of([&](int c, int w) { return team.of(sh, c).staying[turn][w]; }, before);
    }

    // What the lanes before this one have, and (in *all) the warp.
    __device__ __forceinline__ int before_lane(int mine, int* all) const {
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        *all = __shfl_sync(0xffffffffu, upto, 31);
        return upto - mine;
    }

    // Sets aside the warp's keys up to `most`, if they are few.
    __device__ void set_aside(uint32_t most) {
        int mine = 0;
        each([&](uint32_t key, int) { mine += key <= most; });
        int place = before_lane(mine, &few);
        if (few > Sh::kFew) {
            few = -1;
            return;
        }
        each([&](uint32_t key, int slot) {
            if (key <= most) sh.few[warp][place++] = (uint16_t)slot;
        });
        __syncwarp();
    }

    // The keys in [low, low + THREADS 2^shift) in THREADS parts: sh.part is the one in which `target` is reached (by count, or by weight), sh.part_count has that many
    // keys, and sh.less_* lies before it.  Parts are within an octave.
    __device__ void divide(uint32_t low, int shift, bool by_count, u64 target, uint32_t less_count, u64 less_weight) {
        const int t = threadIdx.x;
        sh.count[t] = sh.low[t] = sh.high[t] = 0u;
        __syncthreads();
        const auto look = [&](uint32_t key, int) {
            const uint32_t part = (key - low) >> shift;
            if (part >= (uint32_t)THREADS) return;
            atomicAdd(&sh.count[part], 1u);
            if (!by_count) {
                const uint32_t m = digits(key);
                atomicAdd(&sh.low[part], m & 0xfffu);
                atomicAdd(&sh.high[part], m >> 12);
            }
        };
        few >= 0 ? each_aside(look) : each(look);
        team.wait();
        uint32_t count = 0u;
        u64 weight = 0ull;
#pragma unroll
        for (int c = 0; c < kMostCtas; ++c) {
            if (c >= team.ctas) break;
            const Sh& other = team.of(sh, c);
            count += other.count[t];
            if (!by_count) weight += (u64)other.low[t] + ((u64)other.high[t] << 12);
        }
        const uint32_t d = (low + ((uint32_t)t << shift)) >> 23;
        if (d <= 21u) weight <<= 21u - d;
        const u64 weight_upto = by_count ? 0ull : warp_upto(weight);
        uint32_t count_upto = count;
#pragma unroll
        for (int apart = 1; apart < 32; apart <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, count_upto, apart);
            if (lane >= apart) count_upto += v;
        }
        if (lane == 31) {
            sh.scan[warp] = weight_upto;
            sh.scan_count[warp] = count_upto;
        }
        __syncthreads();
        u64 before = less_weight + weight_upto - weight;
        uint32_t count_before = less_count + count_upto - count;
        for (int w = 0; w < warp; ++w) {
            before += sh.scan[w];
            count_before += sh.scan_count[w];
        }
        const u64 from = by_count ? count_before : before, to = from + (by_count ? count : weight);
        if (from < target && target <= to) {
            sh.part = t;
            sh.part_count = count;
            sh.less_count = count_before;
            sh.less_weight = before;
        }
        team.wait();                                  // (the histogram may be written anew)
    }

    // The tokens with keys from `low` to `high` to the first CTA's list; false where there are too many.  sh.listed is 0 before.  (best: no key of the lane is smaller.)
    __device__ bool gather(uint32_t low, uint32_t high, uint32_t best) {
        Sh& head = team.of(sh, 0);
        const bool aside = few >= 0, any = aside || best <= high;
        int mine = 0;
        const auto count = [&](uint32_t key, int) { mine += key - low <= high - low; };
        if (any) aside ? each_aside(count) : each(count);
        int all;
        int place = before_lane(mine, &all);
        if (all > 0) {
            int at = 0;
            if (lane == 0) at = (int)atomicAdd(&head.listed, (uint32_t)all);
            place += __shfl_sync(0xffffffffu, at, 0);
            const auto put = [&](uint32_t key, int slot) {
                if (key - low > high - low) return;
                if (place < kListed) head.list[place] = composite(key, slot);
                ++place;
            };
            if (mine > 0) aside ? each_aside(put) : each(put);
        }
        team.wait();
        return head.listed <= kListed;
    }

    // A token of the list: several neighbouring lanes may have it.
    struct Listed { u64 own, weight; bool one; };     // one: of these lanes
    __device__ Listed of_list(int n, int& split) {
        const int t = threadIdx.x;
        for (int i = t; i < n; i += THREADS) sh.weights[i] = weight_of((uint32_t)(sh.list[i] >> kNumberBits));
        __syncthreads();
        split = 1;
        while (split < 32 && n * split * 2 <= THREADS) split *= 2;
        const int i = t / split;
        return {i < n ? sh.list[i] : 0ull, i < n ? sh.weights[i] : 0ull, i < n && t % split == 0};
    }
    // How many tokens of the list a test holds for, and their weights.
    template <class F>
    __device__ void count_list(int n, int split, F&& before, uint32_t* count, u64* weight) {
        uint32_t c = 0u;
        u64 w = 0ull;
        if ((int)threadIdx.x / split < n)
            for (int j = threadIdx.x % split; j < n; j += split)
                if (before(sh.list[j])) {
                    ++c;
                    w += sh.weights[j];
                }
        for (int d = split / 2; d > 0; d >>= 1) {
            c += __shfl_xor_sync(0xffffffffu, c, d);
            w += __shfl_xor_sync(0xffffffffu, w, d);
        }
        *count = c;
        *weight = w;
    }

    // In the first CTA: sets sh.cut to the list's token at which the weight `target` is reached, less_weight before the list (by_count: the target-th, less_count before).
    __device__ void pick(bool by_count, u64 target, uint32_t less_count, u64 less_weight) {
        const int n = (int)sh.listed;
        int split;
        const Listed l = of_list(n, split);
        uint32_t count;
        u64 before;
        count_list(n, split, [&](u64 other) { return other < l.own; }, &count, &before);
        before += less_weight;
        if (l.one && (by_count ? less_count + count + 1 == target : before < target && target <= before + l.weight)) sh.cut = l.own;
    }

    // In the first CTA: draws from the list, which holds the k best tokens and maybe others.  The token's number is then in sh.cut.
    __device__ void draw(int k, const Wanted& wanted, u64 top_weight) {
        constexpr u64 kNumbers = (1ull << kNumberBits) - 1;
        const int n = (int)sh.listed;
        int split;
        const Listed l = of_list(n, split);
        uint32_t count;
        u64 before;
        count_list(n, split, [&](u64 other) { return other < l.own; }, &count, &before);
        if (l.one && (int)count == k - 1) sh.kept = before + l.weight;
        __syncthreads();
        const u64 limit = wanted.top_p < 1.0f ? max(share_up(steps(wanted.top_p, 0xffffffu), sh.kept), 1ull) : ~0ull;
        const bool stays = (int)count < k && before < limit && l.weight >= share_up(wanted.min_p, top_weight);
        __syncthreads();
        if (l.one && !stays) sh.weights[threadIdx.x / split] = 0ull;
        __syncthreads();
        // those that stay, in order of their numbers
        u64 total;
        count_list(n, split, [&](u64) { return true; }, &count, &total);
        count_list(n, split, [&](u64 other) { return (other & kNumbers) < (l.own & kNumbers); }, &count, &before);
        const u64 drawn = share(wanted.uniform, total).whole;
        if (l.one && stays && before <= drawn && drawn < before + l.weight) sh.cut = l.own & kNumbers;
        __syncthreads();
    }

    // The cut, of which is known that it is one of the tokens with these keys; false where there are too many.
    __device__ bool listed(uint32_t low, uint32_t high, bool by_count, u64 target, uint32_t less_count, u64 less_weight, u64* cut) {
        const bool fits = gather(low, high, low);
        if (fits && rank == 0) pick(by_count, target, less_count, less_weight);
        team.wait();
        *cut = team.of(sh, 0).cut;
        if (rank == 0 && threadIdx.x == 0) sh.listed = 0u;
        team.wait();
        return fits;
    }

    // The r-th token, by number, of those with this key.
    __device__ u64 equal_one(uint32_t key, u64 r) {
        uint32_t own = 0u;
        each([&](uint32_t k, int) { own += k == key; });
        own = __reduce_add_sync(0xffffffffu, own);
        if (lane == 0) sh.ties[warp] = own;
        team.wait();
        u64 before;
        total_of([&](int c, int w) { return (u64)team.of(sh, c).ties[w]; }, &before);
        if (before < r && r <= before + own) {
            uint32_t need = (uint32_t)(r - before);
            for (int q = first + lane; q - lane < last; q += 32) {
                const uint4 k = quad(q);
                const uint32_t is = (k.x == key) | (k.y == key) << 1 | (k.z == key) << 2 | (k.w == key) << 3;
                uint32_t upto = __popc(is);
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += v;
                }
                const uint32_t reached = __ballot_sync(0xffffffffu, upto >= need);
                if (reached) {
                    if (lane == __ffs(reached) - 1) {
                        uint32_t left = is;
                        for (uint32_t i = upto - __popc(is) + 1; i < need; ++i) left &= left - 1;
                        team.of(sh, 0).cut = composite(key, q * 4 + __ffs(left) - 1);
                    }
                    break;
                }
                need -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        team.wait();
        const u64 cut = team.of(sh, 0).cut;
        team.wait();
        return cut;
    }

    // The cut, which is among the keys up to `most`.
    __device__ u64 find(bool by_count, u64 target, uint32_t most) {
        constexpr int kBits = THREADS == 512 ? 9 : 8;
        static_assert(1 << kBits == THREADS);
        int shift = 0;
        while (most >> shift >= (uint32_t)THREADS) ++shift;           // (at most 21: parts of a quarter of an octave)
        few = -1;
        if (!by_count) set_aside(most);
        uint32_t low = 0u, less_count = 0u;
        u64 less_weight = 0ull;
        for (;; shift -= kBits) {
            const int by = max(shift, 0);
            divide(low, by, by_count, target, less_count, less_weight);
            low += sh.part << by;
            less_count = sh.less_count;
            less_weight = sh.less_weight;
            const uint32_t left = sh.part_count;
            __syncthreads();
            u64 cut;
            if (left <= kListed && listed(low, low + (1u << by) - 1u, by_count, target, less_count, less_weight, &cut)) return cut;
            if (by == 0) {
                const u64 each_weight = weight_of(low);
                return equal_one(low, by_count ? target - less_count : (target - less_weight + each_weight - 1) / each_weight);
            }
        }
    }
};

// What a thread's tokens add up to.
struct Sums {
    Units units;                                      // of the weights
    double sum = 0.0;                                 // of the e
    float rest = 0.0f;                                // of what f' leaves of f, where t has bits below 2^-23, times 2^floor t
    double banned = 0.0;                              // of banned tokens' exponentials
    uint32_t best = kOut, live = 0u;
};

// t -> key.  A t far below the largest becomes an e below 2^-125, which is no weight and adds nothing.  NEAR: both shifts within 2^20, where a whole part is the low bits of a sum
// (the conversion instructions have a quarter of the rate of sums).
template <bool NEAR, bool BANNED, bool COUNT>
__device__ __forceinline__ uint32_t key_of(Sums& s, float t, float shift, float shift_all, bool out) {
    constexpr float kMagic = 12582912.0f;             // 3 2^22: its pattern's low nine bits are zeros
    const float v = NEAR ? fmaxf(t, shift - 126.0f) : fmaxf(t, -3e38f), placed = __fadd_rd(v, kMagic);
    const float whole = NEAR ? fadd(placed, -kMagic) : floorf(v), lin = __fadd_rd(1.0f, __fadd_rd(v, -whole));      // lin = 1 + f'
    // (f - f' = t - ((1 + f') + (floor t - 1)), to a part in 2^24 of itself; 0 where |t| >= 1)
    const float rest = NEAR || fabsf(v) < 1.0f ? fadd(v, -fadd(lin, fadd(whole, -1.0f))) : 0.0f;
    if (BANNED && out) {
        if (t > -INFINITY) s.banned += ((double)lin + (double)rest) * power_of(whole - shift_all);
        return kOut;
    }
    s.rest = __fmaf_rn(rest, __fmaf_rn(whole, 0.5f, 1.0f), s.rest);                  // (2^whole for 0 and -1)
    const uint32_t bits = NEAR ? (uint32_t)f2i(lin) + ((uint32_t)f2i(placed) << 23) - ((uint32_t)f2i(fadd(shift, kMagic)) << 23)
                               : (uint32_t)f2i(lin) - ((uint32_t)min((int)(shift - whole), 126) << 23);
    const double e = widened(bits);
    s.sum += e;
    s.units.add(e);
    const uint32_t key = kTop - bits < kEnd ? kTop - bits : kOut;
    if (COUNT) {
        s.best = min(s.best, key);
        s.live += key != kOut;
    }
    return key;
}

template <bool NEAR, bool BANNED, bool COUNT>
__device__ __forceinline__ void make_keys(Sums& sums, uint32_t* keys, const unsigned char* flags, int first, int last, float shift, float shift_all) {
#pragma unroll 2
    for (int q = first; q < last; q += 32) {
        const float4 v = reinterpret_cast<const float4*>(keys)[q];
        const uint32_t out = BANNED && flags ? flags[q] : 0u;
        const auto key = [&](float t, uint32_t bit) { return key_of<NEAR, BANNED, COUNT>(sums, t, shift, shift_all, out & bit); };
        reinterpret_cast<uint4*>(keys)[q] = make_uint4(key(v.x, 1u), key(v.y, 2u), key(v.z, 4u), key(v.w, 8u));
    }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) sample_kernel(const Sample a) {
    constexpr int kWarps = THREADS / 32;
    // (the e of a thread's tokens stay below 2^8 together)
    static_assert((kMostKeys / 512 * THREADS / 4 / THREADS + 2) * 4 * 2 < 256);
    extern __shared__ __align__(16) unsigned char memory[];
    Shared<THREADS>& sh = *reinterpret_cast<Shared<THREADS>*>(memory);
    uint32_t* keys = reinterpret_cast<uint32_t*>(memory + (sizeof(sh) + 15) / 16 * 16);
    unsigned char* flags = reinterpret_cast<unsigned char*>(keys + a.part + 4);       // four bits for each quad: banned
    Team team{cg::this_cluster(), 0};
    team.ctas = (int)team.cluster.num_blocks();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rank = team.ctas == 1 ? 0 : (int)team.cluster.block_rank();
    const int64_t row = blockIdx.x / team.ctas;
    const int begin = min(rank * a.part, a.vocab), n = min(a.part, a.vocab - begin);
    const unsigned char* banned = a.banned ? a.banned + row * a.ban_row + begin : nullptr;
    const float temperature = a.temperatures ? __ldg(a.temperatures + row) : a.temperature;
    const float top_p = a.top_ps ? __ldg(a.top_ps + row) : a.top_p, min_p = a.min_ps ? __ldg(a.min_ps + row) : a.min_p;
    const int64_t top_k = a.top_ks ? __ldg(reinterpret_cast<const long long*>(a.top_ks) + row) : a.top_k;
    const Wanted wanted{top_p, steps(min_p, 1u << 24), steps(__ldg(a.uniform + row), 0xffffffu)};
    const bool cut_by_k = top_k > 0 && top_k < a.vocab;
    const Scaling scaled(temperature);

    // slots of four at aligned addresses: the first one may begin before the part, the last one end behind it
    const float* part = a.logits + row * a.x_row + begin;
    const int phase = (int)((reinterpret_cast<uintptr_t>(part) >> 2) & 3);
    const float* slots = part - phase;
    const int quads = n > 0 ? (n + phase + 3) / 4 : 0, each = (quads + kWarps - 1) / kWarps, first = min(warp * each, quads), last = min(first + each, quads);
    if (t == 0) sh.listed = 0u;

    // the row's t, and the largest of all and of those that may be drawn
    float top_all = -INFINITY, top_ok = -INFINITY;
    uint32_t any_out = 0u;
    bool bad = !(temperature > 0.0f && temperature <= i2f(0x7f7fffff));
    constexpr int kAhead = 4;
    const int full_from = phase ? 1 : 0, full_to = max((n + phase) / 4, full_from);    // quads that are all the part's
    // A byte of flags for each of a quad's tokens.
    const auto flags_of = [&](int q) {
        const int s = q * 4 - phase;
        if (!banned) return 0u;
        if (s >= 4 && s + 8 <= n) {                   // (two aligned words hold the four)
            const uintptr_t at = reinterpret_cast<uintptr_t>(banned + s);
            const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
            return __funnelshift_r(__ldg(words), __ldg(words + 1), (uint32_t)(at & 3) * 8u);
        }
        uint32_t all = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (s + j >= 0 && s + j < n) all |= (uint32_t)__ldg(banned + s + j) << (8 * j);
        return all;
    };
    const auto scale = [&](int q, const float4& x, uint32_t flag) {
        float4 v;
        if (max(max(scaled.beyond(x.x), scaled.beyond(x.y)), max(scaled.beyond(x.z), scaled.beyond(x.w))) < scaled.span) {
            v = make_float4(scaled.plainly(x.x), scaled.plainly(x.y), scaled.plainly(x.z), scaled.plainly(x.w));
        } else {
            v = make_float4(scaled.any(x.x), scaled.any(x.y), scaled.any(x.z), scaled.any(x.w));
            bad = bad || v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w;
        }
        const float most = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
        top_all = fmaxf(top_all, most);
        if (banned) {
            uint32_t out = 0u;
            if (flag) out = ((flag & 0xffu) != 0) | ((flag & 0xff00u) != 0) << 1 | ((flag & 0xff0000u) != 0) << 2 | ((flag & 0xff000000u) != 0) << 3;
            flags[q] = (unsigned char)out;
            any_out |= out;
            top_ok = fmaxf(top_ok, !out ? most : fmaxf(fmaxf(out & 1u ? -INFINITY : v.x, out & 2u ? -INFINITY : v.y), fmaxf(out & 4u ? -INFINITY : v.z, out & 8u ? -INFINITY : v.w)));
        }
        reinterpret_cast<float4*>(keys)[q] = v;
    };
    const auto edge = [&](int q) {
        const int s = q * 4 - phase;
        const auto at = [&](int i) { return i >= 0 && i < n ? __ldcs(part + i) : -INFINITY; };
        scale(q, make_float4(at(s), at(s + 1), at(s + 2), at(s + 3)), flags_of(q));
    };
    {
        int q = first + lane;
        if (q < full_from && q < last) {
            edge(q);
            q += 32;
        }
        const int stop = min(last, full_to);
        const float4* from = reinterpret_cast<const float4*>(slots);
        for (; q + 32 * (kAhead - 1) < stop; q += 32 * kAhead) {
            float4 x[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) x[k] = __ldcs(from + q + 32 * k);
            uint32_t flag[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) flag[k] = flags_of(q + 32 * k);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) scale(q + 32 * k, x[k], flag[k]);
        }
        float4 x[kAhead - 1];
#pragma unroll
        for (int k = 0; k < kAhead - 1; ++k)
            if (q + 32 * k < stop) x[k] = __ldcs(from + q + 32 * k);
#pragma unroll
        for (int k = 0; k < kAhead - 1; ++k)
            if (q + 32 * k < stop) scale(q + 32 * k, x[k], flags_of(q + 32 * k));
        if (full_to >= first && full_to < last && (full_to - first) % 32 == lane) edge(full_to);
    }
    top_all = warp_max(top_all);
    top_ok = banned ? warp_max(top_ok) : top_all;
    if (lane == 0) {
        sh.warp_all[warp] = top_all;
        sh.warp_ok[warp] = top_ok;
    }
    const int any_bad = __syncthreads_or(bad);
    top_all = warp_max(lane < kWarps ? sh.warp_all[lane] : -INFINITY);
    top_ok = warp_max(lane < kWarps ? sh.warp_ok[lane] : -INFINITY);
    int no_token = any_bad;
    if (team.ctas > 1) {
        if (t == 0) {
            sh.all = top_all;
            sh.ok = top_ok;
            sh.bad = any_bad;
        }
        team.wait();
        const Shared<THREADS>& other = team.of(sh, lane < team.ctas ? lane : 0);
        top_all = warp_max(other.all);
        top_ok = warp_max(other.ok);
        no_token = __any_sync(0xffffffffu, other.bad);
    }
    if (no_token || !(top_ok > -INFINITY)) {                                          // (all CTAs of the cluster alike)
        if (rank == 0 && t == 0) {
            a.tokens[row] = -1;
            a.scores[row] = -INFINITY;
        }
        team.wait();
        return;
    }
    const float shift_all = floorf(top_all), shift = floorf(top_ok);
    const float lin_top = __fadd_rd(1.0f, __fadd_rd(top_ok, -shift));
    const uint32_t top_key = kTop - (uint32_t)f2i(lin_top);

    // keys in place of the t, and the sums
    Sums sums;
    const bool bans = banned && __any_sync(0xffffffffu, any_out);      // (one of the warp's tokens)
    if (!bans) flags = nullptr;
    if (fmaxf(fabsf(shift), fabsf(shift_all)) < 1048576.0f) {
        if (bans)
            cut_by_k ? make_keys<true, true, true>(sums, keys, flags, first + lane, last, shift, shift_all) : make_keys<true, true, false>(sums, keys, flags, first + lane, last, shift, shift_all);
        else
            cut_by_k ? make_keys<true, false, true>(sums, keys, flags, first + lane, last, shift, shift_all) : make_keys<true, false, false>(sums, keys, flags, first + lane, last, shift, shift_all);
    } else {
        make_keys<false, true, true>(sums, keys, flags, first + lane, last, shift, shift_all);
    }
    u64 weight = warp_sum(sums.units.get());
    const double sum = warp_sum(sums.sum + (shift >= -1.0f ? (double)sums.rest * power_of(-shift) : 0.0));     // (|t| < 1 only above)
    const double banned_sum = bans ? warp_sum(sums.banned) : 0.0;
    if (lane == 0) {
        sh.parts[warp] = weight;
        sh.sums[warp] = sum;
        sh.banned_sums[warp] = banned_sum;
    }
    // of the lanes' best the q-th best, where q of each warp are k at least
    const int warps = team.ctas * kWarps, q = cut_by_k ? (int)((min(top_k, (int64_t)kListed) + warps - 1) / warps) : 0;
    const bool bounded = cut_by_k && top_k <= kListed / 2 && q <= 32;
    if (cut_by_k) {
        const uint32_t live = __reduce_add_sync(0xffffffffu, sums.live);
        if (lane == 0) sh.live[warp] = live;
        if (bounded) {
            int before = 0;
#pragma unroll
            for (int d = 0; d < 32; ++d) {
                const uint32_t other = __shfl_sync(0xffffffffu, sums.best, d);
                before += other < sums.best || (other == sums.best && d < lane);
            }
            if (before == q - 1) sh.bounds[warp] = sums.best;
        }
    }
    team.wait();
    Search<THREADS> search{sh, team, keys, first, last, lane, warp, begin - phase, rank};
    if (t < warps) {
        const Shared<THREADS>& other = team.of(sh, t / kWarps);
        sh.every_sum[t] = other.sums[t % kWarps] * power_of(shift - shift_all) + (banned ? other.banned_sums[t % kWarps] : 0.0);
        if (bounded) sh.every_bound[t] = other.bounds[t % kWarps];
    }
    u64 upto, total = search.total_of([&](int c, int w) { return team.of(sh, c).parts[w]; }, &upto);
    const auto all_sums = [&] {                       // (of a whole warp)
        double all = 0.0;
        for (int w = lane; w < warps; w += 32) all += sh.every_sum[w];
        return warp_sum(all);
    };
    const auto answer = [&](int token, double all) {
        const float chosen = div(__ldg(part + (token - begin)), temperature, 0);
        a.tokens[row] = token;
        a.scores[row] = (float)((double)chosen - log_sum((double)shift_all, all));
    };

    // what stays
    u64 cut = ~0ull;
    bool weighed = true;                              // `total`, `weight` and `upto` are of what stays
    int turn = 0;
    if (cut_by_k) {
        // (fewer than k may have a weight: then all of these stay)
        uint32_t live = 0u;
        for (int w = lane; w < warps; w += 32) live += team.of(sh, w / kWarps).live[w % kWarps];
        live = __reduce_add_sync(0xffffffffu, live);
        if (top_k < live) {
            if (bounded) {
                // of the warps' the one that as many reach as make k
                const int enough = (int)((top_k + q - 1) / q);
                if (t < warps) {
                    const uint32_t own = sh.every_bound[t];
                    int before = 0;
                    for (int w = 0; w < warps; ++w) before += sh.every_bound[w] < own || (sh.every_bound[w] == own && w < t);
                    if (before == enough - 1) sh.bound = own;
                }
                __syncthreads();
                if (sh.bound != kOut) {
                    const bool fits = search.gather(0u, sh.bound, sums.best);
                    if (fits) {
                        team.done();
                        if (rank == 0) {
                            search.draw((int)top_k, wanted, weight_of(top_key));
                            if (warp == 0) {
                                const double all = all_sums();
                                if (lane == 0) answer((int)sh.cut, all);
                            }
                        }
                        team.all_done();
                        return;
                    }
                    team.wait();
                    if (rank == 0 && t == 0) sh.listed = 0u;          // (there are waits before the next list)
                }
            }
            cut = search.find(true, (u64)top_k, kEnd - 1u);
            weighed = false;
            if (top_p < 1.0f) {
                total = search.weigh(cut, turn, &weight, &upto);
                turn ^= 1;
            }
        }
    }
    if (top_p < 1.0f) {
        const u64 target = max(share_up(steps(top_p, 0xffffffu), total), 1ull);
        // tokens so light that as many as the vocabulary's power of two would not make up what is left out: 2^(45 - d) of them <= total - target
        uint32_t most = kEnd - 1u;
        const u64 each_less = (total - target) >> a.vocab_bits;
        if (each_less > 0) most = min(most, ((uint32_t)max(45 - (63 - __clzll((long long)each_less)), 1) << 23) - 1u);
        if (cut != ~0ull) most = min(most, (uint32_t)(cut >> kNumberBits));
        cut = search.find(false, target, most);
        weighed = false;
    }
    if (wanted.min_p > 0u) {
        // the key of the least e with floor(2^44 e) as large as that share
        const u64 least = share_up(wanted.min_p, weight_of(top_key));
        const u64 by_share = (u64)(kTop - (uint32_t)f2i(__double2float_ru((double)least * 0x1p-44))) << kNumberBits | ((1u << kNumberBits) - 1u);
        if (by_share < cut) {
            cut = by_share;
            weighed = false;
        }
    }
    if (!weighed) total = search.weigh(cut, turn, &weight, &upto);
    team.done();
    const u64 drawn = share(wanted.uniform, total).whole;
    if (upto <= drawn && drawn < upto + weight) {
        // this warp has the token
        const double all = all_sums();
        for (int q = first; q < last; q += 32) {
            const uint4 k = search.quad(q + lane);
            const uint32_t key[4] = {k.x, k.y, k.z, k.w};
            u64 w[4], own = 0ull;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = key[j] != kOut && search.composite(key[j], (q + lane) * 4 + j) <= cut;
                w[j] = in ? weight_of(key[j]) : 0ull;
                own += w[j];
            }
            const u64 run = upto + warp_upto(own);
            const uint32_t reached = __ballot_sync(0xffffffffu, run > drawn);
            if (reached) {
                if (lane == __ffs(reached) - 1) {
                    u64 at = run - own;
                    int j = 0;
                    while (j < 3 && at + w[j] <= drawn) at += w[j++];
                    answer(search.begin + (q + lane) * 4 + j, all);
                }
                break;
            }
            upto = __shfl_sync(0xffffffffu, run, 31);
        }
    }
    team.all_done();                                                                  // (no CTA leaves while others read its memory)
}

// CTAs of a row: as many as its keys need, and more where rows are few.  (64 rows of 10000 tokens: one CTA 12.3 us, two 10.3, eight 12.4; 640 rows: one 22.5, two 25.7; 16 rows of 50001:
// two 16.5, eight 12.3.  What the CTAs of a cluster wait for one another is what more of them cost: 256 rows of 151643, 16 CTAs of 256 threads 148, eight of 512 124.)
int ctas_of(int64_t rows, int64_t vocab) {
    int c = 1;
    while (c < kMostCtas && (int64_t)c * kMostKeys < vocab) c *= 2;
    while (c < kMostCtas && rows * c * 2 <= sm_count() && vocab >= 4096 * c) c *= 2;
    return c;
}

// (what the kernels may ask for, whatever a call needs: calls of two threads set the same)
template <int THREADS>
constexpr size_t kFixed = (sizeof(Shared<THREADS>) + 15) / 16 * 16;
template <int THREADS>
constexpr size_t kMostMemory = kFixed<THREADS> + (kMostKeys / 512 * THREADS + 4) * 4 + kMostKeys / 512 * THREADS / 4 + 4;
static_assert(kMostMemory<512> <= 220 * 1024);

template <int THREADS>
int launch(const Sample& a, int64_t rows, int ctas, cudaStream_t st) {
    const size_t memory = kFixed<THREADS> + (size_t)(a.part + 4) * 4 + (a.banned ? a.part / 4 + 4 : 0);
    if (memory > kMostMemory<THREADS>) return PAMK_ERR_SIZE;                          // (no plan comes near)
    if (memory > 40 * 1024) {
        const cudaError_t err = cudaFuncSetAttribute(sample_kernel<THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostMemory<THREADS>);
        if (err != cudaSuccess) return record_cuda_error(err);
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)ctas, 1u, 1u};
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(rows * ctas));
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = memory;
    config.stream = st;
    config.attrs = &attr;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, sample_kernel<THREADS>, a);
    count_launch();
    return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
}

}  // namespace
}  // namespace pamk

extern "C" {

int pamk_sample(const float* logits, const float* uniform, const unsigned char* banned, int64_t* tokens, float* scores, int64_t rows, int64_t vocab,
                int64_t logits_row, int64_t banned_row, const float* temperatures, float temperature, const int64_t* top_ks, int64_t top_k, const float* top_ps,
                float top_p, const float* min_ps, float min_p, void* stream) {
    using namespace pamk;
    if (rows < 0 || vocab < 1 || (rows > 0 && (!logits || !uniform || !tokens || !scores))) return PAMK_ERR_ARG;
    if (vocab > (int64_t)kMostCtas * kMostKeys || rows > 0x7fffffff / kMostCtas) return PAMK_ERR_SIZE;
    if (rows == 0) return PAMK_OK;
    const int ctas = ctas_of(rows, vocab);
    Sample a{};
    a.logits = logits;
    a.uniform = uniform;
    a.banned = banned;
    a.x_row = logits_row;
    a.ban_row = banned_row;
    a.temperatures = temperatures;
    a.top_ps = top_ps;
    a.min_ps = min_ps;
    a.top_ks = top_ks;
    a.temperature = temperature;
    a.top_p = top_p;
    a.min_p = min_p;
    a.top_k = top_k;
    a.vocab = (int)vocab;
    while (((int64_t)1 << a.vocab_bits) < vocab) ++a.vocab_bits;
    a.part = (int)((vocab + ctas - 1) / ctas + 31) / 32 * 32;
    a.tokens = tokens;
    a.scores = scores;
    // (640 rows of 10000 tokens: 256 threads 22 us, 512 30)
    return a.part <= kMostKeys / 2 ? launch<256>(a, rows, ctas, (cudaStream_t)stream) : launch<512>(a, rows, ctas, (cudaStream_t)stream);
}

}
