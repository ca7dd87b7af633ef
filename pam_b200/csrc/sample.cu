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
// A row belongs to a cluster of up to eight CTAs, each of which keeps its part in shared memory as keys d 2^23 + (1 - f') 2^23 - 1, smaller for larger weights, after
// reading the logits once.  A cut is found in three steps of 11, 9 and 9 bits of the key, each a histogram of numbers and weights that the CTAs of the cluster
// read of one another.
#include <cooperative_groups.h>

#include "common.cuh"
#include "pam_scalar.cuh"

namespace pamk {
namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMasked = -1e30f;                     // a logit as low as this is masked
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMostCtas = 8, kMostKeys = 32768;       // of a cluster; of a CTA
constexpr uint32_t kOut = 0xffffffffu;                // the key of a token without weight
constexpr int kBins = 2048;

struct Sample {
    const float *logits, *uniform;
    const unsigned char* banned;                      // or null
    int64_t x_row, ban_row;
    const float *temperatures, *top_ps, *min_ps;      // one for each row, or null: the same for all
    const int64_t* top_ks;
    float temperature, top_p, min_p;
    int64_t top_k;
    int vocab, part;                                  // a CTA's tokens
    int64_t* tokens;
    float* scores;
};

struct Pair { unsigned long long weight; uint32_t count; };

struct Shared {
    uint32_t count[kBins], low[kBins], high[kBins];   // of each bin: keys, and the sum of their weights' digits by 12 bits
    Pair scan[kWarps];
    unsigned long long near[kWarps], far[kWarps], kept[kWarps];
    float top_all[kWarps], top_ok[kWarps];
    // what the other CTAs of the cluster read
    struct { float all, ok; int bad; unsigned long long near, far, kept; unsigned long long part[kWarps]; uint32_t ties[kWarps]; } mine;
    // what a step of the search found
    uint32_t bin, less_count;
    unsigned long long less_weight;
    unsigned long long before;                        // of the warp that has the token
    int owner;
    long long token;
};

__device__ __forceinline__ unsigned long long weight_of(uint32_t key) {
    const uint32_t d = key >> 23, m = 0x800000u | (~key & 0x7fffffu);
    return d <= 21u ? (unsigned long long)m << (21u - d) : (unsigned long long)(m >> min(d - 21u, 31u));
}

// floor and the rest of fraction 2^-24 total
struct Share { unsigned long long whole; bool rest; };
__device__ __forceinline__ Share share(uint32_t fraction, unsigned long long total) {
    const unsigned long long low = total * fraction;
    return {__umul64hi(total, fraction) << 40 | low >> 24, (low & 0xffffffu) != 0};
}
__device__ __forceinline__ unsigned long long share_up(uint32_t fraction, unsigned long long total) {
    const Share s = share(fraction, total);
    return s.whole + s.rest;
}
// A fraction in steps of 2^-24, NaN as 0.
__device__ __forceinline__ uint32_t steps(float f, uint32_t most) { return f > 0.0f ? min((uint32_t)fminf(f * 16777216.0f, 16777216.0f), most) : 0u; }

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// pad(M + log2(S), log2 e) in 64 bits, log2(2^i (1 + f)) = i + f, S >= 1
__device__ double log_sum(double shift, double total) {
    const long long bits = __double_as_longlong(total);
    const double fraction = __longlong_as_double((bits & 0xfffffffffffffll) | 0x3ff0000000000000ll) - 1.0;
    const double log2 = shift + ((double)((bits >> 52) - 1023) + fraction), by = (double)kLog2e;
    if (fabs(log2 / by) < 1e-37) return 0.0;
    return __longlong_as_double(__double_as_longlong(log2) - __double_as_longlong(by) + 0x3ff0000000000000ll);
}

// The digits of a key's weight without its shift (which is the same for all keys of a bin).
__device__ __forceinline__ uint32_t digits(uint32_t key) {
    const uint32_t d = key >> 23, m = 0x800000u | (~key & 0x7fffffu);
    return d <= 21u ? m : m >> (d - 21u);
}

// Where in the order of the keys a count or a weight is reached: the keys of bin `prefix` (of `shift + bits` low bits) in bins of 2^shift, less_* before them.
// Sets sh.bin to the bin in which `target` is reached (by count, else by weight) and sh.less_* to what lies before it.
__device__ void search(Shared& sh, const uint32_t* keys, int n, cg::cluster_group& cluster, uint32_t prefix, int shift, int bits, uint32_t less_count,
                       unsigned long long less_weight, bool by_count, unsigned long long target) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, bins = 1 << bits;
    for (int b = t; b < bins; b += kThreads) sh.count[b] = sh.low[b] = sh.high[b] = 0u;
    __syncthreads();
    for (int j = t; j < n; j += kThreads) {
        const uint32_t key = keys[j];
        if (key == kOut || key >> (shift + bits) != prefix) continue;
        const uint32_t b = key >> shift & (bins - 1), m = digits(key);
        atomicAdd(&sh.count[b], 1u);
        atomicAdd(&sh.low[b], m & 0xfffu);
        atomicAdd(&sh.high[b], m >> 12);
    }
    cluster.sync();
    const int each = bins / kThreads;                 // 4 or 1 neighbouring bins
    Pair own[4], sum{0ull, 0u};
    const int ctas = (int)cluster.num_blocks();
    for (int k = 0; k < each; ++k) {
        const int b = t * each + k;
        uint32_t count = 0u;
        unsigned long long digits_sum = 0ull;
        for (int c = 0; c < ctas; ++c) {
            const Shared* other = cluster.map_shared_rank(&sh, c);
            count += other->count[b];
            digits_sum += (unsigned long long)other->low[b] + ((unsigned long long)other->high[b] << 12);
        }
        const uint32_t d = (prefix << bits | b) >> (23 - shift);
        own[k] = {d <= 21u ? digits_sum << (21u - d) : digits_sum, count};
        sum.weight += own[k].weight;
        sum.count += own[k].count;
    }
    Pair upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long w = __shfl_up_sync(0xffffffffu, upto.weight, d);
        const uint32_t c = __shfl_up_sync(0xffffffffu, upto.count, d);
        if (lane >= d) {
            upto.weight += w;
            upto.count += c;
        }
    }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    Pair before{less_weight, less_count};
    for (int w = 0; w < warp; ++w) {
        before.weight += sh.scan[w].weight;
        before.count += sh.scan[w].count;
    }
    before.weight += upto.weight - sum.weight;
    before.count += upto.count - sum.count;
    for (int k = 0; k < each; ++k) {
        const unsigned long long from = by_count ? before.count : before.weight, to = from + (by_count ? own[k].count : own[k].weight);
        if (from < target && target <= to) {
            sh.bin = t * each + k;
            sh.less_count = before.count;
            sh.less_weight = before.weight;
        }
        before.weight += own[k].weight;
        before.count += own[k].count;
    }
    cluster.sync();                                   // (the histograms may be written anew)
}

struct Cut {
    uint32_t key;                                     // the last one that stays
    uint32_t less_count, ties;                        // so many smaller ones; so many equal ones stay
    unsigned long long less_weight;
    __device__ unsigned long long weight() const { return less_weight + ties * weight_of(key); }
};

__device__ Cut find_cut(Shared& sh, const uint32_t* keys, int n, cg::cluster_group& cluster, bool by_count, unsigned long long target) {
    uint32_t prefix = 0u, less_count = 0u;
    unsigned long long less_weight = 0ull;
    constexpr int kBits[3] = {11, 9, 9}, kShift[3] = {18, 9, 0};
    for (int step = 0; step < 3; ++step) {
        search(sh, keys, n, cluster, prefix, kShift[step], kBits[step], less_count, less_weight, by_count, target);
        prefix = prefix << kBits[step] | sh.bin;
        less_count = sh.less_count;
        less_weight = sh.less_weight;
        __syncthreads();
    }
    Cut cut{prefix, less_count, 0u, less_weight};
    const unsigned long long each = weight_of(prefix);
    cut.ties = (uint32_t)(by_count ? target - less_count : (target - less_weight + each - 1) / each);
    return cut;
}

__global__ void __launch_bounds__(kThreads) sample_kernel(const Sample a) {
    extern __shared__ __align__(16) unsigned char memory[];
    Shared& sh = *reinterpret_cast<Shared*>(memory);
    uint32_t* keys = reinterpret_cast<uint32_t*>(memory + sizeof(Shared));
    uint32_t* flags = keys + (a.part + 31) / 32 * 32;                                 // a bit for each token: banned
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
    const int64_t row = blockIdx.x / ctas;
    const int begin = min(rank * a.part, a.vocab), n = min(a.part, a.vocab - begin);
    const float* x = a.logits + row * a.x_row;
    const unsigned char* banned = a.banned ? a.banned + row * a.ban_row : nullptr;
    const float temperature = a.temperatures ? __ldg(a.temperatures + row) : a.temperature;
    const float top_p = a.top_ps ? __ldg(a.top_ps + row) : a.top_p, min_p = a.min_ps ? __ldg(a.min_ps + row) : a.min_p;
    const int64_t top_k = a.top_ks ? __ldg(reinterpret_cast<const long long*>(a.top_ks) + row) : a.top_k;
    const Divisor by_temperature = make_divisor(temperature, 0);

    // the row's t, and the largest of all and of those that may be drawn
    float top_all = -INFINITY, top_ok = -INFINITY;
    bool bad = !(temperature > 0.0f && temperature <= i2f(0x7f7fffff));
    for (int j = t; j < (n + 31) / 32 * 32; j += kThreads) {
        const float raw = j < n ? __ldg(x + begin + j) : -INFINITY;
        const float v = raw <= kMasked ? -INFINITY : mul(div_by(raw, by_temperature), kLog2e, 0);
        const bool out = j < n && banned && banned[begin + j];
        const uint32_t word = __ballot_sync(0xffffffffu, out);
        if (lane == 0) flags[j >> 5] = word;
        bad = bad || v != v;
        if (j < n) keys[j] = (uint32_t)f2i(v);
        top_all = fmaxf(top_all, v);
        if (!out) top_ok = fmaxf(top_ok, v);
    }
    top_all = warp_max(top_all);
    top_ok = warp_max(top_ok);
    if (lane == 0) {
        sh.top_all[warp] = top_all;
        sh.top_ok[warp] = top_ok;
    }
    const int any_bad = __syncthreads_or(bad);
    if (t == 0) {
        float all = -INFINITY, ok = -INFINITY;
        for (int w = 0; w < kWarps; ++w) {
            all = fmaxf(all, sh.top_all[w]);
            ok = fmaxf(ok, sh.top_ok[w]);
        }
        sh.mine.all = all;
        sh.mine.ok = ok;
        sh.mine.bad = any_bad;
    }
    cluster.sync();
    int no_token = 0;
    for (int c = 0; c < ctas; ++c) {
        const Shared* other = cluster.map_shared_rank(&sh, c);
        top_all = fmaxf(top_all, other->mine.all);
        top_ok = fmaxf(top_ok, other->mine.ok);
        no_token |= other->mine.bad;
    }
    if (no_token || !(top_ok > -INFINITY)) {                                          // (all CTAs of the cluster alike)
        if (rank == 0 && t == 0) {
            a.tokens[row] = -1;
            a.scores[row] = -INFINITY;
        }
        cluster.sync();
        return;
    }
    const float shift_all = floorf(top_all), shift_ok = floorf(top_ok);
    const uint32_t top_key = ~f2i(__fadd_rd(1.0f, __fadd_rd(top_ok, -shift_ok))) & 0x7fffffu;

    // keys in place of the t, and the sums
    unsigned long long near = 0ull, far = 0ull, kept = 0ull;
    for (int j = t; j < n; j += kThreads) {
        const float v = i2f((int32_t)keys[j]);
        const float whole = floorf(v);
        uint32_t key = kOut;
        if (v > -INFINITY) {
            const float lin = __fadd_rd(1.0f, __fadd_rd(v, -whole));                  // 1 + f'
            const uint32_t m = 0x800000u | (f2i(lin) & 0x7fffff);
            const int d = (int)fminf(shift_all - whole, 63.0f);
            // (what f' leaves of f, where t has bits below 2^-23: f - f' = t - ((1 + f') + (floor t - 1)), to a part in 2^24 of itself)
            if (fabsf(v) < 1.0f) far += (unsigned long long)(uint32_t)fmul(fadd(v, -fadd(lin, fadd(whole, -1.0f))), 0x1p44f) << 18 >> d;
            if (d <= 21)
                near += (unsigned long long)m << (21 - d);
            else if (d < 63)
                far += d <= 39 ? (unsigned long long)m << (39 - d) : (unsigned long long)(m >> (d - 39));
            const float below = shift_ok - whole;
            if (below <= 44.0f && !(flags[j >> 5] >> (j & 31) & 1u)) {
                key = (uint32_t)below << 23 | (~m & 0x7fffffu);
                kept += weight_of(key);
            }
        }
        keys[j] = key;
    }
    near = warp_sum(near);
    far = warp_sum(far);
    kept = warp_sum(kept);
    if (lane == 0) {
        sh.near[warp] = near;
        sh.far[warp] = far;
        sh.kept[warp] = kept;
    }
    __syncthreads();
    if (t == 0) {
        near = far = kept = 0ull;
        for (int w = 0; w < kWarps; ++w) {
            near += sh.near[w];
            far += sh.far[w];
            kept += sh.kept[w];
        }
        sh.mine.near = near;
        sh.mine.far = far;
        sh.mine.kept = kept;
    }
    cluster.sync();
    near = far = kept = 0ull;
    for (int c = 0; c < ctas; ++c) {
        const Shared* other = cluster.map_shared_rank(&sh, c);
        near += other->mine.near;
        far += other->mine.far;
        kept += other->mine.kept;
    }

    // what stays
    Cut cut{kOut - 1u, 0u, 0u, kept};
    if (top_k > 0 && top_k < a.vocab) {
        // (fewer than k may have a weight)
        uint32_t mine = 0u;
        for (int j = t; j < n; j += kThreads) mine += keys[j] != kOut;
        const uint32_t warps = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) sh.mine.ties[warp] = warps;
        cluster.sync();
        uint32_t all = 0u;
        for (int c = 0; c < ctas; ++c)
            for (int w = 0; w < kWarps; ++w) all += cluster.map_shared_rank(&sh, c)->mine.ties[w];
        if (top_k < all) {
            cut = find_cut(sh, keys, n, cluster, true, (unsigned long long)top_k);
            kept = cut.weight();
        }
        cluster.sync();
    }
    if (top_p < 1.0f) {
        const unsigned long long target = max(share_up(steps(top_p, 0xffffffu), kept), 1ull);
        cut = find_cut(sh, keys, n, cluster, false, target);
    }
    const unsigned long long least = share_up(steps(min_p, 1u << 24), weight_of(top_key));
    const unsigned long long tie = weight_of(cut.key);
    const bool ties_stay = tie >= least;

    // the sums of what stays, by warps in the order of the vocabulary
    const int each = ((n + kWarps - 1) / kWarps + 31) / 32 * 32, from = min(warp * each, n), to = min(from + each, n);
    unsigned long long sum = 0ull;
    uint32_t ties = 0u;
    for (int j = from + lane; j < to; j += 32) {
        const uint32_t key = keys[j];
        if (key < cut.key) {
            const unsigned long long w = weight_of(key);
            if (w >= least) sum += w;
        } else if (key == cut.key) {
            ++ties;
        }
    }
    sum = warp_sum(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) {
        sh.mine.part[warp] = sum;
        sh.mine.ties[warp] = ties;
    }
    if (t == 0) sh.owner = -1;
    cluster.sync();
    unsigned long long total = 0ull, upto = 0ull;
    uint32_t ties_before = 0u;
    {
        uint32_t seen = 0u;
        for (int c = 0; c < ctas; ++c)
            for (int w = 0; w < kWarps; ++w) {
                const Shared* other = cluster.map_shared_rank(&sh, c);
                if (c == rank && w == warp) {
                    upto = total;
                    ties_before = seen;
                }
                const uint32_t here = other->mine.ties[w], stay = ties_stay ? min(here, cut.ties - min(seen, cut.ties)) : 0u;
                total += other->mine.part[w] + stay * tie;
                seen += here;
            }
    }
    const unsigned long long drawn = share(steps(__ldg(a.uniform + row), 0xffffffu), total).whole;
    const uint32_t stay = ties_stay ? min(ties, cut.ties - min(ties_before, cut.ties)) : 0u;
    if (upto <= drawn && drawn < upto + sum + stay * tie) {
        // this warp has the token
        for (int first = from; first < to; first += 32) {
            const int j = first + lane;
            const uint32_t key = j < to ? keys[j] : kOut;
            const uint32_t equal = __ballot_sync(0xffffffffu, key == cut.key);
            unsigned long long w = 0ull;
            if (key < cut.key)
                w = weight_of(key);
            else if (key == cut.key && ties_before + __popc(equal & ((1u << lane) - 1u)) < cut.ties)
                w = tie;
            if (w < least) w = 0ull;
            ties_before += __popc(equal);
            unsigned long long run = w;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const unsigned long long v = __shfl_up_sync(0xffffffffu, run, d);
                if (lane >= d) run += v;
            }
            const uint32_t reached = __ballot_sync(0xffffffffu, upto + run > drawn);
            if (reached) {
                if (lane == __ffs(reached) - 1) {
                    const int token = begin + j;
                    const float chosen = div_by(__ldg(x + token), by_temperature);
                    a.tokens[row] = token;
                    a.scores[row] = (float)((double)chosen - log_sum((double)shift_all, (double)near * 0x1p-44 + (double)far * 0x1p-62));
                }
                break;
            }
            upto += __shfl_sync(0xffffffffu, run, 31);
        }
    }
    cluster.sync();                                                                   // (no CTA leaves while others read its memory)
}

// CTAs of a row: as many as its keys need, and more where rows are few.
int ctas_of(int64_t rows, int64_t vocab) {
    int c = 1;
    while (c < kMostCtas && (int64_t)c * kMostKeys < vocab) c *= 2;
    while (c < kMostCtas && rows * c * 2 <= sm_count() && vocab >= 4096 * c) c *= 2;
    return c;
}

// (what the kernel may ask for, whatever a call needs: calls of two threads set the same)
constexpr size_t kMostMemory = sizeof(Shared) + kMostKeys * 4 + kMostKeys / 8;
static_assert(kMostMemory <= 220 * 1024);

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
    a.part = (int)((vocab + ctas - 1) / ctas + 31) / 32 * 32;
    a.tokens = tokens;
    a.scores = scores;
    const size_t memory = sizeof(Shared) + (size_t)a.part * 4 + (size_t)a.part / 8;
    if (memory > 40 * 1024) {
        const cudaError_t err = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostMemory);
        if (err != cudaSuccess) return record_cuda_error(err);
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)ctas, 1u, 1u};
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(rows * ctas));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = memory;
    config.stream = (cudaStream_t)stream;
    config.attrs = &attr;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, sample_kernel, a);
    count_launch();
    return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
}

}
