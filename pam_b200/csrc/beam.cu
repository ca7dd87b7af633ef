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
// The logits are read once.  A first kernel takes up to 4096 of a beam's logits into the registers of a CTA and leaves
// their maximum, their sum and the best k of them: the k-th largest of a warp's 32 thread maxima bounds the k-th largest
// logit from below, the largest such bound of the eight warps leaves a few dozen candidates, and each of those counts how many are
// larger.  Keys (logit, then lower token) are all different, so a candidate's rank is its place, and no order of atomics shows.  A
// second kernel joins the parts of each beam and picks the k best of the group from the lists in the same way.
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
    int32_t off;
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

__global__ void __launch_bounds__(kThreads) pick_kernel(const Select a) {
    __shared__ unsigned long long found[kMostLogits];
    __shared__ unsigned long long warp_least[kThreads / 32];
    __shared__ double warp_total[kThreads / 32];
    __shared__ float warp_top[kThreads / 32];
    __shared__ int count;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t beam = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x % a.parts);
    if (dead(a.scores[beam])) return;                                             // (its logits are not looked at)
    const int64_t group = beam / a.rows, row = beam % a.rows;
    const int begin = part * a.part, end = min(begin + a.part, a.vocab);
    const float* x = a.logits + group * a.x_group + row * a.x_row;
    const unsigned char* banned = a.banned ? a.banned + group * a.ban_group + row * a.ban_row : nullptr;
    // vectors start at addresses that are multiples of 16 bytes: the first one may begin before the range
    const int first = begin - (int)((reinterpret_cast<uintptr_t>(x + begin) >> 2) & 3);
    float v[kEach];
    uint32_t key[kEach];
#pragma unroll
    for (int i = 0; i < kEach / 4; ++i) {
        const int j = first + (i * kThreads + t) * 4;
        if (j >= begin && j + 4 <= end) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(x + j));
            v[4 * i] = w.x; v[4 * i + 1] = w.y; v[4 * i + 2] = w.z; v[4 * i + 3] = w.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * i + e] = j + e >= begin && j + e < end ? __ldg(x + j + e) : -INFINITY;
        }
    }
    if (t == 0) count = 0;
    float top = -INFINITY;
    unsigned long long best = 0ull;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int j = first + ((i / 4) * kThreads + t) * 4 + i % 4;
        const bool inside = j >= begin && j < end, masked = !(v[i] > kMasked);    // (NaN: the beam has no finite sum, and no candidates)
        const bool ban = banned && inside && banned[j];
        if (!masked || v[i] != v[i]) top = fmaxf(top, v[i]);
        key[i] = !inside ? 0u : masked || ban ? kMaskedKey : ordered(v[i]);
        const unsigned long long full = inside ? (unsigned long long)key[i] << 32 | (uint32_t)~j : 0ull;
        best = full > best ? full : best;
    }
    // the k-th largest of the warp's thread maxima (0 if there are fewer)
    int rank = 0;
#pragma unroll 8
    for (int l = 0; l < 32; ++l) rank += __shfl_sync(0xffffffffu, best, l) > best;
    const unsigned who = __ballot_sync(0xffffffffu, rank == a.k - 1 && best != 0ull);
    const unsigned long long least = who ? __shfl_sync(0xffffffffu, best, __ffs(who) - 1) : 0ull;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (lane == 0) {
        warp_least[warp] = least;
        warp_top[warp] = top;
    }
    __syncthreads();
    unsigned long long from = 1ull;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        from = warp_least[w] > from ? warp_least[w] : from;
        top = fmaxf(top, warp_top[w]);
    }
    const float shift = floorf(mul(top, kLog2e, a.off));
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int j = first + ((i / 4) * kThreads + t) * 4 + i % 4;
        const unsigned long long full = (unsigned long long)key[i] << 32 | (uint32_t)~j;
        if (key[i] && full >= from) found[atomicAdd(&count, 1)] = full;
        if (v[i] > kMasked || v[i] != v[i]) {
            const float s = mul(v[i], kLog2e, a.off), whole = floorf(s), lin = fadd(1.0f, fadd(s, -whole));
            const float down = fadd(whole, -shift);
            total += down >= -126.0f ? (double)fmul(lin, i2f(((int32_t)down + 127) << 23)) : down != down ? (double)down : 0.0;
        }
    }
    total = warp_sum(total);
    if (lane == 0) warp_total[warp] = total;
    __syncthreads();
    const int64_t list = beam * a.parts + part;
    if (t == 0) {
        double sum = warp_total[0];
#pragma unroll
        for (int w = 1; w < kThreads / 32; ++w) sum += warp_total[w];
        a.sums[list] = sum;
        a.shifts[list] = shift;
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
__device__ __forceinline__ double over_log2e(double x, int32_t off) {
    const long long by = __double_as_longlong((double)kLog2e), one = __double_as_longlong(1.0);
    if (!(fabs(x) < 1e37)) return (double)quiet_nan();                             // (also NaN)
    if (fabs(x / (double)kLog2e) < 1e-37) return 0.0;
    return __longlong_as_double(__double_as_longlong(x) - by + one - ((long long)off << 29));
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

__global__ void __launch_bounds__(kThreads) merge_kernel(const Select a) {
    extern __shared__ __align__(16) unsigned char shared[];
    __shared__ Candidate least;
    __shared__ int count;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int lists = a.rows * a.parts;
    double* lse = reinterpret_cast<double*>(shared);                              // [rows], NaN for a beam without finite sum
    unsigned long long* heads = reinterpret_cast<unsigned long long*>(lse + a.rows);   // [lists]
    const int64_t first_beam = (int64_t)blockIdx.x * a.rows;
    after_previous();
    for (int r = warp; r < a.rows; r += kThreads / 32) {
        double value = (double)quiet_nan();
        if (!dead(a.scores[first_beam + r])) {
            const int64_t at = (first_beam + r) * a.parts;
            float m = -INFINITY;
            double sum = 0.0;
            for (int c = lane; c < a.parts; c += 32) m = fmaxf(m, __ldcg(a.shifts + at + c));
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            for (int c = lane; c < a.parts; c += 32) {
                const double s = __ldcg(a.sums + at + c);
                sum += s == 0.0 ? 0.0 : s * exp2_int_d(fadd(__ldcg(a.shifts + at + c), -m));
            }
            sum = warp_sum(sum);
            if (sum > 0.0 && sum < 1e300) value = over_log2e((double)m + affine_log2(sum), a.off);
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
    // entry i of a list as a candidate; a beam without finite sum has its first tokens at -inf
    const auto candidate = [&](int list, int i) {
        Candidate c;
        c.beam = list / a.parts;
        const double by = lse[c.beam];
        const float score = a.scores[first_beam + c.beam];
        if (by != by) {
            c.key = list % a.parts == 0 && i < a.vocab ? (unsigned long long)kMaskedKey << 32 | (uint32_t)~i : 0ull;
            c.value = c.key ? ordered((double)-INFINITY) : 0ull;
            return c;
        }
        c.key = __ldcg(a.lists + (first_beam * a.parts + list) * a.k + i);
        const uint32_t x = (uint32_t)(c.key >> 32);
        c.value = c.key == 0ull ? 0ull
                                : ordered(x == kMaskedKey ? (double)-INFINITY : ((double)of_ordered(x) - by) + (double)score);
        return c;
    };
    // The k-th best head of a list bounds the k-th best candidate: only k lists reach it.
    const bool bounded = lists >= a.k;
    if (bounded) {
        for (int i = t; i < lists; i += kThreads) heads[i] = candidate(i, 0).value;
        __syncthreads();
        for (int i = t; i < lists; i += kThreads) {
            const Candidate mine = candidate(i, 0);
            int r = 0;
            for (int o = 0; o < lists; ++o) {
                const unsigned long long other = heads[o];
                r += other > mine.value || (other == mine.value && o != i && candidate(o, 0).before(mine));
            }
            if (r == a.k - 1 && mine.value != 0ull) least = mine;
        }
        __syncthreads();
    }
    Candidate* found = reinterpret_cast<Candidate*>(heads + (lists + 1) / 2 * 2);
    for (int i = t; i < lists; i += kThreads)
        for (int e = 0; e < a.k; ++e) {
            const Candidate c = candidate(i, e);
            if (c.value == 0ull || (bounded && least.before(c))) break;
            found[atomicAdd(&count, 1)] = c;
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
            const float score = a.scores[first_beam + mine.beam];
            a.out_scores[to] = x == kMaskedKey ? -INFINITY : (float)(((double)of_ordered(x) - lse[mine.beam]) + (double)score);
            a.out_beams[to] = mine.beam;
            a.out_tokens[to] = (int64_t)(uint32_t)~(uint32_t)mine.key;
        }
    }
}

size_t aligned(size_t n) { return (n + 255) / 256 * 256; }

// (a range may begin inside a vector of four)
constexpr int kMostPart = kMostLogits - 4;
int parts_of(int64_t vocab) { return (int)((vocab + kMostPart - 1) / kMostPart); }

// The shared memory of the second kernel: at most k lists of k entries reach the bound, fewer lists than k are taken whole.
size_t merge_bytes(int64_t rows, int64_t parts, int64_t k) {
    const int64_t lists = rows * parts, entries = (lists < k ? lists : k) * k;
    return (size_t)(rows * 8 + (lists + 1) / 2 * 16 + entries * sizeof(Candidate) + 16);
}

// ---- reordering ------------------------------------------------------------------------------------------------

constexpr int kStatesPerLaunch = 256;

struct States {
    char* base[kStatesPerLaunch];
    int64_t group[kStatesPerLaunch], row[kStatesPerLaunch], bytes[kStatesPerLaunch], unit[kStatesPerLaunch];   // strides, a row's and a position's bytes
    unsigned first[kStatesPerLaunch + 1];             // blocks [first[k], first[k + 1]) move tensor k
    int used;
};

// A thread takes one piece of a row's bytes in every row of a group: all rows that something is taken from are read before the first
// is written, so the move needs no second copy of the states.
template <class T, int ROWS>
__global__ void __launch_bounds__(kThreads) reorder_kernel(const States s, const int64_t* parents, const int64_t* positions, int rows) {
    __shared__ int parent[ROWS];
    int lo = 0, hi = s.used - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (s.first[mid] <= blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    int64_t bytes = s.bytes[lo];
    if (positions) {
        const int64_t n = *positions, most = bytes / s.unit[lo];
        bytes = (n < 0 ? 0 : n < most ? n : most) * s.unit[lo];
    }
    const int64_t blocks = (s.bytes[lo] + (int64_t)kThreads * sizeof(T) - 1) / ((int64_t)kThreads * (int64_t)sizeof(T));
    const int64_t block = blockIdx.x - s.first[lo], group = block / blocks;
    const int64_t at = ((block % blocks) * kThreads + threadIdx.x) * (int64_t)sizeof(T);
    if (threadIdx.x < ROWS) {
        const int64_t p = threadIdx.x < rows ? parents[group * rows + threadIdx.x] : -1;
        parent[threadIdx.x] = p >= 0 && p < rows ? (int)p : threadIdx.x;           // (a parent that does not exist leaves the row as it is)
    }
    __syncthreads();
    if (at >= bytes) return;
    char* base = s.base[lo] + group * s.group[lo] + at;
    T x[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (r < rows && parent[r] != r) x[r] = *reinterpret_cast<const T*>(base + parent[r] * s.row[lo]);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (r < rows && parent[r] != r) *reinterpret_cast<T*>(base + r * s.row[lo]) = x[r];
}

template <class T>
int launch_reorder(const States& s, unsigned blocks, const int64_t* parents, const int64_t* positions, int rows, cudaStream_t st) {
    if (rows <= 4) reorder_kernel<T, 4><<<blocks, kThreads, 0, st>>>(s, parents, positions, rows);
    else if (rows <= 8) reorder_kernel<T, 8><<<blocks, kThreads, 0, st>>>(s, parents, positions, rows);
    else if (rows <= 16) reorder_kernel<T, 16><<<blocks, kThreads, 0, st>>>(s, parents, positions, rows);
    else reorder_kernel<std::conditional_t<sizeof(T) == 16, uint32_t, T>, 64><<<blocks, kThreads, 0, st>>>(s, parents, positions, rows);
    return check_launch();
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
                     int64_t banned_group, int64_t banned_row, float offset, void* workspace, size_t workspace_bytes, void* stream) {
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
    a.off = offset_bits(offset);
    char* ws = static_cast<char*>(workspace);
    a.sums = reinterpret_cast<double*>(ws);
    ws += aligned((size_t)(groups * lists) * 8);
    a.shifts = reinterpret_cast<float*>(ws);
    ws += aligned((size_t)(groups * lists) * 4);
    a.lists = reinterpret_cast<unsigned long long*>(ws);
    a.out_scores = out_scores; a.out_beams = out_beams; a.out_tokens = out_tokens;
    pick_kernel<<<(unsigned)(groups * lists), kThreads, 0, st>>>(a);
    const int status = check_launch();
    if (status != PAMK_OK) return status;
    const size_t bytes = merge_bytes(rows, parts, k);
    if (bytes > 48 * 1024) {
        const cudaError_t err = cudaFuncSetAttribute(merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (err != cudaSuccess) return record_cuda_error(err);
    }
    merge_kernel<<<(unsigned)groups, kThreads, bytes, st>>>(a);
    return check_launch();
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
                const uint64_t more = (uint64_t)((moved_bytes[i] + kThreads * piece - 1) / (kThreads * piece)) * (uint64_t)groups;
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
