// Embedding: rows of a table by token, scaled by a PAM product, with positions added and dropout, and the table's gradient.
//     x_i = pam(w[token_i], scale) + pos[i mod T]        y_i = kept ? pam(x_i, s) : 0       (philox.cuh; every step but the first is left out on demand)
//     dw[v] = sum over i with token_i = v of pam(drop'(g_i), scale)   (approximate gradients; exact ones: times slope(w[v], scale))
// with drop'(g) = kept ? pam(g, s) : 0 (exact: g slope(x, s)).  The row of the padding token has no gradient.
// A token outside the table reads nothing: its row is NaN, and it has no gradient.
//
// The gradient is a sort and a segmented sum, so that every row of g is read once, wherever its token occurs, and no atomics decide on an order:
//   sort   the places of the tokens in the order (token, place).  Up to 4096 tokens each counts those before it, which all SMs share (4096 tokens: 17 million comparisons);
//          more are cut into tiles and moved by two digits of at most 11 bits, each pass stable.  The other CTAs of these launches fill the gradient with zeros
//          meanwhile.  (One CTA that moves up to 8192 tokens by digits in its shared memory: 14 us for 4096.)
//   sums   a warp adds the rows of 16 neighbours in that order (32 where there are many), 128 columns of them, and writes the tokens that lie within;
//   joins  a token with neighbours in several such chunks has its parts added in their order, by a warp for each 128 columns, or by a CTA where they are many.
#include "common.cuh"
#include "pam_scalar.cuh"
#include "philox.cuh"
#include "times.cuh"

namespace pamk {
namespace {

constexpr int kThreads = 256;

struct Embedding {
    const int64_t* tokens;
    const float *table, *pos;             // pos or null
    int64_t count, table_row, pos_row, pos_count, vocab, padding;
    int dim;
    bool scaled, drops;
    Times scale, keep;                    // pam(x, scale); pam(x, s)
    Dropping drop;
};

__device__ __forceinline__ int64_t token_at(const int64_t* tokens, int64_t i) { return __ldg(reinterpret_cast<const long long*>(tokens) + i); }

__device__ __forceinline__ float looked_up(const Embedding& a, int64_t i, int c) {
    const int64_t token = token_at(a.tokens, i);
    if ((uint64_t)token >= (uint64_t)a.vocab) return quiet_nan();
    float x = __ldg(a.table + token * a.table_row + c);
    if (a.scaled) x = a.scale.one(x);
    return a.pos ? fadd(x, __ldg(a.pos + (a.pos_count == 1 ? 0 : i % a.pos_count) * a.pos_row + c)) : x;
}

// The output element of a sum x: dropped out; SLOPES: g times the slope of the dropout at x, where it is kept.
template <bool SLOPES>
__device__ __forceinline__ float finished(const Embedding& a, float x, uint32_t bits, float g) {
    if (!a.drops) return x;
    return bits < a.drop.below ? 0.0f : SLOPES ? mul_bwd(x, a.keep.s, g, a.keep.off) : a.keep.one(x);
}

// A thread takes four neighbouring elements of the output, which is what a block of the counter has bits for; here of any row length and number.
template <bool SLOPES>
__global__ void __launch_bounds__(kThreads) embed_kernel(const Embedding a, const float* g, float* out) {
    const int64_t e = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4, n = a.count * a.dim;
    if (e >= n) return;
    int64_t i = e / a.dim;
    int c = (int)(e - i * a.dim);
    const uint4 w = a.drops ? philox((uint64_t)e >> 2, key_of(a.drop)) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t bits[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (e + k >= n) return;
        out[e + k] = finished<SLOPES>(a, looked_up(a, i, c), bits[k], SLOPES ? __ldg(g + e + k) : 0.0f);
        if (++c == a.dim) {
            c = 0;
            ++i;
        }
    }
}

// n / d for n < 2^31 (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994): with 2^s the power of two next to d from above,
// floor(n (2^32 + m) / 2^(32 + s)) for m = floor(2^32 (2^s - d) / d) + 1.
struct Divide {
    uint32_t d, m, s;
    explicit Divide(uint32_t by) : d(by), s(0) {
        while (((uint64_t)1 << s) < by) ++s;
        m = (uint32_t)(((((uint64_t)1 << s) - by) << 32) / by + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

// Rows of whole quads at aligned addresses, fewer than 2^31 quads.  A thread has a few, with all of its loads on their way before the first product: as far apart as
// a CTA is wide, or (SENTENCES) those of as many sentences at one position, which they read once.  What bounds it where the table lies in the L2 is the L2: 2^20 tokens of 128
// columns with a table of positions, 9.4 TB/s of table, positions and output, 172 us with quads of neighbours.
constexpr int kQuads = 4;
template <bool SLOPES, bool SENTENCES>
__global__ void __launch_bounds__(kThreads) embed_quads_kernel(const Embedding a, const float* g, float* out, uint32_t quads, Divide by_row, Divide by_pos) {
    const uint32_t sentence = SENTENCES ? (uint32_t)a.pos_count * by_row.d : 0u, at = blockIdx.x * (SENTENCES ? kThreads : kThreads * kQuads) + threadIdx.x;
    const uint32_t first = SENTENCES ? at + blockIdx.y * kQuads * sentence : at, step = SENTENCES ? sentence : kThreads;
    const uint2 key = a.drops ? key_of(a.drop) : make_uint2(0u, 0u);
    if (SENTENCES && at >= sentence) return;
    uint32_t row[kQuads];
    int64_t token[kQuads];
    float4 x[kQuads], p[kQuads], d[kQuads];
    if (SENTENCES) row[0] = by_row(first);
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
        const uint32_t q = first + k * step;
        row[k] = SENTENCES ? row[0] + k * (uint32_t)a.pos_count : by_row(q);
        token[k] = q < quads ? token_at(a.tokens, row[k]) : -1;
    }
    if (SENTENCES) p[0] = __ldg(reinterpret_cast<const float4*>(a.pos + (int64_t)by_row(at) * a.pos_row + (at - by_row(at) * by_row.d) * 4));
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
        const uint32_t q = first + k * step, c = (SENTENCES ? first - row[0] * by_row.d : q - row[k] * by_row.d) * 4;
        x[k] = make_float4(quiet_nan(), quiet_nan(), quiet_nan(), quiet_nan());
        d[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if ((uint64_t)token[k] < (uint64_t)a.vocab) x[k] = __ldg(reinterpret_cast<const float4*>(a.table + token[k] * a.table_row + c));
        if (SENTENCES)
            p[k] = p[0];
        else
            p[k] = a.pos && q < quads ? __ldg(reinterpret_cast<const float4*>(a.pos + (int64_t)(row[k] - by_pos(row[k]) * by_pos.d) * a.pos_row + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (SLOPES && q < quads) d[k] = __ldg(reinterpret_cast<const float4*>(g) + q);
    }
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
        const uint32_t q = first + k * step;
        if (q >= quads) return;
        float4 y = a.scaled ? a.scale.of(x[k]) : x[k];
        if (a.pos) y = make_float4(fadd(y.x, p[k].x), fadd(y.y, p[k].y), fadd(y.z, p[k].z), fadd(y.w, p[k].w));
        if (a.drops) {
            const uint4 w = philox(q, key);
            y = SLOPES ? make_float4(mul_bwd(y.x, a.keep.s, d[k].x, a.keep.off), mul_bwd(y.y, a.keep.s, d[k].y, a.keep.off), mul_bwd(y.z, a.keep.s, d[k].z, a.keep.off),
                                     mul_bwd(y.w, a.keep.s, d[k].w, a.keep.off))
                       : a.keep.of(y);
            y = make_float4(w.x < a.drop.below ? 0.0f : y.x, w.y < a.drop.below ? 0.0f : y.y, w.z < a.drop.below ? 0.0f : y.z, w.w < a.drop.below ? 0.0f : y.w);
        }
        reinterpret_cast<float4*>(out)[q] = y;
    }
}

// Rows of any length of at least four and at any address, fewer than 2^31 elements: quads of the output, most of which lie within a row.
template <bool SLOPES>
__global__ void __launch_bounds__(kThreads) embed_odd_kernel(const Embedding a, const float* g, float* out, uint32_t n, Divide by_row, Divide by_pos) {
    const uint32_t q = blockIdx.x * kThreads + threadIdx.x, e = q * 4;
    if (e >= n) return;
    const uint2 key = a.drops ? key_of(a.drop) : make_uint2(0u, 0u);
    const uint32_t i = by_row(e), c = e - i * by_row.d;
    const auto at = [&](uint32_t column, int64_t token) {
        float x = quiet_nan();
        if ((uint64_t)token < (uint64_t)a.vocab) x = __ldg(a.table + token * a.table_row + column);
        return x;
    };
    const auto place = [&](uint32_t row, uint32_t column) { return a.pos ? __ldg(a.pos + (int64_t)(row - by_pos(row) * by_pos.d) * a.pos_row + column) : 0.0f; };
    const int64_t token = token_at(a.tokens, i);
    float x[4], p[4], d[4];
    int64_t next = -1;
    if (c + 3 >= by_row.d && i + 1 < (uint32_t)a.count) next = token_at(a.tokens, i + 1);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const bool behind = c + k >= by_row.d;
        const uint32_t row = i + behind, column = c + k - (behind ? by_row.d : 0u);
        x[k] = p[k] = d[k] = 0.0f;
        if (e + k >= n) continue;
        x[k] = at(column, behind ? next : token);
        p[k] = place(row, column);
        if (SLOPES) d[k] = __ldg(g + e + k);
    }
    float4 y = make_float4(x[0], x[1], x[2], x[3]);
    if (a.scaled) y = a.scale.of(y);
    if (a.pos) y = make_float4(fadd(y.x, p[0]), fadd(y.y, p[1]), fadd(y.z, p[2]), fadd(y.w, p[3]));
    if (a.drops) {
        const uint4 w = philox(q, key);
        if (!SLOPES) y = a.keep.of(y);
        const auto last = [&](float v, uint32_t bits, float dv) { return bits < a.drop.below ? 0.0f : SLOPES ? mul_bwd(v, a.keep.s, dv, a.keep.off) : v; };
        y = make_float4(last(y.x, w.x, d[0]), last(y.y, w.y, d[1]), last(y.z, w.z, d[2]), last(y.w, w.w, d[3]));
    }
    const float v[4] = {y.x, y.y, y.z, y.w};
    if (aligned16(out) && e + 4 <= n)
        reinterpret_cast<float4*>(out)[q] = y;
    else
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (e + k < n) out[e + k] = v[k];
}

// ---- the order of the tokens ------------------------------------------------------------------------------------

// Tokens that count each other (10000 words of 512 columns, dropout, backward: 2048 tokens 23 us, 29 by digits; 4096 29 and 30; 8192 49 and 35); a CTA's, one of a lane.
constexpr int kMostCounted = 4096, kRanked = 32;
// (Tiles of 1024: what a warp does one after the other, ranks by __match_any_sync of many different digits above all, takes 0.5 us for 32 tokens.  65536 tokens of 512 columns backward:
// 86 us with tiles of 4096, 78 of 2048, 72.)
constexpr int kTileThreads = 512, kTileWarps = kTileThreads / 32, kRounds = 2, kTile = kTileThreads * kRounds;
constexpr int kMostTiles = 296;           // each reads the counts of all (2^19 tokens of 4000000 words backward: 512 of them 320 us, 296 173; 2^22 of 200000 788 and 807)
constexpr uint32_t kNone = 0xffffffffu;

struct Entry { uint32_t token, place; };

struct Sort {
    const int64_t* tokens;
    int64_t count, vocab, padding;
    int low_bits, high_bits;
    int tiles, tile;                      // of `tile` tokens, a multiple of kTile
    uint32_t *counts_low, *counts_high;   // [tiles][1 << bits]
    Entry *by_low, *sorted;
    uint32_t* totals;                     // [0]: tokens that have a gradient; [1], [2]: those in several chunks, in many
    float* zeros;                         // the gradient
    int64_t zero_count;
    int fillers;                          // CTAs that fill
};

// A share of the zeros: part `part` of `parts`, by the CTAs from `first` on.
__device__ void fill(const Sort& a, int first, int part, int parts) {
    const int64_t quads = aligned16(a.zeros) ? a.zero_count / 4 : 0, per = (quads + parts - 1) / parts, begin = per * part, end = min(begin + per, quads);
    const int64_t mine = (int64_t)(blockIdx.x - first) * blockDim.x + threadIdx.x, stride = (int64_t)a.fillers * blockDim.x;
    const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float4* to = reinterpret_cast<float4*>(a.zeros) + begin + mine;
    int64_t left = end - begin - mine;
    for (; left > 3 * stride; left -= 4 * stride, to += 4 * stride) {
        to[0] = zero;
        to[stride] = zero;
        to[2 * stride] = zero;
        to[3 * stride] = zero;
    }
    for (; left > 0; left -= stride, to += stride) *to = zero;
    if (part == parts - 1)                            // (what is no whole quad; all of them at an odd address)
        for (int64_t e = quads * 4 + mine; e < a.zero_count; e += stride) a.zeros[e] = 0.0f;
}

__device__ __forceinline__ uint32_t token_of(const Sort& a, int64_t i) {
    if (i >= a.count) return kNone;
    const int64_t token = token_at(a.tokens, i);
    return (uint64_t)token < (uint64_t)a.vocab && token != a.padding ? (uint32_t)token : kNone;
}

// How many of the warp's earlier elements have the same digit (kNone: no element), which its counts are left with.
template <int ROUNDS>
__device__ __forceinline__ void rank_in_warp(uint16_t* counts, const uint32_t (&digit)[ROUNDS], uint32_t (&rank)[ROUNDS]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool is = digit[r] != kNone;
        const uint32_t peers = __match_any_sync(0xffffffffu, digit[r]);
        const uint32_t before = is ? counts[digit[r]] : 0u;
        rank[r] = before + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (is && lane == __ffs(peers) - 1) counts[digit[r]] = (uint16_t)(before + __popc(peers));
        __syncwarp();
    }
}

// Sums before each of the n <= 2 * 1024 values in shared memory, in place; `warps` holds a value for each warp.  Ends with a barrier.
__device__ uint32_t sums_before(uint32_t* values, int n, uint32_t* warps) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, threads = blockDim.x, each = (n + threads - 1) / threads;
    uint32_t own[4], sum = 0u;
    __syncthreads();
    for (int k = 0; k < each; ++k) {
        own[k] = t * each + k < n ? values[t * each + k] : 0u;
        sum += own[k];
    }
    uint32_t upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) warps[warp] = upto;
    __syncthreads();
    uint32_t before = upto - sum, total = 0u;
    for (int w = 0; w < threads / 32; ++w) {
        if (w < warp) before += warps[w];
        total += warps[w];
    }
    for (int k = 0; k < each; ++k) {
        if (t * each + k < n) values[t * each + k] = before;
        before += own[k];
    }
    __syncthreads();
    return total;
}

// counts [warps][bins] -> what the warps before have, in place; totals [bins]
__device__ void sums_over_warps(uint16_t* counts, uint32_t* totals, int bins, int warps) {
    for (int b = threadIdx.x; b < bins; b += blockDim.x) {
        uint32_t run = 0u;
        for (int w = 0; w < warps; ++w) {
            const uint32_t c = counts[w * bins + b];
            counts[w * bins + b] = (uint16_t)run;
            run += c;
        }
        totals[b] = run;
    }
}

// A lane has a token and each warp of the CTA a part of the others: those before it in the order are its place there.
__global__ void __launch_bounds__(kThreads) rank_kernel(const Sort a, int rankers) {
    __shared__ __align__(16) uint32_t tokens[kMostCounted];
    __shared__ uint32_t before[kThreads / 32][kRanked];
    __shared__ uint32_t live[kThreads / 32];
    if ((int)blockIdx.x >= rankers) {
        fill(a, rankers, 0, 1);
        next_may_start();
        return;
    }
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, count = (int)a.count, padded = (count + 3) / 4 * 4;
    uint32_t mine = 0u, loaded[kMostCounted / kThreads];
#pragma unroll
    for (int k = 0; k < kMostCounted / kThreads; ++k) loaded[k] = token_of(a, t + k * kThreads);
#pragma unroll
    for (int k = 0; k < kMostCounted / kThreads; ++k) {
        if (t + k * kThreads < padded) tokens[t + k * kThreads] = loaded[k];
        mine += loaded[k] != kNone;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) live[warp] = mine;
    __syncthreads();
    const int first = blockIdx.x * kRanked, i = first + lane;
    const uint32_t own = i < count ? tokens[i] : kNone;
    // (whole quads before the CTA's tokens, around them, behind them)
    const int quads = padded / 4, each = (quads + kThreads / 32 - 1) / (kThreads / 32), from = min(warp * each, quads), to = min(from + each, quads);
    const int around = min(max(first / 4, from), to), behind = min(max((first + kRanked) / 4, from), to);
    uint32_t less = 0u;
    const uint4* quad = reinterpret_cast<const uint4*>(tokens);
#pragma unroll 4
    for (int q = from; q < around; ++q) {
        const uint4 v = quad[q];
        less += (v.x <= own) + (v.y <= own) + (v.z <= own) + (v.w <= own);
    }
    for (int j = around * 4; j < behind * 4; ++j) less += tokens[j] < own || (tokens[j] == own && j < i);
#pragma unroll 4
    for (int q = behind; q < to; ++q) {
        const uint4 v = quad[q];
        less += (v.x < own) + (v.y < own) + (v.z < own) + (v.w < own);
    }
    before[warp][lane] = less;
    __syncthreads();
    if (t < kRanked && own != kNone) {
        for (int w = 1; w < kThreads / 32; ++w) less += before[w][lane];
        a.sorted[less] = {own, (uint32_t)i};
    }
    if (blockIdx.x == 0 && t == 0) {
        for (int w = 1; w < kThreads / 32; ++w) mine += live[w];
        a.totals[0] = mine;
        a.totals[1] = a.totals[2] = 0u;
    }
    next_may_start();
}

// The low digits of each tile of tokens.
__global__ void __launch_bounds__(kTileThreads) count_kernel(const Sort a) {
    extern __shared__ __align__(16) unsigned char memory[];
    if ((int)blockIdx.x >= a.tiles) {
        fill(a, a.tiles, 0, 3);
        next_may_start();
        return;
    }
    uint32_t* counts = reinterpret_cast<uint32_t*>(memory);
    const int bins = 1 << a.low_bits, high = 1 << a.high_bits;
    for (int b = threadIdx.x; b < bins; b += kTileThreads) counts[b] = 0u;
    for (int b = threadIdx.x; b < high; b += kTileThreads) a.counts_high[(int64_t)blockIdx.x * high + b] = 0u;
    if (blockIdx.x == 0 && threadIdx.x < 3) a.totals[threadIdx.x] = 0u;
    __syncthreads();
    const int64_t begin = (int64_t)blockIdx.x * a.tile;
    for (int i = threadIdx.x; i < a.tile; i += kTile) {
        uint32_t token[kRounds];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) token[r] = token_of(a, begin + i + r * kTileThreads);
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
            if (token[r] != kNone) atomicAdd(&counts[token[r] & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kTileThreads) a.counts_low[(int64_t)blockIdx.x * bins + b] = counts[b];
    next_may_start();
}

// Moves the elements of a tile to their places by one digit.  The counts of all tiles say where each starts.
template <bool HIGH>
__global__ void __launch_bounds__(kTileThreads) scatter_kernel(const Sort a) {
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ uint32_t warp_sums[kTileWarps];
    if ((int)blockIdx.x >= a.tiles) {
        // (not before the launch in front has ended: a chain of launches ends in their order only if each waits for the one before)
        after_previous();
        fill(a, a.tiles, HIGH ? 2 : 1, 3);
        next_may_start();
        return;
    }
    const int bits = HIGH ? a.high_bits : a.low_bits, bins = 1 << bits, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    uint32_t* start = reinterpret_cast<uint32_t*>(memory);                            // where the tile's next element of each digit goes
    uint32_t* totals = start + bins;
    uint16_t* counts = reinterpret_cast<uint16_t*>(totals + bins);
    for (int b = t; b < bins; b += kTileThreads) start[b] = totals[b] = 0u;
    __syncthreads();
    after_previous();
    const int64_t tile_begin = (int64_t)blockIdx.x * a.tile;
    uint32_t token[kRounds], place[kRounds], digit[kRounds], rank[kRounds];
    const auto load = [&](int64_t begin) {            // (of the second pass also what lies behind the last one: it is not looked at)
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int64_t i = begin + (warp * kRounds + r) * 32 + lane;
            if (HIGH) {
                const uint2 e = i < a.count ? __ldcg(reinterpret_cast<const uint2*>(a.by_low) + i) : make_uint2(kNone, 0u);
                token[r] = e.x;
                place[r] = e.y;
            } else {
                token[r] = token_of(a, i);
                place[r] = (uint32_t)i;
            }
        }
    };
    load(tile_begin);
    {
        // a thread adds four neighbouring digits of every so-many-th tile
        const uint4* all = reinterpret_cast<const uint4*>(HIGH ? a.counts_high : a.counts_low);
        const int quad_bits = bits - 2, quad = t & ((1 << quad_bits) - 1), groups = kTileThreads >> quad_bits;
        uint4 sum = make_uint4(0u, 0u, 0u, 0u), before = sum;
#pragma unroll 8
        for (int k = t >> quad_bits; k < a.tiles; k += groups) {
            const uint4 v = __ldcg(all + ((int64_t)k << quad_bits) + quad);
            sum = make_uint4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
            if (k < (int)blockIdx.x) before = make_uint4(before.x + v.x, before.y + v.y, before.z + v.z, before.w + v.w);
        }
        const uint32_t s[4] = {sum.x, sum.y, sum.z, sum.w}, p[4] = {before.x, before.y, before.z, before.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (s[k]) atomicAdd(&start[quad * 4 + k], s[k]);
            if (p[k]) atomicAdd(&totals[quad * 4 + k], p[k]);
        }
    }
    const uint32_t live = sums_before(start, bins, warp_sums);
    for (int b = t; b < bins; b += kTileThreads) start[b] += totals[b];
    if (!HIGH && blockIdx.x == 0 && t == 0) a.totals[0] = live;
    const int64_t tile_end = min(tile_begin + a.tile, HIGH ? (int64_t)live : a.count);
    for (int64_t begin = tile_begin; begin < tile_end; begin += kTile) {
        if (begin != tile_begin) load(begin);
        for (int i = t; i < bins * kTileWarps / 2; i += kTileThreads) reinterpret_cast<uint32_t*>(counts)[i] = 0u;
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const bool is = begin + (warp * kRounds + r) * 32 + lane < tile_end && token[r] != kNone;
            digit[r] = !is ? kNone : HIGH ? token[r] >> a.low_bits : token[r] & (bins - 1);
        }
        __syncthreads();
        rank_in_warp<kRounds>(counts + warp * bins, digit, rank);
        __syncthreads();
        sums_over_warps(counts, totals, bins, kTileWarps);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            if (digit[r] == kNone) continue;
            const uint32_t to = start[digit[r]] + counts[warp * bins + digit[r]] + rank[r];
            (HIGH ? a.sorted : a.by_low)[to] = {token[r], place[r]};
            if (!HIGH) atomicAdd(a.counts_high + ((int64_t)(to / (uint32_t)a.tile) << a.high_bits) + (token[r] >> a.low_bits), 1u);
        }
        __syncthreads();
        for (int b = t; b < bins; b += kTileThreads) start[b] += totals[b];
        __syncthreads();
    }
    next_may_start();
}

// ---- sums ---------------------------------------------------------------------------------------------------------

constexpr int kColumns = 128;             // of a warp: four of a lane

struct Sums {
    const float *g, *table;
    float* dw;
    const Entry* sorted;
    uint32_t* totals;
    float* parts;                         // [chunks][2][dim]: what continues from the chunk before; what the next continues
    uint32_t* list;                       // chunks in which a token starts that the next continues, from the back those of the tokens that go on in many
    int64_t table_row;
    int dim, slabs, chunk;
    uint32_t chunks;
    bool scaled, drops;
    Times scale, keep;
    Dropping drop;
};

constexpr uint32_t kMany = 12;            // chunks of a token that a warp adds alone (its loads wait twice; 2^18 tokens of 4 columns backward: 48 chunks 73.4 us, 24 71.3, 12 69.9)

__device__ __forceinline__ Entry entry_at(const Entry* sorted, uint32_t i) {
    const uint2 e = __ldcg(reinterpret_cast<const uint2*>(sorted) + i);
    return {e.x, e.y};
}

// A lane has four neighbouring columns.  VEC: rows of whole quads at aligned addresses.
__device__ __forceinline__ int column(int slab, int lane) { return slab * kColumns + lane * 4; }

template <bool VEC>
__device__ __forceinline__ void load_columns(const float* row, int slab, int lane, int dim, float (&v)[4]) {
    const int c = column(slab, lane);
    if (VEC) {
        const float4 x = c < dim ? __ldg(reinterpret_cast<const float4*>(row + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = c + k < dim ? __ldg(row + c + k) : 0.0f;
    }
}

template <bool VEC>
__device__ __forceinline__ void store_columns(float* row, int slab, int lane, int dim, const float (&v)[4]) {
    const int c = column(slab, lane);
    if (VEC) {
        if (c < dim) *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k < dim) row[c + k] = v[k];
    }
}

// Bound by instructions with dropout (194 for each quad of a row, 70 of them its random bits): 64 x 1024 rows of 512 columns in 70 us, by the trips to memory without.  Four CTAs per
// SM with four rows on their way each, not three with eight: 4 us less with dropout and without, of 103 and 71 for all of the backward pass.
template <bool VEC, bool SLOPES>
__global__ void __launch_bounds__(kThreads, 4) sum_kernel(const Sums a) {
    constexpr int kAhead = 4;             // rows on their way
    const int lane = threadIdx.x & 31;
    const uint32_t unit = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const uint32_t chunk = unit / (uint32_t)a.slabs;
    const int slab = (int)(unit - chunk * a.slabs);
    after_previous();
    const uint32_t live = __ldcg(a.totals), begin = chunk * (uint32_t)a.chunk;
    if (chunk >= a.chunks || begin >= live) return;
    const int n = (int)min((uint32_t)a.chunk, live - begin);
    const uint2 key = a.drops ? key_of(a.drop) : make_uint2(0u, 0u);
    const Entry mine = lane < n ? entry_at(a.sorted, begin + lane) : Entry{kNone, 0u};
    const uint32_t token_before = begin > 0 ? entry_at(a.sorted, begin - 1).token : kNone;
    const uint32_t token_after = begin + n < live ? entry_at(a.sorted, begin + n).token : kNone;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, slope[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    uint32_t now = kNone;
    for (int first = 0; first < n; first += kAhead) {
        float v[kAhead][4];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const uint32_t place = __shfl_sync(0xffffffffu, mine.place, (first + j) & 31);
            if (first + j < n) load_columns<VEC>(a.g + (int64_t)place * a.dim, slab, lane, a.dim, v[j]);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (first + j >= n) break;
            const uint32_t token = __shfl_sync(0xffffffffu, mine.token, first + j), place = __shfl_sync(0xffffffffu, mine.place, first + j);
            if (token != now) {
                // a token ends and one starts
                if (now != kNone) {
                    const bool whole = now != token_before;
                    store_columns<VEC>(whole ? a.dw + (int64_t)now * a.dim : a.parts + (int64_t)chunk * 2 * a.dim, slab, lane, a.dim, sum);
                }
                now = token;
                sum[0] = sum[1] = sum[2] = sum[3] = 0.0f;
                if (SLOPES && a.scaled) {
                    load_columns<VEC>(a.table + (int64_t)token * a.table_row, slab, lane, a.dim, slope);
#pragma unroll
                    for (int k = 0; k < 4; ++k) slope[k] = mul_slope(slope[k], a.scale.s, a.scale.off);
                }
            }
            float4 x = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
            if (a.drops) {
                const uint64_t e = (uint64_t)place * a.dim + column(slab, lane);
                uint4 w = philox(e >> 2, key);
                if (!VEC && a.dim % 4) {              // (the four may lie in two blocks)
                    const uint4 next = philox((e >> 2) + 1, key);
                    if (e & 1) w = make_uint4(w.y, w.z, w.w, next.x);
                    if (e & 2) w = e & 1 ? make_uint4(w.z, w.w, next.y, next.z) : make_uint4(w.z, w.w, next.x, next.y);
                }
                x = a.keep.of(x);
                x = make_float4(w.x < a.drop.below ? 0.0f : x.x, w.y < a.drop.below ? 0.0f : x.y, w.z < a.drop.below ? 0.0f : x.z, w.w < a.drop.below ? 0.0f : x.w);
            }
            if (a.scaled) x = SLOPES ? make_float4(fmul(x.x, slope[0]), fmul(x.y, slope[1]), fmul(x.z, slope[2]), fmul(x.w, slope[3])) : a.scale.of(x);
            sum[0] = fadd(sum[0], x.x);
            sum[1] = fadd(sum[1], x.y);
            sum[2] = fadd(sum[2], x.z);
            sum[3] = fadd(sum[3], x.w);
        }
    }
    const bool from_before = now == token_before, goes_on = now == token_after;
    if (!from_before && !goes_on) {
        store_columns<VEC>(a.dw + (int64_t)now * a.dim, slab, lane, a.dim, sum);
    } else {
        store_columns<VEC>(a.parts + ((int64_t)chunk * 2 + !from_before) * a.dim, slab, lane, a.dim, sum);
        if (!from_before && slab == 0 && lane == 0) {
            const uint64_t far = (uint64_t)(chunk + kMany) * a.chunk;
            if (far < live && entry_at(a.sorted, (uint32_t)far).token == now)
                a.list[a.chunks - 1 - atomicAdd(a.totals + 2, 1u)] = chunk;
            else
                a.list[atomicAdd(a.totals + 1, 1u)] = chunk;
        }
    }
    next_may_start();
}

// A token's parts from..to - 1: the end of the chunk that it starts in, the beginnings of those that it goes on in.  Those that are on their way together are added pair by pair in
// 32 bits, these sums in 64: there may be 2^26 parts, and the error does not grow with them.  (2^20 rows of one token, 128 columns, backward: 735 us, with every part in 64 bits 833; 4096 of
// 512 28.7, in 32 bits alone 28.1.)
template <bool VEC, int kAhead>
__device__ __forceinline__ void add_parts(const Sums& a, uint32_t chunk, uint32_t from, uint32_t to, int slab, int lane, double (&sum)[4]) {
    const int c = column(slab, lane);
    for (uint32_t first = from; first < to; first += kAhead) {
        float v[kAhead][4];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const uint32_t part = first + j;
            v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.0f;
            if (part >= to) continue;
            const float* row = a.parts + ((int64_t)(chunk + part) * 2 + (part == 0)) * a.dim;
            if (VEC) {
                const float4 x = c < a.dim ? __ldcg(reinterpret_cast<const float4*>(row + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                v[j][0] = x.x, v[j][1] = x.y, v[j][2] = x.z, v[j][3] = x.w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[j][k] = c + k < a.dim ? __ldcg(row + c + k) : 0.0f;
            }
        }
#pragma unroll
        for (int apart = 1; apart < kAhead; apart *= 2)
#pragma unroll
            for (int j = 0; j < kAhead; j += 2 * apart)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[j][k] = fadd(v[j][k], v[j + apart][k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += v[0][k];
    }
}

// How many parts the token has that starts in this chunk: a warp looks at the next 32 chunks, then at 32 places of what is left, and so on.
__device__ __forceinline__ uint32_t parts_of(const Sums& a, uint32_t chunk, uint32_t live, int lane, uint32_t* token) {
    *token = entry_at(a.sorted, (chunk + 1) * (uint32_t)a.chunk).token;
    uint32_t last = chunk + 1, end = a.chunks, step = 1;              // chunks that begin with the token, and with another or behind the last one
    for (;; step = (end - last + 31) / 32) {
        const uint64_t at = (last + (uint64_t)step * (lane + 1)) * a.chunk;
        const uint32_t other = __ballot_sync(0xffffffffu, at >= live || entry_at(a.sorted, (uint32_t)at).token != *token);
        if (other) end = min(end, last + step * __ffs(other));
        last += step * (other ? __ffs(other) - 1 : 32);
        if (last + 1 >= end) return end - chunk;
    }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads, 2) join_kernel(const Sums a) {
    constexpr int kWarps = kThreads / 32;
    __shared__ double stage[kWarps][kColumns];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slab = blockIdx.y;
    after_previous();
    const uint32_t live = __ldcg(a.totals), some = __ldcg(a.totals + 1), many = __ldcg(a.totals + 2);
    uint32_t token;
    for (uint32_t i = blockIdx.x; i < many; i += gridDim.x) {
        // a warp has neighbouring parts
        const uint32_t chunk = __ldcg(a.list + a.chunks - 1 - i), count = parts_of(a, chunk, live, lane, &token);
        const uint32_t each = (count + kWarps - 1) / kWarps, from = min(warp * each, count), to = min(from + each, count);
        double sum[4] = {0.0, 0.0, 0.0, 0.0};
        add_parts<VEC, VEC ? 16 : 8>(a, chunk, from, to, slab, lane, sum);
#pragma unroll
        for (int k = 0; k < 4; ++k) stage[warp][lane * 4 + k] = sum[k];
        __syncthreads();
        if (threadIdx.x < kColumns && slab * kColumns + threadIdx.x < a.dim) {
            double s = stage[0][threadIdx.x];
            for (int w = 1; w < kWarps; ++w) s += stage[w][threadIdx.x];
            a.dw[(int64_t)token * a.dim + slab * kColumns + threadIdx.x] = (float)s;
        }
        __syncthreads();
    }
    for (uint32_t i = blockIdx.x * kWarps + warp; i < some; i += gridDim.x * kWarps) {
        const uint32_t chunk = __ldcg(a.list + i), count = parts_of(a, chunk, live, lane, &token);
        double sum[4] = {0.0, 0.0, 0.0, 0.0};
        add_parts<VEC, 8>(a, chunk, 0u, count, slab, lane, sum);
        const float rounded[4] = {(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]};
        store_columns<VEC>(a.dw + (int64_t)token * a.dim, slab, lane, a.dim, rounded);
    }
}

constexpr int64_t kMostTokens = 0x7fffffff, kMostRows = 1 << 22;

int check_sizes(const Embedding& a, double p) {
    if (a.count < 0 || a.dim < 0 || a.vocab < 0 || !(p >= 0.0 && p < 1.0) || (a.pos && (a.pos_count < 1 || a.count % a.pos_count))) return PAMK_ERR_ARG;
    if (a.count > kMostTokens || a.vocab > kMostRows) return PAMK_ERR_SIZE;
    return PAMK_OK;
}

Embedding described(const int64_t* tokens, const float* table, const float* pos, int64_t count, int64_t vocab, int64_t dim, int64_t table_row,
                    int64_t pos_row, int64_t pos_count, int64_t padding, int scaled, float scale, double p, const int64_t* seed_at, int64_t seed, float offset) {
    Embedding a{};
    a.tokens = tokens;
    a.table = table;
    a.pos = pos;
    a.count = count;
    a.table_row = table_row;
    a.pos_row = pos_row;
    a.pos_count = pos_count;
    a.vocab = vocab;
    a.padding = padding;
    a.dim = (int)dim;
    a.scaled = scaled != 0;
    a.scale = Times(scale, offset_bits(offset));
    a.drops = p > 0.0;
    if (a.drops) {
        a.drop = dropping(p, seed_at, seed);
        a.keep = Times(a.drop.scale, offset_bits(offset));
    }
    return a;
}

// How the gradient of a table is worked on, and where its scratch lies.
struct Plan {
    int low_bits, high_bits, tiles, tile, chunk;
    int64_t chunks;
    size_t totals, counts_low, counts_high, by_low, sorted, list, parts, bytes;
};

Plan planned(int64_t count, int64_t vocab, int64_t dim) {
    Plan p{};
    int bits = 4;                         // (digits of two at least, whose counts are read by four)
    while (((int64_t)1 << bits) < vocab) ++bits;
    p.low_bits = (bits + 1) / 2;
    p.high_bits = bits - p.low_bits;
    if (count > kMostCounted) {
        const int64_t each = (count + kMostTiles - 1) / kMostTiles;
        p.tile = (int)((each + kTile - 1) / kTile * kTile);
        p.tiles = (int)((count + p.tile - 1) / p.tile);
    }
    p.chunk = count > 32768 ? 32 : 16;    // (2^20 tokens of 128 columns backward: 16 rows 261 us, 32 221; 4096 of 512: 28.3 and 34.9)
    p.chunks = (count + p.chunk - 1) / p.chunk;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.totals = take(3 * sizeof(uint32_t));
    p.counts_low = take((size_t)p.tiles << p.low_bits << 2);
    p.counts_high = take((size_t)p.tiles << p.high_bits << 2);
    p.by_low = take(p.tiles ? (size_t)count * sizeof(Entry) : 0);
    p.sorted = take((size_t)count * sizeof(Entry));
    p.list = take((size_t)p.chunks * sizeof(uint32_t));
    p.parts = take((size_t)p.chunks * 2 * (size_t)dim * sizeof(float));
    p.bytes = at;
    return p;
}

// (what the kernels may ask for, whatever a call needs: calls of two threads set the same)
constexpr int kMostBins = 1 << 11;
constexpr size_t kTileMemory = kMostBins * 8 + kMostBins * kTileWarps * 2;
static_assert(kTileMemory <= 100 * 1024);

template <class K>
int allow(K* kernel, size_t memory, size_t most) {
    if (memory <= 40 * 1024) return PAMK_OK;
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
}

template <class... P, class... A>
int launch_next(void (*kernel)(P...), dim3 grid, unsigned threads, size_t memory, cudaStream_t st, A... args) {
    cudaLaunchAttribute overlap{};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = memory;
    config.stream = st;
    config.attrs = &overlap;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
    count_launch();
    return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
}

int sort_tokens(const Plan& p, Sort s, cudaStream_t st) {
    const int64_t fill_ctas = (s.zero_count + kThreads * 16 - 1) / (kThreads * 16);
    if (!p.tiles) {
        const int rankers = (int)((s.count + kRanked - 1) / kRanked);
        s.fillers = (int)(fill_ctas < 8 * sm_count() ? fill_ctas : 8 * sm_count());
        rank_kernel<<<rankers + s.fillers, kThreads, 0, st>>>(s, rankers);
        return check_launch();
    }
    s.fillers = (int)(fill_ctas < 4 * sm_count() ? fill_ctas : 4 * sm_count());
    const size_t low = ((size_t)8 << p.low_bits) + ((size_t)kTileWarps * 2 << p.low_bits), high = ((size_t)8 << p.high_bits) + ((size_t)kTileWarps * 2 << p.high_bits);
    if (const int status = allow(scatter_kernel<false>, low, kTileMemory)) return status;
    if (const int status = allow(scatter_kernel<true>, high, kTileMemory)) return status;
    const unsigned ctas = (unsigned)(p.tiles + s.fillers);
    count_kernel<<<ctas, kTileThreads, (size_t)4 << p.low_bits, st>>>(s);
    if (const int status = check_launch()) return status;
    if (const int status = launch_next(scatter_kernel<false>, dim3(ctas), kTileThreads, low, st, s)) return status;
    return launch_next(scatter_kernel<true>, dim3(ctas), kTileThreads, high, st, s);
}

}  // namespace
}  // namespace pamk

extern "C" {

int pamk_embedding(const int64_t* tokens, const float* table, const float* positions, const float* dy, float* out, int64_t count, int64_t vocab, int64_t dim,
                   int64_t table_row, int64_t positions_row, int64_t positions_count, int has_scale, float scale, double p, const int64_t* seed_at, int64_t seed,
                   float offset, void* stream) {
    using namespace pamk;
    if (dim < 0 || dim > 0x7fffffff - 4) return dim < 0 ? PAMK_ERR_ARG : PAMK_ERR_SIZE;
    const Embedding a = described(tokens, table, positions, count, vocab, dim, table_row, positions_row, positions_count, -1, has_scale, scale, p, seed_at, seed, offset);
    if (const int status = check_sizes(a, p)) return status;
    if (count == 0 || dim == 0) return PAMK_OK;
    if (!tokens || !out || (vocab > 0 && !table) || (dy && !a.drops)) return PAMK_ERR_ARG;
    const int64_t n = count * dim;
    const auto st = (cudaStream_t)stream;
    if (dim % 4 == 0 && n < ((int64_t)1 << 33) && aligned16(table) && table_row % 4 == 0 && aligned16(positions) && positions_row % 4 == 0 && aligned16(dy) && aligned16(out)) {
        const uint32_t quads = (uint32_t)(n / 4);
        const Divide by_row((uint32_t)(dim / 4)), by_pos(positions ? (uint32_t)positions_count : 1u);
        // (of sentences at one position: two at least, and positions enough for a wave of CTAs or so)
        const int64_t sentence = positions_count * (dim / 4), sentences = positions && positions_count > 1 ? count / positions_count : 1;
        const int64_t groups = (sentences + kQuads - 1) / kQuads;
        if (sentences >= 2 && groups <= 65535 && sentence >= kThreads) {
            const dim3 grid((unsigned)((sentence + kThreads - 1) / kThreads), (unsigned)groups);
            (dy ? embed_quads_kernel<true, true> : embed_quads_kernel<false, true>)<<<grid, kThreads, 0, st>>>(a, dy, out, quads, by_row, by_pos);
        } else {
            const uint32_t ctas = (quads + kThreads * kQuads - 1) / (kThreads * kQuads);
            (dy ? embed_quads_kernel<true, false> : embed_quads_kernel<false, false>)<<<ctas, kThreads, 0, st>>>(a, dy, out, quads, by_row, by_pos);
        }
        return check_launch();
    }
    if (dim >= 4 && n < ((int64_t)1 << 31) - 4) {
        const uint32_t ctas = (uint32_t)((n + 4 * kThreads - 1) / (4 * kThreads));
        (dy ? embed_odd_kernel<true> : embed_odd_kernel<false>)<<<ctas, kThreads, 0, st>>>(a, dy, out, (uint32_t)n, Divide((uint32_t)dim),
                                                                                          Divide(positions ? (uint32_t)positions_count : 1u));
        return check_launch();
    }
    const int64_t ctas = (n + 4 * kThreads - 1) / (4 * kThreads);
    if (ctas > 0x7fffffff) return PAMK_ERR_SIZE;
    (dy ? embed_kernel<true> : embed_kernel<false>)<<<(unsigned)ctas, kThreads, 0, st>>>(a, dy, out);
    return check_launch();
}

size_t pamk_embedding_bwd_workspace_bytes(int64_t count, int64_t vocab, int64_t dim) {
    using namespace pamk;
    if (count < 1 || count > kMostTokens || vocab < 1 || vocab > kMostRows || dim < 1 || dim > 0x7fffffff - 4) return 0;
    return planned(count, vocab, dim).bytes;
}

int pamk_embedding_bwd(const int64_t* tokens, const float* dy, const float* table, float* dtable, int64_t count, int64_t vocab, int64_t dim, int64_t table_row,
                       int64_t padding, int has_scale, float scale, double p, const int64_t* seed_at, int64_t seed, float offset, int approx_bwd, void* workspace,
                       size_t workspace_bytes, void* stream) {
    using namespace pamk;
    if (dim < 0 || dim > 0x7fffffff - 4) return dim < 0 ? PAMK_ERR_ARG : PAMK_ERR_SIZE;
    const Embedding a = described(tokens, table, nullptr, count, vocab, dim, table_row, 0, 0, padding, has_scale, scale, p, seed_at, seed, offset);
    if (const int status = check_sizes(a, p)) return status;
    if (vocab == 0 || dim == 0) return PAMK_OK;
    if (!dtable || (count > 0 && (!tokens || !dy)) || (!approx_bwd && (a.drops || (has_scale && !table)))) return PAMK_ERR_ARG;
    const auto st = (cudaStream_t)stream;
    if (count == 0) {
        const cudaError_t err = cudaMemsetAsync(dtable, 0, (size_t)vocab * dim * sizeof(float), st);
        return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
    }
    const Plan plan = planned(count, vocab, dim);
    const int64_t slabs = (dim + kColumns - 1) / kColumns, ctas = (plan.chunks * slabs + kThreads / 32 - 1) / (kThreads / 32);
    if (slabs > 65535 || ctas > (1 << 28)) return PAMK_ERR_SIZE;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < plan.bytes) return PAMK_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    Sort s{};
    s.tokens = tokens;
    s.count = count;
    s.vocab = vocab;
    s.padding = padding;
    s.low_bits = plan.low_bits;
    s.high_bits = plan.high_bits;
    s.tiles = plan.tiles;
    s.tile = plan.tile;
    s.counts_low = reinterpret_cast<uint32_t*>(ws + plan.counts_low);
    s.counts_high = reinterpret_cast<uint32_t*>(ws + plan.counts_high);
    s.by_low = reinterpret_cast<Entry*>(ws + plan.by_low);
    s.sorted = reinterpret_cast<Entry*>(ws + plan.sorted);
    s.totals = reinterpret_cast<uint32_t*>(ws + plan.totals);
    s.zeros = dtable;
    s.zero_count = vocab * dim;
    if (const int status = sort_tokens(plan, s, st)) return status;
    Sums u{};
    u.g = dy;
    u.table = table;
    u.dw = dtable;
    u.sorted = s.sorted;
    u.totals = s.totals;
    u.parts = reinterpret_cast<float*>(ws + plan.parts);
    u.list = reinterpret_cast<uint32_t*>(ws + plan.list);
    u.table_row = table_row;
    u.dim = (int)dim;
    u.slabs = (int)slabs;
    u.chunk = plan.chunk;
    u.chunks = (uint32_t)plan.chunks;
    u.scaled = a.scaled;
    u.drops = a.drops;
    u.scale = a.scale;
    u.keep = a.keep;
    u.drop = a.drop;
    const bool slopes = !approx_bwd && a.scaled;
    const bool vec = dim % 4 == 0 && aligned16(dy) && aligned16(dtable) && (!slopes || (aligned16(table) && table_row % 4 == 0));
    const auto sums = vec ? (slopes ? sum_kernel<true, true> : sum_kernel<true, false>) : (slopes ? sum_kernel<false, true> : sum_kernel<false, false>);
    if (const int status = launch_next(sums, dim3((unsigned)ctas), kThreads, 0, st, u)) return status;
    const int64_t wide = (2 * sm_count() + slabs - 1) / slabs;
    const unsigned joins = (unsigned)(plan.chunks < wide ? plan.chunks : wide);
    return launch_next(vec ? join_kernel<true> : join_kernel<false>, dim3(joins, (unsigned)slabs), kThreads, 0, st, u);
}

}
