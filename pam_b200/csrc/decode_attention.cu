// Attention of single-token rows over a key/value cache, in PAM arithmetic.
//
// For one row q of a head and the positions j that it sees (those its group shares, then its own):
//     s_j = sum_d pam(q_d, k_jd)       t_j = pam(s_j, log2 e)          m: a whole number near max_j t_j
//     e_j = exp2(t_j - m)              p_j = pad(e_j, sum_j e_j)       out_d = sum_j pam(p_j, v_jd)
// with the piecewise affine exp2 and -inf scores at probability 0, as in the chain bmm -> softmax -> bmm
// (pam/pam_ops.py:82-101, 305-328).  The chain's shift is the floor of the maximum of the whole tensor, here it is the row's own: a
// whole number either way, and exp2(t - m) = exp2(t) 2^-m exactly, so only the rounding of t - m differs.
//
// pam is not linear: pam(pad(e, S), v) summed is not pad(sum of pam(e, v), S).  A running maximum and sum with one
// joint pass over keys and values is therefore not to be had; the sum must be known before the first value is
// weighted.  So there are two passes.  The keys leave t (rows times positions, a small part of what the keys are) and each CTA's sum of exponentials with its shift,
// kept as it goes: whole shifts scale exponentials exactly.  The values read them, turn t into p on the way, and leave sums
// of products; where the positions of a row are dealt out to several CTAs, a third kernel adds these.  Where one CTA has all positions of its rows
// and they are few, it makes both passes, with t in its shared memory.
//
// Rows that see the same positions are worked on together, up to 8 per CTA: every key and value is loaded once for these (more rows are several such tiles, each of which
// loads them), by asynchronous copies into a ring that each warp has for itself, so that the warps run without barriers until their last sums.
// Keys: a lane owns a position, 32 floats of it per stage, and reads the queries from
// shared memory.  Values: a lane owns four columns.  A product is one integer and one floating-point add; the range rule
// (pam_scalar.cuh) is decided per stage: where every exponent field of both sides lies in [66, 187], every product passes it.
#include <limits.h>

#include <algorithm>

#include <cuda_pipeline_primitives.h>

#include "common.cuh"
#include "pam_scalar.cuh"

namespace pamk {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kSlice = 32, kQuads = kSlice / 4;         // floats of a key in a stage
constexpr int kKeyBytes = 32 * kSlice * 4;              // a stage of keys: 32 positions
constexpr int kMostRows = 8, kWarps = 4, kMostWarps = 8;

// Positions that the rows of a unit see together: a group's shared ones (all its rows and a key head's query heads), or a row's own (its query heads).
struct Segment {
    const float *k, *v;
    const int64_t* lengths;                       // one per unit, or null: all slots
    int64_t k_group, k_row, k_pos, k_head, v_group, v_row, v_pos, v_head;
    int slots, per_row;
    int tiles, tile_rows, ranks;                  // CTAs of a (unit, key head): tiles of rows, shares of the positions
    int first_part;                               // where its parts begin among a row's
    float* scores;                                // t: [rows with the same positions, a tile at a time][blocks of 32 positions][the tile's rows][32]
    int width;                                    // positions, a multiple of 32
};

struct Attention {
    const float* q;
    float* out;
    int64_t q_group, q_row, q_head;
    int rows, kv_heads, share, dim;               // `share` query heads on each key head
    int has_beside, beside;                       // the next kernel runs beside this one; this one beside the one before, and ends after it
    int split;                                    // keys: the slices of a piece are dealt out to warps too
    float2* stats;                                // [(group, key head, row, head of the key head)][parts]: a whole number near the maximum, the sum of exponentials shifted by it
    float* sums;                                  // [the same][parts][dim], or null: straight to out
    int parts;
    int two, one, least;                          // 2, 1 and INT32_MIN, as values that the compiler does not know (see sum_on_alu)
};

// A packed add takes both floating-point pipes of an SM partition for as long as an integer add takes the integer pipe, and a multiply-add can stand for an
// integer add on one of the others: five of eight sums belong on the integer pipe, beside what else it does.  Left to choose, the compiler forms
// six of ten as multiply-adds (8 rows of 64 floats 91 -> 88 us).
__device__ __forceinline__ int sum_on_alu(int x, int y, int least) { return __viaddmax_s32(x, y, least); }
__device__ __forceinline__ int sum_on_fma(int x, int y, int one) {
    int d;
    asm("mad.lo.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(one), "r"(y));
    return d;
}


// 0 .. below kBand where the exponent field lies in [66, 187]
__device__ __forceinline__ uint32_t beyond(int32_t x) { return 2u * (uint32_t)x - 2u * (66u << 23); }
constexpr uint32_t kBand = 2u * ((188u - 66u) << 23);
__device__ __forceinline__ uint32_t beyond(int4 x) { return max(max(beyond(x.x), beyond(x.y)), max(beyond(x.z), beyond(x.w))); }

// (as a multiply-add, beside the sums on the integer pipe: 1 %)
__device__ __forceinline__ uint32_t beyond(int32_t x, int two) {
    uint32_t d;
    asm("mad.lo.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(two), "r"(0u - 2u * (66u << 23)));
    return d;
}
__device__ __forceinline__ uint32_t beyond(int4 x, int two) { return max(max(beyond(x.x, two), beyond(x.y, two)), max(beyond(x.z, two), beyond(x.w, two))); }

__device__ __forceinline__ void add_pair(float2& acc, int p0, int p1) { acc = __fadd2_rn(acc, make_float2(i2f(p0), i2f(p1))); }

__device__ __forceinline__ float warp_max(float m) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
}
__device__ __forceinline__ float warp_sum(float m) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fadd(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
}

// 2^e for whole e from -126 to 127: e + 127 are the low bits of the sum
__device__ __forceinline__ float power_of(float e) { return i2f(f2i(fadd(e, 8388608.0f + 127.0f)) << 23); }

// 2^floor(x) (1 + (x - floor(x))) for x from -126 on, below 65: the whole part is the exponent and the fraction the mantissa (rounded once) of the pattern x 2^23
// + kBias.
__device__ __forceinline__ int32_t exponent(float x) { return __float2int_rn(fmul(x, 8388608.0f)); }
__device__ __forceinline__ float power(float x) { return i2f(iadd(exponent(x), kBias)); }

// e of one scaled score, of which t - shift is below 65.  What is below 2^-126 divides to 0.  (NaN scores do not reach the shift; they reach the sum.)
__device__ __forceinline__ float exponential(float t, float shift) {
    const float x = fadd(t, -shift);
    return x >= -126.0f ? power(x) : x != x && t != -INFINITY ? x : 0.0f;
}

// A sum (y) whose shift rises from x to `top`.
__device__ __forceinline__ float rescaled(float2 s, float top) {
    const float down = fadd(s.x, -top);
    return down >= -126.0f ? fmul(s.y, power_of(down)) : s.y == s.y ? 0.0f : s.y;
}

// A shift and a sum from those of `count` parts.
template <class F>
__device__ __forceinline__ float2 joined(F&& part, int count) {
    float top = -INFINITY, sum = 0.0f;
    for (int i = 0; i < count; ++i) top = fmaxf(top, part(i).x);
    for (int i = 0; i < count; ++i) sum = fadd(sum, rescaled(part(i), top));
    return make_float2(top, sum);
}

// A whole number near the maximum, and the sum of exponentials shifted by it, as scores come.  Sums shifted by any whole number are the same but for a power
// of two, so it is raised where exponentials would become large, not with every maximum.
struct Running {
    float shift = -INFINITY, sum = 0.0f;
    __device__ __forceinline__ void add(float t) {
        const float most = fadd(t, -shift) < 64.0f ? shift : fmaxf(shift, floorf(t));         // (the first score raises it; -inf and NaN do not)
        sum = fadd(rescaled(make_float2(shift, sum), most), exponential(t, most));
        shift = most;
    }
};

// A warp's ring of two stages: one is read while the other one arrives.  (Four stages for warps that have no more than that in all cost more places
// than they save: 128 x 5 rows with up to 64 own positions 41 -> 50 us.)
template <int BYTES>
struct Ring {
    char* to;                                     // where the next copies go; what has arrived, once they have been issued
    int turn = BYTES;
    __device__ __forceinline__ Ring(char* memory, int warp) : to(memory + warp * 2 * BYTES) {}
    __device__ __forceinline__ char* next() {
        char* now = to;
        to += turn;
        turn = -turn;
        return now;
    }
};

// Four neighbouring floats to shared memory, those below `dim` of them.
template <bool VEC>
__device__ __forceinline__ void copy_quad(char* to, const float* from, int d, int dim) {
    if (VEC) {
        __pipeline_memcpy_async(to, from, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < dim) __pipeline_memcpy_async(to + 4 * e, from + e, 4);
    }
}

__host__ __device__ constexpr int padded(int dim) { return (dim + 3) / 4 * 4; }

// What a CTA works on.
struct Share {
    int64_t group, base;                          // `base`: the tile's first row among all
    int rank, kv_head, row, first, rows;          // the tile's rows [first, first + rows) among those that see the positions
    int begin, count;                             // positions
};

// Every CTA of a row takes the same number of positions, a multiple of 32, until there are none left.
__device__ __forceinline__ Share share_of(const Attention& a, const Segment& g) {
    Share s;
    unsigned at = blockIdx.x;
    s.rank = (int)(at % g.ranks);
    at /= g.ranks;
    const int tile = (int)(at % g.tiles);
    at /= g.tiles;
    s.kv_head = (int)(at % a.kv_heads);
    at /= a.kv_heads;
    s.row = g.per_row ? (int)(at % a.rows) : 0;
    s.group = g.per_row ? at / a.rows : at;
    const int together = g.per_row ? a.share : a.rows * a.share;
    s.first = tile * g.tile_rows;
    s.rows = min(g.tile_rows, together - s.first);
    s.base = (s.group * a.kv_heads + s.kv_head) * ((int64_t)a.rows * a.share) + s.row * a.share + s.first;
    int live = g.slots;
    if (g.lengths) {
        const int64_t n = g.lengths[at];
        live = n < 0 ? 0 : n < g.slots ? (int)n : g.slots;
    }
    const int each = ((live + g.ranks - 1) / g.ranks + 31) / 32 * 32;
    s.begin = min(s.rank * each, live);
    s.count = min(each, live - s.begin);
    return s;
}

// The kernels of a call are set up behind one another, each when the one before it has come to its last sums.  Those of the own positions run beside those
// of the shared ones: they need nothing of them, only what these have waited for themselves before they let the next one start, and what comes after both
// waits for them.
__device__ __forceinline__ void enter(const Attention& a) {
    if (!a.beside) after_previous();
    if (a.has_beside) next_may_start();
}
__device__ __forceinline__ void leave(const Attention& a) {
    if (a.beside) after_previous();
}

// ---- keys --------------------------------------------------------------------------------------------------------

// Quad c of position p of a stage lies where quad c ^ (p & 7) would: eight neighbouring positions' quads c are in different banks.
__device__ __forceinline__ int swizzled(int p, int c) { return p * (kSlice * 4) + (c ^ (p & 7)) * 16; }

// The copies of one warp, in order: 32 positions (every `step`-th such piece from `first` on), 32 floats of them at a time (every slice, or one alone).
template <bool VEC>
struct KeyCopies {
    const float* from;                            // the lane's quad of the next copy
    int64_t stride;
    int left, step, slice, only, slices;          // `left`: positions from the next piece on
    __device__ __forceinline__ KeyCopies(const Attention& a, const Segment& g, const Share& s, int first, int step_, int only_)
        : stride(g.k_pos), left(s.count - first * 32), step(step_ * 32), slice(max(only_, 0)), only(only_), slices((a.dim + kSlice - 1) / kSlice) {
        const int lane = threadIdx.x & 31;
        from = g.k + s.group * g.k_group + s.row * g.k_row + s.kv_head * g.k_head + (s.begin + first * 32 + lane / kQuads) * stride + slice * kSlice +
               lane % kQuads * 4;
    }
    __device__ __forceinline__ void issue(const Attention& a, Ring<kKeyBytes>& ring) {
        constexpr int kAtOnce = 32 / kQuads;                                     // positions whose copies are one instruction
        const int lane = threadIdx.x & 31, sub = lane / kQuads;
        char* to = ring.next() + swizzled(sub, lane % kQuads);            // (every fourth position: the quad's place alternates)
        if (left > 0) {
            const int other = swizzled(sub + kAtOnce, lane % kQuads) - swizzled(sub, lane % kQuads);
            const auto place = [&](int i) { return to + i / 2 * (2 * kAtOnce * kSlice * 4) + (i % 2 ? other : 0); };
            const float* p = from;
            const int64_t far = kAtOnce * stride;
            if (VEC && left >= 32 && (slice + 1) * kSlice <= a.dim) {
#pragma unroll
                for (int i = 0; i < kQuads; ++i, p += far) copy_quad<true>(place(i), p, 0, 4);
            } else {
                const int d = slice * kSlice + lane % kQuads * 4;
                for (int i = 0; i < kQuads; ++i, p += far)
                    if (i * kAtOnce + sub < left && d < a.dim) copy_quad<VEC>(place(i), p, d, a.dim);
            }
            from += kSlice;
            if (only >= 0 || ++slice == slices) {
                from += step * stride - (only >= 0 ? 1 : slices) * kSlice;
                slice = max(only, 0);
                left -= step;
            }
        }
        __pipeline_commit();
    }
};

// Sums of a stage's products: 32 floats of the lane's key against the same of each row's query.  They are two sums of 16 by themselves before they join those of the stages before:
// a score's rounding grows with 16 and the number of stages instead of all its products (26 x 5 rows, 16 heads of 256 floats, 165 positions: off by 2.3e-7 of the result
// instead of 4.9e-7; 16 x 3 rows, 32 heads on 8 of 128: 3.4e-7 instead of 5.7e-7).  The first products of a stage start their sums, so there are no more adds, and four rows at a
// time keep the registers: 8 rows, 4 heads of 256 floats, 64 positions of 256 groups 70.9 -> 71.4 us (all eight rows at once spill, 77; two at once leave the pipes idle: 12
// rows on a key head of 128, 115 -> 121 us).
template <int ROWS, bool VEC>
__device__ __forceinline__ void key_stage(const Attention& a, float2 (&sum)[ROWS], const char* stage, const int32_t* q, int pitch, int left, bool valid, bool plain) {
    const int lane = threadIdx.x & 31;
    constexpr int kTogether = 4;
    const auto quad = [&](int c) { return *reinterpret_cast<const int4*>(stage + swizzled(lane, c)); };
    if (left >= kSlice) {
        int4 k[kQuads];
        uint32_t far = 0u;
#pragma unroll
        for (int c = 0; c < kQuads; ++c) {
            k[c] = quad(c);
            far = max(far, beyond(k[c], a.two));
        }
        if (__all_sync(0xffffffffu, plain && (far < kBand || !valid))) {
#pragma unroll
            for (int n0 = 0; n0 < ROWS; n0 += kTogether) {
                float2 part[kTogether];
#pragma unroll
                for (int c = 0; c < kQuads; ++c)
#pragma unroll
                    for (int i = 0; i < kTogether && n0 + i < ROWS; ++i) {
                        const int4 w = *reinterpret_cast<const int4*>(q + (n0 + i) * pitch + 4 * c);
                        const int x = sum_on_alu(w.x, k[c].x, a.least), y = sum_on_fma(w.y, k[c].y, a.one);
                        if (c == 0) part[i] = make_float2(i2f(x), i2f(y));
                        else add_pair(part[i], x, y);
                        add_pair(part[i], sum_on_alu(w.z, k[c].z, a.least), c & 1 ? sum_on_fma(w.w, k[c].w, a.one) : sum_on_alu(w.w, k[c].w, a.least));
                    }
#pragma unroll
                for (int i = 0; i < kTogether && n0 + i < ROWS; ++i) sum[n0 + i] = __fadd2_rn(sum[n0 + i], part[i]);
            }
            return;
        }
    }
    // a last stage of few floats, or a value for the range rule
    float2 part[ROWS] = {};
    const int quads = min(kQuads, (left + 3) / 4);
#pragma unroll 1
    for (int c = 0; c < quads; ++c) {
        const int4 x = quad(c);
        const int width = VEC ? 4 : min(4, left - 4 * c);
        const bool easy = __all_sync(0xffffffffu, plain && width == 4 && (beyond(x) < kBand || !valid));
#pragma unroll
        for (int n = 0; n < ROWS; ++n) {
            const int4 w = *reinterpret_cast<const int4*>(q + n * pitch + 4 * c);
            if (easy) {
                add_pair(part[n], iadd(w.x, x.x), iadd(w.y, x.y));
                add_pair(part[n], iadd(w.z, x.z), iadd(w.w, x.w));
            } else {
                part[n].x = fadd(part[n].x, mul(i2f(iadd(w.x, kBias)), i2f(x.x), 0));
                if (width > 1) part[n].y = fadd(part[n].y, mul(i2f(iadd(w.y, kBias)), i2f(x.y), 0));
                if (width > 2) part[n].x = fadd(part[n].x, mul(i2f(iadd(w.z, kBias)), i2f(x.z), 0));
                if (width > 3) part[n].y = fadd(part[n].y, mul(i2f(iadd(w.w, kBias)), i2f(x.w), 0));
            }
        }
    }
#pragma unroll
    for (int n = 0; n < ROWS; ++n) sum[n] = __fadd2_rn(sum[n], part[n]);
}

// What the warps of a CTA share while they read keys.
template <int ROWS>
struct KeyMemory {
    float2 red[kMostWarps * ROWS];
    float dealt[kMostWarps * ROWS * 32];          // (split: sums of each warp's slice)
    int odd_query;
};

// t of the tile's rows and the CTA's positions, stored by the lane that has it (row n, position p: place(p)[n * pitch]), and what the sums need of them.
template <int ROWS, bool VEC, class Place>
__device__ __forceinline__ void key_pass(const Attention& a, const Segment& g, const Share& s, Ring<kKeyBytes>& ring, int32_t* q, KeyMemory<ROWS>& shared,
                                         Running (&stats)[ROWS], Place&& place, int row_pitch) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5, pitch = (a.dim + 31) / 32 * 32, slices = pitch / kSlice;
    // the queries come as they are, and become patterns where each thread finds what it copied itself
    const auto each_of_query = [&](auto&& one) {
        for (int n = warp; n < ROWS; n += warps)
            for (int d = lane; d < pitch; d += 32) one(n, d);
    };
    each_of_query([&](int n, int d) {
        const int r = s.row * a.share + s.first + n;
        if (n < s.rows && d < a.dim)
            __pipeline_memcpy_async(q + n * pitch + d, a.q + s.group * a.q_group + (r / a.share) * a.q_row + (s.kv_head * a.share + r % a.share) * a.q_head + d, 4);
    });
    __pipeline_commit();
    const int step = a.split ? warps / slices : warps, first = a.split ? warp / slices : warp;
    KeyCopies<VEC> copies(a, g, s, first, step, a.split ? warp % slices : -1);
    copies.issue(a, ring);
    if (t == 0) shared.odd_query = 0;
    __syncthreads();
    __pipeline_wait_prior(1);
    bool plain = true;
    each_of_query([&](int n, int d) {
        int32_t* x = q + n * pitch + d;
        const bool there = n < s.rows && d < a.dim;
        plain = plain && (!there || beyond(*x) < kBand);
        *x = there ? isub(*x, kBias) : 0;
    });
    if (!plain) shared.odd_query = 1;
    __syncthreads();
    plain = shared.odd_query == 0;

    // (in most cases: products for which the range rule need not be looked at, and exponentials that the shifts are right for)
    const auto done = [&](const float (&x)[ROWS], int at) {
        float* to = place(at);
        float y[ROWS], z[ROWS], least = 0.0f, most = 0.0f;
        uint32_t far = 0u;
#pragma unroll
        for (int n = 0; n < ROWS; ++n) {
            far = max(far, beyond(f2i(x[n])));
            y[n] = i2f(iadd(f2i(x[n]), isub(f2i(kLog2e), kBias)));
        }
        if (at < 32 * step && far < kBand) {                                     // (the lane's first position)
#pragma unroll
            for (int n = 0; n < ROWS; ++n) stats[n].shift = floorf(y[n]);
        }
#pragma unroll
        for (int n = 0; n < ROWS; ++n) {
            z[n] = fadd(y[n], -stats[n].shift);
            least = fminf(least, z[n]);
            most = fmaxf(most, z[n]);
        }
        if (far < kBand && least >= -126.0f && most < 64.0f) {
#pragma unroll
            for (int n = 0; n < ROWS; ++n) stats[n].sum = fadd(stats[n].sum, power(z[n]));
        } else {
#pragma unroll
            for (int n = 0; n < ROWS; ++n) {
                y[n] = x[n] == -INFINITY ? -INFINITY : mul(x[n], kLog2e, 0);
                stats[n].add(y[n]);
            }
        }
#pragma unroll
        for (int n = 0; n < ROWS; ++n)
            if (n < s.rows) to[n * row_pitch] = y[n];
    };
    // (split: as many pieces as warps take one; the loop runs once, for all warps)
    for (int piece = first; piece * 32 < s.count || (a.split && piece == first); piece += step) {
        const bool valid = piece * 32 + lane < s.count;
        float2 sum[ROWS];
#pragma unroll
        for (int n = 0; n < ROWS; ++n) sum[n] = make_float2(0.0f, 0.0f);
        for (int d = a.split ? warp % slices * kSlice : 0; d < a.dim; d += kSlice) {
            __pipeline_wait_prior(0);
            __syncwarp();
            copies.issue(a, ring);
            key_stage<ROWS, VEC>(a, sum, ring.to, q + d, pitch, a.dim - d, valid, plain);
            if (a.split) break;
        }
        float x[ROWS];
        if (a.split) {
#pragma unroll
            for (int n = 0; n < ROWS; ++n) shared.dealt[(warp * ROWS + n) * 32 + lane] = fadd(sum[n].x, sum[n].y);
            __syncthreads();
            if (warp % slices != 0) break;
#pragma unroll
            for (int n = 0; n < ROWS; ++n) {
                x[n] = shared.dealt[(warp * ROWS + n) * 32 + lane];
                for (int w = 1; w < slices; ++w) x[n] = fadd(x[n], shared.dealt[((warp + w) * ROWS + n) * 32 + lane]);
            }
        } else {
#pragma unroll
            for (int n = 0; n < ROWS; ++n) x[n] = fadd(sum[n].x, sum[n].y);
        }
        if (valid) done(x, piece * 32 + lane);
    }
    __pipeline_wait_prior(0);
}

// The warps' maxima and sums to shared.red; what row n has in all, by joined_row after the next barrier.
template <int ROWS>
__device__ __forceinline__ void leave_stats(KeyMemory<ROWS>& shared, const Running (&stats)[ROWS]) {
#pragma unroll
    for (int n = 0; n < ROWS; ++n) {
        const float top = warp_max(stats[n].shift);
        const float sum = warp_sum(rescaled(make_float2(stats[n].shift, stats[n].sum), top));
        if ((threadIdx.x & 31) == 0) shared.red[(threadIdx.x >> 5) * ROWS + n] = make_float2(top, sum);
    }
}
template <int ROWS>
__device__ __forceinline__ float2 joined_row(const KeyMemory<ROWS>& shared, int n) {
    return joined([&](int w) { return shared.red[w * ROWS + n]; }, blockDim.x >> 5);
}

// 64 groups of 8 rows of 64 floats over 8192 positions: 43 us with a cold cache, 6.3 T products per second.  Bound by instructions: 3.1 per product, of which 1.5 are the product's
// two adds and 0.25 the load of a query; the schedulers issue in 65 % of the cycles and the packed adds take a second slot each, from 16 warps per SM (128 registers; 20 warps
// at 102 spill, both passes back to back 76 -> 89 us).  One row of 64 floats, 60001 positions of 8 heads: 123 MB in 30 us with a cold cache, 4.0 TB/s, bound by memory and the start
// of the kernel.
template <int ROWS, bool VEC>
__global__ void __launch_bounds__(32 * kMostWarps, 2) key_kernel(const Attention a, const Segment g) {
    extern __shared__ __align__(16) char memory[];
    __shared__ KeyMemory<ROWS> shared;
    const int t = threadIdx.x, warp = t >> 5, warps = blockDim.x >> 5;
    Ring<kKeyBytes> ring(memory, warp);
    enter(a);
    const Share s = share_of(a, g);
    Running stats[ROWS];
    float* to = g.scores + s.base * g.width + (int64_t)s.begin * s.rows;
    key_pass<ROWS, VEC>(a, g, s, ring, reinterpret_cast<int32_t*>(memory + warps * 2 * kKeyBytes), shared, stats,
                        [&](int at) { return to + (int64_t)(at / 32) * (32 * s.rows) + at % 32; }, 32);
    if (!a.has_beside) next_may_start();
    leave_stats(shared, stats);
    __syncthreads();
    if (t < s.rows) a.stats[(s.base + t) * a.parts + g.first_part + s.rank] = joined_row(shared, t);
    leave(a);
}

// ---- values ------------------------------------------------------------------------------------------------------

// A stage: 4 KB, as eight quads of each lane, and t of its positions.  `kLanes` lanes cover a position's columns (kCols quads each), four neighbouring
// positions at a time.
template <int SLOTS, int ROWS>
struct ValueShape {
    static constexpr int kLanes = SLOTS >= 4 ? 32 : 8 * SLOTS, kCols = SLOTS == 8 ? 2 : 1, kAcross = 32 / kLanes, kTimes = 2 / kCols;
    static constexpr int kPositions = 4 * kAcross * kTimes, kScores = 4096;      // (kScores: where t lies in a stage)
    static constexpr int kBytes = kScores + ROWS * kPositions * 4;
};

// The copies of one warp, in order: every `step`-th piece of kPositions.  Each lane copies what it will read itself, and some of t.
template <int SLOTS, int ROWS, bool VEC>
struct ValueCopies {
    using S = ValueShape<SLOTS, ROWS>;
    const float *from, *t;                        // the lane's first quad of values in the next piece, and of t of the segment
    int64_t stride;
    int left, step, rows, at;                     // `at`: the next piece's first position
    __device__ __forceinline__ ValueCopies(const Attention& a, const Segment& g, const Share& s, int first, int step_)
        : stride(g.v_pos), left(s.count - first * S::kPositions), step(step_ * S::kPositions), rows(s.rows), at(s.begin + first * S::kPositions) {
        const int lane = threadIdx.x & 31, l = lane % S::kLanes, sub = lane / S::kLanes;
        from = g.v + s.group * g.v_group + s.row * g.v_row + s.kv_head * g.v_head + (at + sub * 4) * stride + l * 4;
        t = g.scores + s.base * g.width + lane / (S::kPositions / 4) * 32 + lane % (S::kPositions / 4) * 4;
    }
    __device__ __forceinline__ void values(const Attention& a, char* to) const {
        const int lane = threadIdx.x & 31, l = lane % S::kLanes, sub = lane / S::kLanes;
        const float* p = from;
        to += lane * 16;
        const auto each = [&](auto&& one) {
#pragma unroll
            for (int m = 0; m < S::kTimes; ++m) {
#pragma unroll
                for (int u = 0; u < 4; ++u, p += stride)
#pragma unroll
                    for (int c = 0; c < S::kCols; ++c)
                        one(to + ((m * 4 + u) * S::kCols + c) * 512, p + S::kLanes * 4 * c, m * 4 * S::kAcross + sub * 4 + u, (l + S::kLanes * c) * 4);
                p += (4 * S::kAcross - 4) * stride;
            }
        };
        if (VEC && left >= S::kPositions && a.dim == 4 * S::kLanes * S::kCols)
            each([&](char* at, const float* x, int, int) { copy_quad<true>(at, x, 0, 4); });
        else
            each([&](char* at, const float* x, int position, int d) {
                if (position < left && d < a.dim) copy_quad<VEC>(at, x, d, a.dim);
            });
    }
    __device__ __forceinline__ void scores(const Attention& a, char* to) const {
        constexpr int kRowQuads = S::kPositions / 4, kRowsAtOnce = 32 / kRowQuads;
        const int lane = threadIdx.x & 31;
        const float* x = t + ((int64_t)(at / 32) * (32 * rows) + at % 32);
#pragma unroll
        for (int n = 0; n < ROWS; n += kRowsAtOnce, x += kRowsAtOnce * 32)
            if (n + lane / kRowQuads < rows) __pipeline_memcpy_async(to + S::kScores + n * S::kPositions * 4 + lane * 16, x, 16);
    }
    __device__ __forceinline__ void advance() {
        from += step * stride;
        at += step;
        left -= step;
    }
    __device__ __forceinline__ void issue(const Attention& a, Ring<S::kBytes>& ring) {
        char* to = ring.next();
        if (left > 0) {
            values(a, to);
            scores(a, to);
            advance();
        }
        __pipeline_commit();
    }
};

// What a row divides by and is shifted by.
struct __align__(16) RowStat {
    float flush_max, pass_max;
    int32_t sub;
    float shift;
};

// `kept` (rows `pitch` apart): t of the stage's positions, where it is not in the stage.
template <int SLOTS, int ROWS, bool VEC, bool KEPT>
__device__ __forceinline__ void value_stage(const Attention& a, int count, int rows, float2 (&acc)[ROWS][2 * ValueShape<SLOTS, ROWS>::kCols], char* slot,
                                            const RowStat* stats, const float* kept, int pitch) {
    using S = ValueShape<SLOTS, ROWS>;
    const int lane = threadIdx.x & 31, l = lane % S::kLanes, sub = lane / S::kLanes;
    // t becomes p, as patterns for the products
    int32_t* probs = reinterpret_cast<int32_t*>(slot + S::kScores);
    constexpr int kTurns = (ROWS * S::kPositions + 31) / 32;
    float x[kTurns];
    int32_t easy[kTurns];
    bool odd = count < S::kPositions;                                           // (a part of a stage, or a probability for the range rule)
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        const int at = i * 32 + lane;
        const bool there = at < rows * S::kPositions;
        const int n = there ? at / S::kPositions : 0;
        x[i] = KEPT ? kept[n * pitch + at % S::kPositions] : i2f(probs[there ? at : 0]);
        const float z = fadd(x[i], -stats[n].shift);
        easy[i] = isub(exponent(z), stats[n].sub);
        // (of the pattern's whole exponent, its sign among it: sums reach 2^94)
        odd = odd || (there && (!(z >= -126.0f) || (uint32_t)easy[i] + ((uint32_t)kBias - (66u << 23)) >= ((188u - 66u) << 23)));
    }
    const bool plain = !__any_sync(0xffffffffu, odd);
    if (!plain)
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int at = i * 32 + lane;
            const RowStat r = stats[at < rows * S::kPositions ? at / S::kPositions : 0];
            const float e = exponential(x[i], r.shift);
            const float p = e <= r.flush_max ? 0.0f : e <= r.pass_max ? i2f(isub(f2i(e), r.sub)) : quiet_nan();
            easy[i] = isub(f2i(p), kBias);
        }
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
        if (i * 32 + lane < rows * S::kPositions) probs[i * 32 + lane] = easy[i];
    __syncwarp();
    probs += sub * 4;
    slot += lane * 16;
#pragma unroll
    for (int m = 0; m < S::kTimes; ++m) {
        int4 v[4][S::kCols];
        uint32_t far = 0u;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < S::kCols; ++c) {
                int4& x = v[u][c];
                x = *reinterpret_cast<const int4*>(slot + ((m * 4 + u) * S::kCols + c) * 512);
                const int d = (l + S::kLanes * c) * 4;
                if (!VEC) {                                                     // (columns past the last hold nothing)
                    if (d >= a.dim) x.x = kBias;
                    if (d + 1 >= a.dim) x.y = kBias;
                    if (d + 2 >= a.dim) x.z = kBias;
                    if (d + 3 >= a.dim) x.w = kBias;
                }
                far = max(far, !VEC || d < a.dim ? beyond(x, a.two) : 0u);
            }
        if (__all_sync(0xffffffffu, plain && far < kBand)) {
#pragma unroll
            for (int n = 0; n < ROWS; n += 2) {
                int4 w[2];
#pragma unroll
                for (int i = n; i < n + 2 && i < ROWS; ++i) w[i - n] = *reinterpret_cast<const int4*>(probs + i * S::kPositions + m * 4 * S::kAcross);
                // (two rows at a time: four chains of adds)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = n; i < n + 2 && i < ROWS; ++i) {
                        const int32_t b = u == 0 ? w[i - n].x : u == 1 ? w[i - n].y : u == 2 ? w[i - n].z : w[i - n].w;
#pragma unroll
                        for (int c = 0; c < S::kCols; ++c) {
                            add_pair(acc[i][2 * c], sum_on_alu(b, v[u][c].x, a.least), sum_on_fma(b, v[u][c].y, a.one));
                            add_pair(acc[i][2 * c + 1], sum_on_alu(b, v[u][c].z, a.least), u & 1 ? sum_on_fma(b, v[u][c].w, a.one) : sum_on_alu(b, v[u][c].w, a.least));
                        }
                    }
            }
            continue;
        }
#pragma unroll 1
        for (int u = 0; u < 4; ++u) {
            if (m * 4 * S::kAcross + sub * 4 + u >= count) break;
#pragma unroll
            for (int c = 0; c < S::kCols; ++c) {
                const int4 x = *reinterpret_cast<const int4*>(slot + ((m * 4 + u) * S::kCols + c) * 512);
#pragma unroll
                for (int n = 0; n < ROWS; ++n) {
                    const float p = i2f(iadd(probs[n * S::kPositions + m * 4 * S::kAcross + u], kBias));
                    acc[n][2 * c].x = fadd(acc[n][2 * c].x, mul(p, i2f(x.x), 0));
                    acc[n][2 * c].y = fadd(acc[n][2 * c].y, mul(p, i2f(x.y), 0));
                    acc[n][2 * c + 1].x = fadd(acc[n][2 * c + 1].x, mul(p, i2f(x.z), 0));
                    acc[n][2 * c + 1].y = fadd(acc[n][2 * c + 1].y, mul(p, i2f(x.w), 0));
                }
            }
        }
    }
}

__device__ __forceinline__ RowStat row_stat(float top, float sum) {
    const Divisor d = make_divisor(sum, 0);
    return {d.flush_max, d.pass_max, d.sub, top};
}

// The sums of a CTA's warps, added and stored.
template <int SLOTS, int ROWS>
__device__ __forceinline__ void store_sums(const Attention& a, const Segment& g, const Share& s, const float2 (&acc)[ROWS][2 * ValueShape<SLOTS, ROWS>::kCols],
                                           char* memory) {
    using V = ValueShape<SLOTS, ROWS>;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
    __syncthreads();                                                             // (the rings become the warps' sums)
    const int columns = padded(a.dim), l = lane % V::kLanes;
    float* sums = reinterpret_cast<float*>(memory);                              // [warp][row][column]
#pragma unroll
    for (int n = 0; n < ROWS; ++n)
#pragma unroll
        for (int c = 0; c < V::kCols; ++c) {
            float4 x = make_float4(acc[n][2 * c].x, acc[n][2 * c].y, acc[n][2 * c + 1].x, acc[n][2 * c + 1].y);
#pragma unroll
            for (int d = V::kLanes; d < 32; d <<= 1) {
                x.x = fadd(x.x, __shfl_xor_sync(0xffffffffu, x.x, d));
                x.y = fadd(x.y, __shfl_xor_sync(0xffffffffu, x.y, d));
                x.z = fadd(x.z, __shfl_xor_sync(0xffffffffu, x.z, d));
                x.w = fadd(x.w, __shfl_xor_sync(0xffffffffu, x.w, d));
            }
            const int d = (l + V::kLanes * c) * 4;
            if (lane < V::kLanes && d < a.dim && n < s.rows) *reinterpret_cast<float4*>(sums + (warp * ROWS + n) * columns + d) = x;
        }
    __syncthreads();
    for (int n = warp; n < s.rows; n += warps) {
        const int r = s.row * a.share + s.first + n;
        float* to = a.sums ? a.sums + ((s.base + n) * a.parts + g.first_part + s.rank) * a.dim
                           : a.out + ((s.group * a.rows + r / a.share) * ((int64_t)a.kv_heads * a.share) + s.kv_head * a.share + r % a.share) * a.dim;
        for (int d = lane; d < a.dim; d += 32) {
            float x = sums[n * columns + d];
            for (int w = 1; w < warps; ++w) x = fadd(x, sums[(w * ROWS + n) * columns + d]);
            to[d] = x;
        }
    }
}

template <int ROWS, int COLS>
__device__ __forceinline__ void clear(float2 (&acc)[ROWS][COLS]) {
#pragma unroll
    for (int n = 0; n < ROWS; ++n)
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[n][c] = make_float2(0.0f, 0.0f);
}

// The same 64 groups of 8 rows: 38 us, 7.0 T products per second, 2.8 instructions each; one row over 60001 positions 30 us.
template <int SLOTS, int ROWS, bool VEC>
__global__ void __launch_bounds__(32 * kMostWarps, 2) value_kernel(const Attention a, const Segment g) {
    extern __shared__ __align__(16) char memory[];
    __shared__ RowStat stats[ROWS];
    using V = ValueShape<SLOTS, ROWS>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    Ring<V::kBytes> ring(memory, warp);
    // The first values are on their way before the scores are there: what the kernels of the keys do not write has been waited for by them.
    const Share s = share_of(a, g);
    ValueCopies<SLOTS, ROWS, VEC> copies(a, g, s, warp, warps);
    char* first = ring.next();
    if (copies.left > 0) copies.values(a, first);
    enter(a);
    if (copies.left > 0) copies.scores(a, first);
    copies.advance();
    __pipeline_commit();
    // a row's shift and sum, from those of its parts
    for (int n = warp; n < s.rows; n += warps) {
        const float2* from = a.stats + (s.base + n) * a.parts;
        const float2 mine = joined([&](int i) { return i * 32 + lane < a.parts ? __ldcg(from + i * 32 + lane) : make_float2(-INFINITY, 0.0f); },
                                   (a.parts + 31) / 32);
        const float top = warp_max(mine.x), sum = warp_sum(rescaled(mine, top));
        if (lane == 0) stats[n] = row_stat(top, sum);
    }
    __syncthreads();

    float2 acc[ROWS][2 * V::kCols];
    clear(acc);
    for (int left = s.count - warp * V::kPositions; left > 0; left -= warps * V::kPositions) {
        __pipeline_wait_prior(0);
        __syncwarp();
        copies.issue(a, ring);
        value_stage<SLOTS, ROWS, VEC, false>(a, left, s.rows, acc, ring.to, stats, nullptr, 0);
    }
    __pipeline_wait_prior(0);
    if (!a.has_beside) next_may_start();
    store_sums<SLOTS, ROWS>(a, g, s, acc, memory);
    leave(a);
}

// Both passes of rows all of whose positions, kMostKept at most, are this CTA's.
constexpr int kMostKept = 256;

template <int SLOTS, int ROWS>
__host__ __device__ constexpr int whole_ring() { return 2 * (ValueShape<SLOTS, ROWS>::kBytes > kKeyBytes ? ValueShape<SLOTS, ROWS>::kBytes : kKeyBytes); }

// (One or two rows need few enough registers for a third more warps on an SM, 22 in CTAs of two, whose shared memory has room for no more, and so more copies on their way: 128 x 5
// rows of 4 heads of 128 floats with up to 64 own positions 32.8 -> 28.9 us.  The kernels of one pass each gain nothing from that, 60001 positions of one row 57 -> 60.)
template <int SLOTS, int ROWS, bool VEC>
__global__ void __launch_bounds__(32 * kMostWarps, ROWS <= 2 ? 3 : 2) whole_kernel(const Attention a, const Segment g) {
    extern __shared__ __align__(16) char memory[];
    __shared__ KeyMemory<ROWS> shared;
    __shared__ RowStat stats[ROWS];
    using V = ValueShape<SLOTS, ROWS>;
    const int t = threadIdx.x, warp = t >> 5, warps = blockDim.x >> 5;
    char* mine = memory + warp * whole_ring<SLOTS, ROWS>();
    float* kept = reinterpret_cast<float*>(memory + warps * whole_ring<SLOTS, ROWS>());      // t: [row][width of the segment]
    Ring<kKeyBytes> keys(mine, 0);
    after_previous();
    const Share s = share_of(a, g);
    Running running[ROWS];
    key_pass<ROWS, VEC>(a, g, s, keys, reinterpret_cast<int32_t*>(kept + ROWS * g.width), shared, running, [&](int at) { return kept + at; }, g.width);
    __syncwarp();
    Ring<V::kBytes> ring(mine, 0);
    ValueCopies<SLOTS, ROWS, VEC> copies(a, g, s, warp, warps);
    const auto issue = [&] {
        char* to = ring.next();
        if (copies.left > 0) copies.values(a, to);
        copies.advance();
        __pipeline_commit();
    };
    issue();
    leave_stats(shared, running);
    __syncthreads();
    if (t < s.rows) {
        const float2 x = joined_row(shared, t);
        stats[t] = row_stat(x.x, x.y);
    }
    __syncthreads();
    float2 acc[ROWS][2 * V::kCols];
    clear(acc);
    for (int at = warp * V::kPositions; at < s.count; at += warps * V::kPositions) {
        __pipeline_wait_prior(0);
        __syncwarp();
        issue();
        value_stage<SLOTS, ROWS, VEC, true>(a, s.count - at, s.rows, acc, ring.to, stats, kept + at, g.width);
    }
    __pipeline_wait_prior(0);
    store_sums<SLOTS, ROWS>(a, g, s, acc, memory);
}

// Adds the parts of a row: every thread those of its column that its turn is, then one thread of a column what these have.  (9 parts of 512 rows of 64 floats: 7.6 us
// alone with a cold cache, most of it launch and a trip to memory.)
__global__ void __launch_bounds__(512) join_kernel(const Attention a) {
    __shared__ float red[512];
    const int64_t row = blockIdx.x;                                              // (group, key head, row, head of the key head)
    const int per = a.rows * a.share, n = (int)(row % per), kv_head = (int)(row / per % a.kv_heads), turns = max(1, (int)blockDim.x / a.dim);
    float* to = a.out + ((row / per / a.kv_heads * a.rows + n / a.share) * ((int64_t)a.kv_heads * a.share) + kv_head * a.share + n % a.share) * a.dim;
    after_previous();
    const int turn = threadIdx.x / a.dim, d = threadIdx.x - turn * a.dim;
    float sum = 0.0f;
    if (turn < turns)
#pragma unroll 16
        for (int r = turn; r < a.parts; r += turns) sum = fadd(sum, __ldcg(a.sums + (row * a.parts + r) * a.dim + d));
    red[threadIdx.x] = sum;
    __syncthreads();
    if (turn == 0) {
        for (int i = 1; i < turns; ++i) sum = fadd(sum, red[i * a.dim + d]);
        to[d] = sum;
    }
}

// ---- planning ------------------------------------------------------------------------------------------------

struct Part {                                     // of the shared positions, or of the own ones
    int rows, tiles, tile_rows, ranks;            // `rows`: the kernels', at least tile_rows
    int key_warps, value_warps, whole_warps;
    bool split;
    int64_t ctas;
};

struct Plan {
    int slots, width[2], parts;                   // `width`: positions, shared and own, in whole blocks of 32
    Part part[2];
    int64_t all_rows;
    bool whole;                                   // one kernel makes both passes
};

int rounded_rows(int n, bool vec) {
    if (!vec) return n <= 1 ? 1 : n <= 4 ? 4 : 8;
    return n <= 6 ? n : 8;
}

constexpr int kPlaces = 4 * 148;                  // CTAs of four warps that the SMs hold at once

// No CTA takes more positions of a row than this, however many rows there are: a warp adds its positions one behind another, and the rounding of such a sum grows with
// their number, where the sums of several CTAs are added in blocks.  One row of 128 floats in each of 600 groups, 32768 positions: off by 8.7e-7 of the result instead of
// 1.8e-6 with three CTAs a row, and with its CTAs more alike 3970 -> 3250 us (2048 positions: 8.8e-7, 3270); 128 groups of 8 heads of 64, 8192 positions: 787 -> 718 us (2048: 730).
constexpr int kMostPositions = 1024;

Part part_of(int64_t units, int together, int64_t positions, int slots, int64_t dim, bool vec) {
    Part p{};
    if (positions == 0) return p;
    p.tiles = (together + kMostRows - 1) / kMostRows;
    p.tile_rows = (together + p.tiles - 1) / p.tiles;
    p.tiles = (together + p.tile_rows - 1) / p.tile_rows;
    p.rows = rounded_rows(p.tile_rows, vec);
    const int64_t all = units * p.tiles, blocks = (positions + 31) / 32;
    // CTAs of a row: what fills the places once, or whole times with nine tenths of them taken, with 8 blocks of 32 positions each at least
    int64_t ranks = std::max<int64_t>(1, kPlaces / all);
    for (int64_t times = 2; times <= 4 && ranks * all * 10 < (times - 1) * kPlaces * 9; ++times) ranks = std::max<int64_t>(1, times * kPlaces / all);
    p.ranks = (int)std::max(std::min(ranks, std::max<int64_t>(1, blocks / 8)), (positions + kMostPositions - 1) / kMostPositions);
    p.ctas = all * p.ranks;
    const int64_t each = (blocks + p.ranks - 1) / p.ranks;
    const int slices = (int)((dim + kSlice - 1) / kSlice), at_once = slots == 1 ? 32 : slots == 2 ? 16 : slots == 4 ? 8 : 4;
    // Warps: one for each block of positions, up to four.  Where that leaves places empty, up to as many as fill them: a row's few positions are then the time
    // of the call, and the slices of a key are dealt out to warps as well.
    const int most = p.ctas <= 2 * 148 ? kMostWarps : kWarps, at_least = p.ctas <= kPlaces ? 1 : 0;
    p.split = at_least && slices > 1 && each * slices <= most;
    p.key_warps = p.split ? (int)(each * slices) : (int)std::min<int64_t>(each, kWarps);
    p.value_warps = (int)std::min<int64_t>((std::min<int64_t>(positions, each * 32) + at_once - 1) / at_once, most);
    p.whole_warps = at_least && !p.split ? std::max(p.key_warps, p.value_warps) : p.key_warps;
    return p;
}

Plan plan_of(int64_t groups, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t shared, int64_t own, bool vec) {
    Plan p;
    p.slots = dim <= 32 ? 1 : dim <= 64 ? 2 : dim <= 128 ? 4 : 8;
    const int share = (int)(heads / kv_heads);
    p.part[0] = part_of(groups * kv_heads, (int)(rows * share), shared, p.slots, dim, vec);
    p.part[1] = part_of(groups * kv_heads * rows, share, own, p.slots, dim, vec);
    p.width[0] = (int)((shared + 31) / 32 * 32);
    p.width[1] = (int)((own + 31) / 32 * 32);
    p.parts = p.part[0].ranks + p.part[1].ranks;
    p.all_rows = groups * rows * heads;
    p.whole = p.parts == 1 && shared + own <= kMostKept;
    return p;
}

size_t aligned(size_t n) { return (n + 255) / 256 * 256; }
size_t score_bytes(const Plan& p) { return aligned((size_t)p.all_rows * ((size_t)p.width[0] + p.width[1]) * 4); }
size_t stat_bytes(const Plan& p) { return aligned((size_t)p.all_rows * p.parts * 8); }
size_t bytes_of(const Plan& p, int64_t dim) { return p.whole ? 0 : score_bytes(p) + stat_bytes(p) + (p.parts > 1 ? aligned((size_t)(p.all_rows * p.parts * dim) * 4) : 0); }

// What a kernel may ask for, whatever a call needs: calls of two threads set the same.  (Eight warps' rings of 10 KB, and t and queries of 8 rows: 96 KB.)
constexpr int kMostMemory = 128 * 1024;

template <class K>
int launch(K* kernel, int64_t ctas, int warps, size_t memory, const Attention& a, const Segment& g, cudaStream_t st) {
    if (memory > kMostMemory) return PAMK_ERR_SIZE;                              // (no plan comes near)
    if (memory > 32 * 1024) {                                                    // (48 KB with what the kernels declare)
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostMemory);
        if (err != cudaSuccess) return record_cuda_error(err);
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;                // (set up behind the kernel before)
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)ctas);
    config.blockDim = dim3(warps * 32);
    config.dynamicSmemBytes = memory;
    config.stream = st;
    config.attrs = &attr;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, kernel, a, g);
    count_launch();
    return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
}

template <int ROWS, bool VEC>
int launch_keys(const Part& p, const Attention& a, const Segment& g, cudaStream_t st) {
    return launch(key_kernel<ROWS, VEC>, p.ctas, p.key_warps, (size_t)p.key_warps * 2 * kKeyBytes + (size_t)ROWS * ((a.dim + 31) / 32 * 32) * 4, a, g, st);
}

template <int SLOTS, int ROWS, bool VEC>
int launch_slots(const Part& p, const Attention& a, const Segment& g, cudaStream_t st) {
    const size_t ring = (size_t)p.value_warps * 2 * ValueShape<SLOTS, ROWS>::kBytes;
    return launch(value_kernel<SLOTS, ROWS, VEC>, p.ctas, p.value_warps, std::max(ring, (size_t)p.value_warps * ROWS * padded(a.dim) * 4), a, g, st);
}

template <int SLOTS, int ROWS, bool VEC>
int launch_whole(const Part& p, const Attention& a, const Segment& g, cudaStream_t st) {
    const size_t memory = (size_t)p.whole_warps * whole_ring<SLOTS, ROWS>() + (size_t)ROWS * (g.width + (a.dim + 31) / 32 * 32) * 4;
    return launch(whole_kernel<SLOTS, ROWS, VEC>, p.ctas, p.whole_warps, std::max(memory, (size_t)p.whole_warps * ROWS * padded(a.dim) * 4), a, g, st);
}

enum Pass { kKeys, kValues, kWhole };

template <int ROWS, bool VEC>
int launch_pass(Pass pass, int slots, const Part& p, const Attention& a, const Segment& g, cudaStream_t st) {
    if (pass == kKeys) return launch_keys<ROWS, VEC>(p, a, g, st);
    const bool values = pass == kValues;
    switch (slots) {
        case 1: return values ? launch_slots<1, ROWS, VEC>(p, a, g, st) : launch_whole<1, ROWS, VEC>(p, a, g, st);
        case 2: return values ? launch_slots<2, ROWS, VEC>(p, a, g, st) : launch_whole<2, ROWS, VEC>(p, a, g, st);
        case 4: return values ? launch_slots<4, ROWS, VEC>(p, a, g, st) : launch_whole<4, ROWS, VEC>(p, a, g, st);
        default: return values ? launch_slots<8, ROWS, VEC>(p, a, g, st) : launch_whole<8, ROWS, VEC>(p, a, g, st);
    }
}

int launch_part(Pass pass, bool vec, int slots, const Part& p, const Attention& a, const Segment& g, cudaStream_t st) {
    if (!vec) {
        switch (p.rows) {
            case 1: return launch_pass<1, false>(pass, slots, p, a, g, st);
            case 4: return launch_pass<4, false>(pass, slots, p, a, g, st);
            default: return launch_pass<8, false>(pass, slots, p, a, g, st);
        }
    }
    switch (p.rows) {
        case 1: return launch_pass<1, true>(pass, slots, p, a, g, st);
        case 2: return launch_pass<2, true>(pass, slots, p, a, g, st);
        case 3: return launch_pass<3, true>(pass, slots, p, a, g, st);
        case 4: return launch_pass<4, true>(pass, slots, p, a, g, st);
        case 5: return launch_pass<5, true>(pass, slots, p, a, g, st);
        case 6: return launch_pass<6, true>(pass, slots, p, a, g, st);
        default: return launch_pass<8, true>(pass, slots, p, a, g, st);
    }
}

bool sizes_ok(int64_t groups, int64_t rows, int64_t heads, int64_t dim, int64_t shared, int64_t own) {
    if (dim > 256 || rows * heads > (1 << 20) || shared > (1 << 30) || own > (1 << 30) - shared || groups > INT32_MAX) return false;
    // (CTAs of the largest grid)
    return groups * rows * heads <= INT32_MAX / (2 + (shared + own) / 64);
}

}  // namespace
}  // namespace pamk

extern "C" {

size_t pamk_cached_attention_workspace_bytes(int64_t groups, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
                                             int64_t shared, int64_t own) {
    using namespace pamk;
    if (groups <= 0 || rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || shared < 0 || own < 0 || shared + own == 0) return 0;
    if (!sizes_ok(groups, rows, heads, dim, shared, own)) return 0;
    return bytes_of(plan_of(groups, rows, heads, kv_heads, dim, shared, own, true), dim);       // (the same whichever way rows are loaded)
}

int pamk_cached_attention(const float* q, float* out, const float* shared_k, const float* shared_v, const int64_t* shared_lengths,
                          const float* own_k, const float* own_v, const int64_t* own_lengths,
                          int64_t groups, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t shared, int64_t own,
                          const int64_t* strides, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace pamk;
    if (groups < 0 || rows < 0 || heads < 0 || kv_heads < 1 || dim < 0 || shared < 0 || own < 0 || heads % kv_heads || !strides) return PAMK_ERR_ARG;
    if (groups == 0 || rows == 0 || heads == 0 || dim == 0) return PAMK_OK;
    if (!q || !out || (shared && (!shared_k || !shared_v)) || (own && (!own_k || !own_v))) return PAMK_ERR_ARG;
    if (!sizes_ok(groups, rows, heads, dim, shared, own)) return PAMK_ERR_SIZE;
    cudaStream_t st = (cudaStream_t)stream;
    if (shared + own == 0) {
        const cudaError_t err = cudaMemsetAsync(out, 0, (size_t)(groups * rows * heads * dim) * 4, st);
        return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
    }
    Attention a{};
    a.q = q; a.out = out;
    a.q_group = strides[0]; a.q_row = strides[1]; a.q_head = strides[2];
    a.rows = (int)rows; a.kv_heads = (int)kv_heads; a.share = (int)(heads / kv_heads); a.dim = (int)dim;
    Segment g[2] = {};
    g[0].k = shared_k; g[0].v = shared_v; g[0].lengths = shared_lengths; g[0].slots = (int)shared;
    g[0].k_group = strides[3]; g[0].k_pos = strides[4]; g[0].k_head = strides[5];
    g[0].v_group = strides[6]; g[0].v_pos = strides[7]; g[0].v_head = strides[8];
    g[1].k = own_k; g[1].v = own_v; g[1].lengths = own_lengths; g[1].slots = (int)own; g[1].per_row = 1;
    g[1].k_group = strides[9]; g[1].k_row = strides[10]; g[1].k_pos = strides[11]; g[1].k_head = strides[12];
    g[1].v_group = strides[13]; g[1].v_row = strides[14]; g[1].v_pos = strides[15]; g[1].v_head = strides[16];
    // 16-byte copies: every address that starts a position's row of a head is a multiple of 16 bytes
    bool vec = dim % 4 == 0;
    for (int i = 3; i < 9 && shared; ++i) vec = vec && strides[i] % 4 == 0;
    for (int i = 9; i < 17 && own; ++i) vec = vec && strides[i] % 4 == 0;
    vec = vec && (!shared || (aligned16(shared_k) && aligned16(shared_v))) && (!own || (aligned16(own_k) && aligned16(own_v)));
    const Plan p = plan_of(groups, rows, heads, kv_heads, dim, shared, own, vec);
    if (p.part[0].ctas > INT32_MAX || p.part[1].ctas > INT32_MAX) return PAMK_ERR_SIZE;
    const size_t bytes = bytes_of(p, dim);
    if (bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < bytes)) return PAMK_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    g[0].scores = reinterpret_cast<float*>(ws);
    g[1].scores = g[0].scores + p.all_rows * p.width[0];
    g[0].width = p.width[0];
    g[1].width = p.width[1];
    a.stats = reinterpret_cast<float2*>(ws + score_bytes(p));
    if (p.parts > 1) a.sums = reinterpret_cast<float*>(ws + score_bytes(p) + stat_bytes(p));
    a.two = 2; a.one = 1; a.least = INT32_MIN;
    a.parts = p.parts;
    g[1].first_part = p.part[0].ranks;
    if (p.whole) {
        const int i = shared ? 0 : 1;
        g[i].tiles = p.part[i].tiles; g[i].tile_rows = p.part[i].tile_rows; g[i].ranks = 1;
        a.split = p.part[i].split;
        return launch_part(kWhole, vec, p.slots, p.part[i], a, g[i], st);
    }
    for (int pass = 0; pass < 2; ++pass)
        for (int i = 0; i < 2; ++i) {
            const Part& part = p.part[i];
            if (!g[i].slots) continue;
            g[i].tiles = part.tiles; g[i].tile_rows = part.tile_rows; g[i].ranks = part.ranks;
            a.split = part.split;
            a.beside = i == 1 && g[0].slots;
            a.has_beside = i == 0 && g[1].slots;
            const int status = launch_part(pass == 0 ? kKeys : kValues, vec, p.slots, part, a, g[i], st);
            if (status != PAMK_OK) return status;
        }
    if (!a.sums) return PAMK_OK;
    return launch_behind(join_kernel, dim3((unsigned)p.all_rows), p.parts > 8 || dim > 128 ? 512 : 128, st, a);
}

}
