// Attention of single-token rows over a key/value cache, in PAM arithmetic.
//
// For one row q of a head and the positions j that it sees (those its group shares, then its own):
//     s_j = sum_d pam(q_d, k_jd)       t_j = pam(s_j, log2 e)          m = floor(max_j t_j)
//     e_j = exp2(t_j - m)              p_j = pad(e_j, sum_j e_j)       out_d = sum_j pam(p_j, v_jd)
// with the piecewise affine exp2 and -inf scores at probability 0, as in the chain bmm -> softmax -> bmm
// (pam/pam_ops.py:82-101, 305-328).  The chain's shift is the floor of the maximum of the whole tensor, here it is the row's: a
// whole number either way, and exp2(t - m) = exp2(t) 2^-m exactly, so only the rounding of t - m differs.
//
// pam is not linear: pam(pad(e, S), v) summed is not pad(sum of pam(e, v), S).  A running maximum and sum with one
// joint pass over keys and values is therefore not to be had; the sum must be known before the first value is
// weighted.  The keys are read in a first kernel, which leaves t and each range's maximum and sum of exponentials, the values in a
// second one; ranges of a long axis are added by a third.
//
// Rows that share positions are worked on together, up to eight per CTA: every key and value is loaded once for all of them.  A
// product is one integer and one floating-point add; the range rule (pam_scalar.cuh) is decided per vector of loaded
// elements: where every exponent field of both sides lies in [66, 187], every product passes it.
#include "common.cuh"
#include "pam_scalar.cuh"

namespace pamk {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxRows = 8;                       // rows of a tile
constexpr int kMostChunk = 512;                   // positions of a range

// Positions that rows see together: those of a group (`per_row` 0: all its rows), or one row's own.
struct Segment {
    const float *k, *v;
    const int64_t* lengths;                       // one per unit, or null: all slots
    int64_t k_group, k_row, k_pos, k_head, v_group, v_row, v_pos, v_head;
    int slots, chunk, chunks, tiles;
    int per_row, rows;                            // rows that share it
    int first_chunk, first_pos;                   // among the chunks and the scores of a row
};

struct Attention {
    const float* q;
    float* out;
    int64_t q_group, q_row, q_head;
    int groups, rows, kv_heads, share, dim;       // `share` query heads on each key head
    int32_t off;
    float* scores;                                // [groups, kv_heads, rows * share, width]
    float2* stats;                                // [groups, kv_heads, rows * share, chunks]: floor of the maximum, sum
    float* parts;                                 // [groups, kv_heads, rows * share, chunks, dim]
    int width, chunks;
};

// Where a CTA works.
struct Place {
    int64_t group, base;                          // `base` + n: index of the tile's n-th row in scores, stats and parts
    int kv_head, row, tile, chunk, begin, end;    // positions [begin, end)
};

__device__ __forceinline__ Place place_of(const Attention& a, const Segment& s, int rows_per_tile) {
    Place p;
    int64_t at = blockIdx.x;
    p.chunk = (int)(at % s.chunks);
    at /= s.chunks;
    p.tile = (int)(at % s.tiles);
    at /= s.tiles;
    p.kv_head = (int)(at % a.kv_heads);
    at /= a.kv_heads;
    p.row = s.per_row ? (int)(at % a.rows) : 0;
    p.group = s.per_row ? at / a.rows : at;
    int64_t live = s.slots;
    if (s.lengths) {
        const int64_t n = s.lengths[at];
        live = n < 0 ? 0 : n < s.slots ? n : s.slots;
    }
    p.begin = p.chunk * s.chunk;
    p.end = (int)(live < p.begin + s.chunk ? live : p.begin + s.chunk);
    p.base = (p.group * a.kv_heads + p.kv_head) * ((int64_t)a.rows * a.share) + p.row * a.share + p.tile * rows_per_tile;
    return p;
}

__device__ __forceinline__ int rows_of(const Segment& s, const Place& p, int rows_per_tile) {
    return min(rows_per_tile, s.rows - p.tile * rows_per_tile);
}

// 0 .. below 2 * (188 - 66) << 23 where the exponent field lies in [66, 187]
__device__ __forceinline__ uint32_t beyond(float x) { return 2u * (uint32_t)f2i(x) - 2u * (66u << 23); }
constexpr uint32_t kBand = 2u * ((188u - 66u) << 23);

// Lane l of eight holds element e of slot i of a row of `dim`: with vectors 16 bytes at a time, else one float after another.
template <bool VEC>
__device__ __forceinline__ int element(int l, int i, int e) { return VEC ? (l + 8 * i) * 4 + e : l + 8 * (4 * i + e); }

template <int SLOTS, bool VEC>
__device__ __forceinline__ void load_row(float (&x)[SLOTS * 4], const float* p, int l, int dim, float absent) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        if (VEC) {
            float4 w = make_float4(absent, absent, absent, absent);
            if ((l + 8 * i) * 4 < dim) w = __ldg(reinterpret_cast<const float4*>(p) + l + 8 * i);
            x[4 * i] = w.x; x[4 * i + 1] = w.y; x[4 * i + 2] = w.z; x[4 * i + 3] = w.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = element<VEC>(l, i, e);
                x[4 * i + e] = d < dim ? __ldg(p + d) : absent;
            }
        }
    }
}

// Adds up N values over the eight lanes of a position; lane l is left with the sum of value l / (8 / P), P the power of two from N on.
template <int N>
__device__ __forceinline__ float sum_over_eight(float (&s)[N], int l) {
    constexpr int P = N > 4 ? 8 : N > 2 ? 4 : N > 1 ? 2 : 1;
    float t[P];
#pragma unroll
    for (int i = 0; i < P; ++i) t[i] = i < N ? s[i] : 0.0f;
#pragma unroll
    for (int w = P / 2, d = 4; d > 0; w >>= 1, d >>= 1) {
        if (w > 0) {
            const bool upper = l & d;
#pragma unroll
            for (int i = 0; i < P / 2; ++i)
                if (i < w) {
                    const float other = __shfl_xor_sync(0xffffffffu, upper ? t[i] : t[i + w], d);
                    t[i] = fadd(upper ? t[i + w] : t[i], other);
                }
        } else {
            t[0] = fadd(t[0], __shfl_xor_sync(0xffffffffu, t[0], d));
        }
    }
    return t[0];
}

// t of the tile's rows for positions [begin, end), to scores[n * stride + position - begin] in shared memory.
template <int SLOTS, int ROWS, bool VEC>
__device__ __forceinline__ void score_range(const Attention& a, const Segment& s, const Place& p, int rows, float* scores, int stride) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int l = lane & 7, sub = lane >> 3;
    constexpr int kAtOnce = SLOTS >= 8 ? 1 : SLOTS == 4 ? 2 : 4;                 // positions of a lane whose loads are on their way together
    // an absent element of the key is 1.0f and the query's biased pattern -bits(1.0f): their product's pattern is +0
    int32_t q[ROWS][SLOTS * 4];
    bool plain = true;
#pragma unroll
    for (int n = 0; n < ROWS; ++n) {
        const int r = p.tile * ROWS + min(n, rows - 1);
        const int row = s.per_row ? p.row : r / a.share, head = p.kv_head * a.share + (s.per_row ? r : r % a.share);
        float x[SLOTS * 4];
        load_row<SLOTS, VEC>(x, a.q + p.group * a.q_group + row * a.q_row + head * a.q_head, l, a.dim, 1.0f);
#pragma unroll
        for (int i = 0; i < SLOTS * 4; ++i) {
            plain = plain && beyond(x[i]) < kBand;
            q[n][i] = element<VEC>(l, i / 4, i % 4) < a.dim ? isub(f2i(x[i]), kBias - a.off) : -kBias;
        }
    }
    plain = __all_sync(0xffffffffu, plain);
    const float* keys = s.k + p.group * s.k_group + p.row * s.k_row + p.kv_head * s.k_head;
    for (int j0 = p.begin + warp * 4 * kAtOnce; j0 < p.end; j0 += warps * 4 * kAtOnce) {
        float k[kAtOnce][SLOTS * 4];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
            load_row<SLOTS, VEC>(k[u], keys + (int64_t)min(j0 + u * 4 + sub, p.end - 1) * s.k_pos, l, a.dim, 1.0f);
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            uint32_t far = 0u;
#pragma unroll
            for (int i = 0; i < SLOTS * 4; ++i) far = max(far, beyond(k[u][i]));
            float sum[ROWS];
            if (__all_sync(0xffffffffu, plain && far < kBand)) {
#pragma unroll
                for (int n = 0; n < ROWS; ++n) {
                    sum[n] = 0.0f;
#pragma unroll
                    for (int i = 0; i < SLOTS * 4; ++i) sum[n] = fadd(sum[n], i2f(iadd(q[n][i], f2i(k[u][i]))));
                }
            } else {
#pragma unroll
                for (int n = 0; n < ROWS; ++n) {
                    sum[n] = 0.0f;
#pragma unroll
                    for (int i = 0; i < SLOTS * 4; ++i)
                        if (element<VEC>(l, i / 4, i % 4) < a.dim)
                            sum[n] = fadd(sum[n], mul(i2f(iadd(q[n][i], kBias - a.off)), k[u][i], a.off));
                }
            }
            const float total = sum_over_eight<ROWS>(sum, l);
            constexpr int kEach = ROWS > 4 ? 1 : ROWS > 2 ? 2 : ROWS > 1 ? 4 : 8;              // lanes with the same sum
            const int n = l / kEach, j = j0 + u * 4 + sub;
            if (n < rows && l % kEach == 0 && j < p.end)
                scores[n * stride + j - p.begin] = total == -INFINITY ? -INFINITY : mul(total, kLog2e, a.off);
        }
    }
}

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

// e of one scaled score.  (NaN scores do not reach the shift; they reach the sum.)
__device__ __forceinline__ float exponential(float t, float shift) {
    return t == -INFINITY ? 0.0f : exp2_compact(fadd(t, -shift));
}

// 2^e for whole e <= 0, also -inf and NaN
__device__ __forceinline__ float power(float e) {
    return e >= -126.0f ? i2f(((int32_t)e + 127) << 23) : e != e ? quiet_nan() : 0.0f;
}

template <int SLOTS, int ROWS, bool VEC>
__global__ void __launch_bounds__(256) score_kernel(const Attention a, const Segment s) {
    __shared__ float tile[ROWS * kMostChunk];
    const Place p = place_of(a, s, ROWS);
    const int rows = rows_of(s, p, ROWS), lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    score_range<SLOTS, ROWS, VEC>(a, s, p, rows, tile, kMostChunk);
    __syncthreads();
    const int count = p.end - p.begin;
    after_previous();                              // (the scores of the other segment are on their way: both are waited for by what follows)
    for (int n = threadIdx.x >> 5; n < rows; n += warps) {
        float m = -INFINITY, sum = 0.0f;
        for (int j = lane; j < count; j += 32) m = fmaxf(m, tile[n * kMostChunk + j]);
        const float shift = floorf(warp_max(m));
        float* to = a.scores + (p.base + n) * a.width + s.first_pos + p.begin;
        for (int j = lane; j < count; j += 32) {
            const float t = tile[n * kMostChunk + j];
            to[j] = t;
            sum = fadd(sum, exponential(t, shift));
        }
        sum = warp_sum(sum);
        if (lane == 0) a.stats[(p.base + n) * a.chunks + s.first_chunk + p.chunk] = make_float2(shift, sum);
    }
}

// The row's shift and sum from those of its chunks, by one warp.
__device__ __forceinline__ float2 row_stats(const float2* stats, int chunks, int lane) {
    float m = -INFINITY, sum = 0.0f;
    for (int c = lane; c < chunks; c += 32) m = fmaxf(m, __ldcg(stats + c).x);
    m = warp_max(m);
    for (int c = lane; c < chunks; c += 32) {
        const float2 t = __ldcg(stats + c);
        sum = fadd(sum, t.y == 0.0f ? 0.0f : fmul(t.y, power(fadd(t.x, -m))));
    }
    return make_float2(m, warp_sum(sum));
}

// sum_j pam(p_j, v_jd) of the tile's rows over positions [begin, end): a warp takes four neighbouring positions (times the rows of values
// that it holds at once), each lane four columns of each.  Leaves the sums of all warps in sums[n * 256 + d].
template <int SLOTS, int ROWS, bool VEC>
__device__ __forceinline__ void weigh_range(const Attention& a, const Segment& s, const Place& p, int rows, const float* probs, int stride,
                                            const unsigned char* odd, float* sums) {
    constexpr int kLanes = SLOTS >= 4 ? 32 : 8 * SLOTS, kCols = SLOTS == 8 ? 2 : 1, kAcross = 32 / kLanes;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int l = lane % kLanes, sub = lane / kLanes;
    float acc[ROWS][kCols * 4];
#pragma unroll
    for (int n = 0; n < ROWS; ++n)
#pragma unroll
        for (int i = 0; i < kCols * 4; ++i) acc[n][i] = 0.0f;
    const float* values = s.v + p.group * s.v_group + p.row * s.v_row + p.kv_head * s.v_head;
    const int count = p.end - p.begin;
    const auto column = [l](int i, int e) { return VEC ? (l + kLanes * i) * 4 + e : l + kLanes * (4 * i + e); };
    for (int j0 = warp * 4 * kAcross; j0 < count; j0 += warps * 4 * kAcross) {
        const int j = j0 + sub * 4;
        float v[4][kCols * 4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float* row = values + (int64_t)(p.begin + j + u) * s.v_pos;
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
                if (VEC) {
                    float4 w = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                    if (j + u < count && column(i, 0) < a.dim) w = __ldg(reinterpret_cast<const float4*>(row) + l + kLanes * i);
                    v[u][4 * i] = w.x; v[u][4 * i + 1] = w.y; v[u][4 * i + 2] = w.z; v[u][4 * i + 3] = w.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][4 * i + e] = j + u < count && column(i, e) < a.dim ? __ldg(row + column(i, e)) : 1.0f;
                }
            }
        }
        uint32_t far = 0u;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < kCols * 4; ++i) far = max(far, beyond(v[u][i]));
        const bool plain = far < kBand && *reinterpret_cast<const uint32_t*>(odd + j) == 0u;
        if (__all_sync(0xffffffffu, plain)) {
#pragma unroll
            for (int n = 0; n < ROWS; ++n) {
                const float4 w = *reinterpret_cast<const float4*>(probs + n * stride + j);
                const float pr[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int32_t b = isub(f2i(pr[u]), kBias - a.off);
#pragma unroll
                    for (int i = 0; i < kCols * 4; ++i) acc[n][i] = fadd(acc[n][i], i2f(iadd(b, f2i(v[u][i]))));
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < ROWS; ++n) {
                const float4 w = *reinterpret_cast<const float4*>(probs + n * stride + j);
                const float pr[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < kCols * 4; ++i) acc[n][i] = fadd(acc[n][i], mul(pr[u], v[u][i], a.off));
            }
        }
    }
#pragma unroll
    for (int n = 0; n < ROWS; ++n)
#pragma unroll
        for (int i = 0; i < kCols * 4; ++i)
#pragma unroll
            for (int d = kLanes; d < 32; d <<= 1) acc[n][i] = fadd(acc[n][i], __shfl_xor_sync(0xffffffffu, acc[n][i], d));
    // one warp after another adds its sums
    for (int w = 0; w < warps; ++w) {
        __syncthreads();
        if (warp == w && sub == 0) {
#pragma unroll
            for (int n = 0; n < ROWS; ++n)
#pragma unroll
                for (int i = 0; i < kCols * 4; ++i) {
                    float* to = sums + n * 256 + column(i / 4, i % 4);
                    *to = w == 0 ? acc[n][i] : fadd(*to, acc[n][i]);
                }
        }
    }
    __syncthreads();
}

__device__ __forceinline__ float* out_row(const Attention& a, const Segment& s, const Place& p, int r) {
    const int row = s.per_row ? p.row : r / a.share, head = p.kv_head * a.share + (s.per_row ? r : r % a.share);
    return a.out + ((p.group * a.rows + row) * ((int64_t)a.kv_heads * a.share) + head) * a.dim;
}

template <int SLOTS, int ROWS, bool VEC>
__global__ void __launch_bounds__(256) weigh_kernel(const Attention a, const Segment s) {
    __shared__ __align__(16) float probs[ROWS * kMostChunk];
    __shared__ __align__(16) float sums[ROWS * 256];
    __shared__ __align__(16) unsigned char odd[kMostChunk];
    __shared__ float2 stats[ROWS];
    const Place p = place_of(a, s, ROWS);
    const int rows = rows_of(s, p, ROWS), lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int count = p.end - p.begin;
    after_previous();
    for (int n = threadIdx.x >> 5; n < rows; n += warps) {
        const float2 t = row_stats(a.stats + (p.base + n) * a.chunks, a.chunks, lane);
        if (lane == 0) stats[n] = t;
    }
    __syncthreads();
    // probabilities; positions past the end get 0, and count as beyond the band
    for (int j = threadIdx.x; j < (count + 3) / 4 * 4 + 16 && j < kMostChunk; j += blockDim.x) {
        bool far = j >= count;
#pragma unroll
        for (int n = 0; n < ROWS; ++n) {
            float pr = 0.0f;
            if (j < count && n < rows) {
                const float2 t = stats[n];
                const float e = exponential(__ldcg(a.scores + (p.base + n) * a.width + s.first_pos + p.begin + j), t.x);
                pr = div(e, t.y, a.off);
            }
            far = far || (n < rows && beyond(pr) >= kBand);
            probs[n * kMostChunk + j] = pr;
        }
        odd[j] = far;
    }
    __syncthreads();
    weigh_range<SLOTS, ROWS, VEC>(a, s, p, rows, probs, kMostChunk, odd, sums);
    for (int i = threadIdx.x; i < rows * a.dim; i += blockDim.x) {
        const int n = i / a.dim, d = i - n * a.dim;
        const float x = sums[n * 256 + d];
        if (a.chunks == 1) out_row(a, s, p, p.tile * ROWS + n)[d] = x;
        else a.parts[((p.base + n) * a.chunks + s.first_chunk + p.chunk) * a.dim + d] = x;
    }
}

// Adds the sums of a row's chunks.
__global__ void __launch_bounds__(256) join_kernel(const Attention a) {
    const int64_t row = blockIdx.x;                                              // (group, key head, row and head of the group)
    const int per = a.rows * a.share;
    const int n = (int)(row % per), kv_head = (int)(row / per % a.kv_heads);
    const int64_t group = row / per / a.kv_heads;
    float* to = a.out + ((group * a.rows + n / a.share) * ((int64_t)a.kv_heads * a.share) + kv_head * a.share + n % a.share) * a.dim;
    after_previous();
    for (int d = threadIdx.x; d < a.dim; d += blockDim.x) {
        float sum = 0.0f;
        for (int c = 0; c < a.chunks; ++c) sum = fadd(sum, __ldcg(a.parts + (row * a.chunks + c) * a.dim + d));
        to[d] = sum;
    }
}

template <int SLOTS, bool VEC>
int most_rows() { return SLOTS == 8 ? 4 : kMaxRows; }

template <int SLOTS, int ROWS, bool VEC>
int launch_pass(int pass, bool behind, const Attention& a, const Segment& s, int64_t ctas, unsigned threads, cudaStream_t st) {
    auto* kernel = pass == 0 ? score_kernel<SLOTS, ROWS, VEC> : weigh_kernel<SLOTS, ROWS, VEC>;
    if (behind) return launch_behind(kernel, dim3((unsigned)ctas), threads, st, a, s);
    kernel<<<(unsigned)ctas, threads, 0, st>>>(a, s);
    return check_launch();
}

template <int SLOTS, bool VEC>
int launch_rows(int rows, int pass, bool behind, const Attention& a, const Segment& s, int64_t ctas, unsigned threads, cudaStream_t st) {
    switch (rows) {
        case 1: return launch_pass<SLOTS, 1, VEC>(pass, behind, a, s, ctas, threads, st);
        case 2: return launch_pass<SLOTS, 2, VEC>(pass, behind, a, s, ctas, threads, st);
        case 4: return launch_pass<SLOTS, 4, VEC>(pass, behind, a, s, ctas, threads, st);
        default: return launch_pass<SLOTS, SLOTS == 8 ? 4 : 8, VEC>(pass, behind, a, s, ctas, threads, st);
    }
}

int launch_slots(bool vec, int slots, int rows, int pass, bool behind, const Attention& a, const Segment& s, int64_t ctas, unsigned threads,
                 cudaStream_t st) {
    if (vec) {
        switch (slots) {
            case 1: return launch_rows<1, true>(rows, pass, behind, a, s, ctas, threads, st);
            case 2: return launch_rows<2, true>(rows, pass, behind, a, s, ctas, threads, st);
            case 4: return launch_rows<4, true>(rows, pass, behind, a, s, ctas, threads, st);
            default: return launch_rows<8, true>(rows, pass, behind, a, s, ctas, threads, st);
        }
    }
    switch (slots) {
        case 1: return launch_rows<1, false>(rows, pass, behind, a, s, ctas, threads, st);
        case 2: return launch_rows<2, false>(rows, pass, behind, a, s, ctas, threads, st);
        case 4: return launch_rows<4, false>(rows, pass, behind, a, s, ctas, threads, st);
        default: return launch_rows<8, false>(rows, pass, behind, a, s, ctas, threads, st);
    }
}

// ---- planning ------------------------------------------------------------------------------------------------

struct Plan {
    int slots, tile_rows[2], tiles[2], chunk[2], chunks[2];      // [shared, own]
    int width, all_chunks;
    int64_t rows;                                                // of scores
};

int round_rows(int rows, int most) {
    const int tiles = (rows + most - 1) / most, each = (rows + tiles - 1) / tiles;
    return each <= 2 ? each : each <= 4 ? 4 : 8;
}

// A range of positions per CTA: the longest of 512 .. 64 that gives every SM two of them, if any does.
Plan plan_of(int64_t groups, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t shared, int64_t own) {
    Plan p;
    p.slots = dim <= 32 ? 1 : dim <= 64 ? 2 : dim <= 128 ? 4 : 8;
    const int most = p.slots == 8 ? 4 : kMaxRows, share = (int)(heads / kv_heads);
    const int64_t together[2] = {rows * share, share}, units[2] = {groups * kv_heads, groups * rows * kv_heads}, slots[2] = {shared, own};
    for (int i = 0; i < 2; ++i) {
        p.tile_rows[i] = round_rows((int)together[i], most);
        p.tiles[i] = (int)((together[i] + p.tile_rows[i] - 1) / p.tile_rows[i]);
        int chunk = kMostChunk;
        while (chunk > 64 && units[i] * p.tiles[i] * ((slots[i] + chunk - 1) / chunk) < 2 * 148) chunk /= 2;
        p.chunk[i] = chunk;
        p.chunks[i] = (int)((slots[i] + chunk - 1) / chunk);
    }
    p.width = (int)(shared + own);
    p.all_chunks = p.chunks[0] + p.chunks[1];
    p.rows = groups * rows * heads;
    return p;
}

size_t aligned(size_t n) { return (n + 255) / 256 * 256; }

bool sizes_ok(int64_t groups, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t shared, int64_t own) {
    if (dim > 256 || rows * heads > (1 << 20) || shared > (1 << 30) || own > (1 << 30) || groups > INT32_MAX) return false;
    // (CTAs of the largest grid)
    return groups * rows * heads <= INT32_MAX / (2 + (shared + own) / 64);
}

}  // namespace
}  // namespace pamk

extern "C" {

size_t pamk_cached_attention_workspace_bytes(int64_t groups, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
                                             int64_t shared, int64_t own) {
    using namespace pamk;
    if (groups <= 0 || rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || shared < 0 || own < 0) return 0;
    if (!sizes_ok(groups, rows, heads, kv_heads, dim, shared, own)) return 0;
    const Plan p = plan_of(groups, rows, heads, kv_heads, dim, shared, own);
    return aligned(p.rows * p.width * 4) + aligned(p.rows * p.all_chunks * 8) + (p.all_chunks > 1 ? aligned(p.rows * p.all_chunks * dim * 4) : 0);
}

int pamk_cached_attention(const float* q, float* out, const float* shared_k, const float* shared_v, const int64_t* shared_lengths,
                          const float* own_k, const float* own_v, const int64_t* own_lengths,
                          int64_t groups, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t shared, int64_t own,
                          const int64_t* strides, float offset, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace pamk;
    if (groups < 0 || rows < 0 || heads < 0 || kv_heads < 1 || dim < 0 || shared < 0 || own < 0 || heads % kv_heads || !strides) return PAMK_ERR_ARG;
    if (groups == 0 || rows == 0 || heads == 0 || dim == 0) return PAMK_OK;
    if (!q || !out || (shared && (!shared_k || !shared_v)) || (own && (!own_k || !own_v))) return PAMK_ERR_ARG;
    if (!sizes_ok(groups, rows, heads, kv_heads, dim, shared, own)) return PAMK_ERR_SIZE;
    cudaStream_t st = (cudaStream_t)stream;
    if (shared + own == 0) {
        const cudaError_t err = cudaMemsetAsync(out, 0, (size_t)(groups * rows * heads * dim) * 4, st);
        return err == cudaSuccess ? PAMK_OK : record_cuda_error(err);
    }
    const Plan p = plan_of(groups, rows, heads, kv_heads, dim, shared, own);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
        workspace_bytes < pamk_cached_attention_workspace_bytes(groups, rows, heads, kv_heads, dim, shared, own))
        return PAMK_ERR_WORKSPACE;
    Attention a{};
    a.q = q; a.out = out;
    a.q_group = strides[0]; a.q_row = strides[1]; a.q_head = strides[2];
    a.groups = (int)groups; a.rows = (int)rows; a.kv_heads = (int)kv_heads; a.share = (int)(heads / kv_heads); a.dim = (int)dim;
    a.off = offset_bits(offset);
    char* ws = static_cast<char*>(workspace);
    a.scores = reinterpret_cast<float*>(ws);
    ws += aligned(p.rows * p.width * 4);
    a.stats = reinterpret_cast<float2*>(ws);
    ws += aligned(p.rows * p.all_chunks * 8);
    a.parts = reinterpret_cast<float*>(ws);
    a.width = p.width;
    a.chunks = p.all_chunks;
    Segment seg[2] = {};
    seg[0].k = shared_k; seg[0].v = shared_v; seg[0].lengths = shared_lengths;
    seg[0].k_group = strides[3]; seg[0].k_pos = strides[4]; seg[0].k_head = strides[5];
    seg[0].v_group = strides[6]; seg[0].v_pos = strides[7]; seg[0].v_head = strides[8];
    seg[0].slots = (int)shared; seg[0].rows = a.rows * a.share;
    seg[1].k = own_k; seg[1].v = own_v; seg[1].lengths = own_lengths;
    seg[1].k_group = strides[9]; seg[1].k_row = strides[10]; seg[1].k_pos = strides[11]; seg[1].k_head = strides[12];
    seg[1].v_group = strides[13]; seg[1].v_row = strides[14]; seg[1].v_pos = strides[15]; seg[1].v_head = strides[16];
    seg[1].slots = (int)own; seg[1].rows = a.share; seg[1].per_row = 1;
    seg[1].first_pos = (int)shared; seg[1].first_chunk = p.chunks[0];
    // 16-byte loads: every address that starts a row of a head is a multiple of 16 bytes
    bool vec = dim % 4 == 0 && aligned16(q);
    for (int i = 0; i < 3; ++i) vec = vec && strides[i] % 4 == 0;
    if (shared) {
        vec = vec && aligned16(shared_k) && aligned16(shared_v);
        for (int i = 3; i < 9; ++i) vec = vec && strides[i] % 4 == 0;
    }
    if (own) {
        vec = vec && aligned16(own_k) && aligned16(own_v);
        for (int i = 9; i < 17; ++i) vec = vec && strides[i] % 4 == 0;
    }
    bool behind = false;
    for (int pass = 0; pass < 2; ++pass)
        for (int i = 0; i < 2; ++i) {
            if (!seg[i].slots) continue;
            seg[i].chunk = p.chunk[i]; seg[i].chunks = p.chunks[i]; seg[i].tiles = p.tiles[i];
            const int64_t ctas = groups * kv_heads * (i ? rows : 1) * p.tiles[i] * p.chunks[i];
            const int status = launch_slots(vec, p.slots, p.tile_rows[i], pass, behind, a, seg[i], ctas, p.chunk[i] > 64 ? 256 : 128, st);
            if (status != PAMK_OK) return status;
            behind = true;
        }
    if (a.chunks > 1) return launch_behind(join_kernel, dim3((unsigned)p.rows), dim <= 64 ? 64 : 128, st, a);
    return PAMK_OK;
}

}
