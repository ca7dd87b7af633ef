// Embedding: rows of a table by token, scaled by a PAM product, with positions added and dropout, and the table's gradient.
//     x_i = pam(w[token_i], scale) + pos[i mod T]        y_i = kept ? pam(x_i, s) : 0       (philox.cuh; every step but the first is left out on demand)
//     dw[v] = sum over i with token_i = v, in order of i, of pam(drop'(g_i), scale)   (approximate gradients; exact ones: times slope(w[v], scale))
// with drop'(g) = kept ? pam(g, s) : 0 (exact: g slope(x, s)).  The row of the padding token has no gradient.
// A token outside the table reads nothing: its row is NaN, and it has no gradient.
#include "common.cuh"
#include "pam_scalar.cuh"
#include "philox.cuh"

namespace pamk {
namespace {

constexpr int kThreads = 256;

struct Embedding {
    const int64_t* tokens;
    const float *table, *pos;             // pos or null
    int64_t count, table_row, pos_row, pos_count, vocab, padding;
    int dim;
    bool scaled, drops;
    float scale;
    int32_t off;
    Dropping drop;
};

__device__ __forceinline__ float looked_up(const Embedding& a, int64_t i, int c) {
    const int64_t token = __ldg(reinterpret_cast<const long long*>(a.tokens) + i);
    if ((uint64_t)token >= (uint64_t)a.vocab) return quiet_nan();
    float x = __ldg(a.table + token * a.table_row + c);
    if (a.scaled) x = mul(x, a.scale, a.off);
    return a.pos ? fadd(x, __ldg(a.pos + (a.pos_count == 1 ? 0 : i % a.pos_count) * a.pos_row + c)) : x;
}

// SLOPES: g times the slope of the dropout at x, where it is kept; else y.  A thread takes four neighbouring elements of the output.
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
        float x = looked_up(a, i, c);
        if (SLOPES)
            x = bits[k] < a.drop.below ? 0.0f : mul_bwd(x, a.drop.scale, __ldg(g + e + k), a.off);
        else if (a.drops)
            x = bits[k] < a.drop.below ? 0.0f : mul(x, a.drop.scale, a.off);
        out[e + k] = x;
        if (++c == a.dim) {
            c = 0;
            ++i;
        }
    }
}

// A warp takes 32 columns of one row of the table and looks through all tokens.
template <bool SLOPES>
__global__ void __launch_bounds__(kThreads) table_grad_kernel(const Embedding a, const float* g, float* dw) {
    const int lane = threadIdx.x & 31, c = blockIdx.y * 32 + lane;
    const int64_t v = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (v >= a.vocab) return;
    const uint2 key = a.drops ? key_of(a.drop) : make_uint2(0u, 0u);
    const bool in = c < a.dim;
    const float slope = SLOPES && a.scaled && in ? mul_slope(__ldg(a.table + v * a.table_row + c), a.scale, a.off) : 1.0f;
    float sum = 0.0f;
    if (v != a.padding) {
        for (int64_t first = 0; first < a.count; first += 32) {
            const int64_t j = first + lane;
            uint32_t here = __ballot_sync(0xffffffffu, j < a.count && a.tokens[j] == v);
            for (; here; here &= here - 1) {
                const int64_t e = (first + __ffs(here) - 1) * a.dim + c;
                if (!in) continue;
                float x = __ldg(g + e);
                if (a.drops) x = philox_word((uint64_t)e, key) < a.drop.below ? 0.0f : mul(x, a.drop.scale, a.off);
                if (a.scaled) x = SLOPES ? fmul(x, slope) : mul(x, a.scale, a.off);
                sum = fadd(sum, x);
            }
        }
    }
    if (in) dw[v * a.dim + c] = sum;
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
    a.scale = scale;
    a.off = offset_bits(offset);
    a.drops = p > 0.0;
    if (a.drops) a.drop = dropping(p, seed_at, seed);
    return a;
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
    const int64_t ctas = (count * dim + 4 * kThreads - 1) / (4 * kThreads);
    if (ctas > 0x7fffffff) return PAMK_ERR_SIZE;
    (dy ? embed_kernel<true> : embed_kernel<false>)<<<(unsigned)ctas, kThreads, 0, (cudaStream_t)stream>>>(a, dy, out);
    return check_launch();
}

size_t pamk_embedding_bwd_workspace_bytes(int64_t count, int64_t vocab, int64_t dim) { return 0 * (size_t)(count + vocab + dim); }

int pamk_embedding_bwd(const int64_t* tokens, const float* dy, const float* table, float* dtable, int64_t count, int64_t vocab, int64_t dim, int64_t table_row,
                       int64_t padding, int has_scale, float scale, double p, const int64_t* seed_at, int64_t seed, float offset, int approx_bwd, void* workspace,
                       size_t workspace_bytes, void* stream) {
    using namespace pamk;
    if (dim < 0 || dim > 0x7fffffff - 4) return dim < 0 ? PAMK_ERR_ARG : PAMK_ERR_SIZE;
    const Embedding a = described(tokens, table, nullptr, count, vocab, dim, table_row, 0, 0, padding, has_scale, scale, p, seed_at, seed, offset);
    if (const int status = check_sizes(a, p)) return status;
    if (vocab == 0 || dim == 0) return PAMK_OK;
    if (!dtable || (count > 0 && (!tokens || !dy)) || (!approx_bwd && (a.drops || (has_scale && !table)))) return PAMK_ERR_ARG;
    const int64_t columns = (dim + 31) / 32;
    if (columns > 65535) return PAMK_ERR_SIZE;
    (approx_bwd ? table_grad_kernel<false> : table_grad_kernel<true>)<<<dim3((unsigned)((vocab + 7) / 8), (unsigned)columns), kThreads, 0, (cudaStream_t)stream>>>(a, dy, dtable);
    return check_launch();
}

}
