// Dropout with the PAM product, its mask drawn from a counter (philox.cuh) in both directions and never stored:
//     y_i = r_i + (kept_i ? pam(x_i, s) : 0)       s = fp32(1 / (1 - p))
//     dx_i = kept_i ? pam(g_i, s) : 0              (approximate gradients: the forward pass on g)
//     dx_i = kept_i ? g_i slope(x_i, s) : 0        (exact gradients)
// A dropped element gives zero whatever it holds.  HBM-bound (8 to 12 bytes per element), if closely: a thread takes quads of neighbouring elements, which is
// what a block of the counter has bits for, and a block is some 70 instructions.  2^26 elements: 87 us (0.94 of the copy rate, issue 75 %), with a residual 118 (1.04); with one quad
// per thread 122 and 135, with four 87 and 119.
#include "common.cuh"
#include "pam_scalar.cuh"
#include "philox.cuh"
#include "times.cuh"

namespace pamk {
namespace {

constexpr int kThreads = 256, kQuads = 2;

template <bool VEC>
__device__ __forceinline__ float4 load_quad(const float* p, int64_t i, int64_t n) {
    if (VEC && i + 4 <= n) return __ldg(reinterpret_cast<const float4*>(p + i));
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (i < n) v.x = __ldg(p + i);
    if (i + 1 < n) v.y = __ldg(p + i + 1);
    if (i + 2 < n) v.z = __ldg(p + i + 2);
    if (i + 3 < n) v.w = __ldg(p + i + 3);
    return v;
}

template <bool VEC>
__device__ __forceinline__ void store_quad(float* p, int64_t i, int64_t n, float4 v) {
    if (VEC && i + 4 <= n) {
        *reinterpret_cast<float4*>(p + i) = v;
        return;
    }
    if (i < n) p[i] = v.x;
    if (i + 1 < n) p[i + 1] = v.y;
    if (i + 2 < n) p[i + 2] = v.z;
    if (i + 3 < n) p[i + 3] = v.w;
}

// SLOPES: x is the gradient and `other` the forward pass's input; else `other` is the residual, or null.
template <bool SLOPES, bool VEC>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const float* x, const float* other, float* out, int64_t n, Dropping drop, Times by) {
    const uint2 key = key_of(drop);
    const int64_t first = ((int64_t)blockIdx.x * kQuads * kThreads + threadIdx.x) * 4;
    float4 v[kQuads], o[kQuads];
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
        const int64_t i = first + k * kThreads * 4;
        v[k] = load_quad<VEC>(x, i, n);
        o[k] = other ? load_quad<VEC>(other, i, n) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
        const int64_t i = first + k * kThreads * 4;
        if (i >= n) return;
        const uint4 w = philox((uint64_t)i >> 2, key);
        float4 y = SLOPES ? make_float4(mul_bwd(o[k].x, by.s, v[k].x, by.off), mul_bwd(o[k].y, by.s, v[k].y, by.off), mul_bwd(o[k].z, by.s, v[k].z, by.off),
                                        mul_bwd(o[k].w, by.s, v[k].w, by.off))
                          : by.of(v[k]);
        y = make_float4(w.x < drop.below ? 0.0f : y.x, w.y < drop.below ? 0.0f : y.y, w.z < drop.below ? 0.0f : y.z, w.w < drop.below ? 0.0f : y.w);
        if (!SLOPES && other) y = make_float4(fadd(y.x, o[k].x), fadd(y.y, o[k].y), fadd(y.z, o[k].z), fadd(y.w, o[k].w));
        store_quad<VEC>(out, i, n, y);
    }
}

template <bool SLOPES>
int launch(const float* x, const float* other, float* out, int64_t n, double p, const int64_t* seed_at, int64_t seed, float offset, cudaStream_t st) {
    const int64_t per_cta = (int64_t)kThreads * kQuads * 4, ctas = (n + per_cta - 1) / per_cta;
    if (ctas > 0x7fffffff) return PAMK_ERR_SIZE;
    const Dropping drop = dropping(p, seed_at, seed);
    const bool vec = aligned16(x) && aligned16(out) && aligned16(other);
    const auto kernel = vec ? dropout_kernel<SLOPES, true> : dropout_kernel<SLOPES, false>;
    kernel<<<(unsigned)ctas, kThreads, 0, st>>>(x, other, out, n, drop, Times(drop.scale, offset_bits(offset)));
    return check_launch();
}

}  // namespace
}  // namespace pamk

extern "C" {

int pamk_dropout(const float* x, const float* residual, float* out, int64_t n, double p, const int64_t* seed_at, int64_t seed, float offset, void* stream) {
    using namespace pamk;
    if (n < 0 || !(p > 0.0 && p < 1.0) || (n > 0 && (!x || !out))) return PAMK_ERR_ARG;
    return n == 0 ? PAMK_OK : launch<false>(x, residual, out, n, p, seed_at, seed, offset, (cudaStream_t)stream);
}

int pamk_dropout_bwd(const float* x, const float* dy, float* dx, int64_t n, double p, const int64_t* seed_at, int64_t seed, float offset, void* stream) {
    using namespace pamk;
    if (n < 0 || !(p > 0.0 && p < 1.0) || (n > 0 && (!x || !dy || !dx))) return PAMK_ERR_ARG;
    return n == 0 ? PAMK_OK : launch<true>(dy, x, dx, n, p, seed_at, seed, offset, (cudaStream_t)stream);
}

}
