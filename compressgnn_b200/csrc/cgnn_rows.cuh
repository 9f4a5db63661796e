// Rows of a matrix held by teams of lanes: what the row operators of a training step (normalisation, loss) share.
//
// A team of TEAM lanes holds one row in registers, VPL vectors of VW elements a lane; lane l has the vectors
// l, l + TEAM, ...  Teams of up to 32 lanes lie inside a warp and meet by shuffles, larger ones are a whole block.
// Elements are widened on arrival: sums and statistics are fp32 for the 16-bit types and fp32, fp64 for fp64.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cgnn_common.cuh"

namespace cgnn {

template <typename T>
struct AccOf {
    using type = float;
};
template <>
struct AccOf<double> {
    using type = double;
};
template <typename T>
using Acc = typename AccOf<T>::type;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

// The one rounding of a result to its type.
template <typename T>
__device__ __forceinline__ T narrow(Acc<T> x) {
    if constexpr (sizeof(T) == 2 && !__is_same(T, __half)) return __float2bfloat16_rn(x);
    else if constexpr (sizeof(T) == 2) return __float2half_rn(x);
    else return x;
}

// (16-bit types go in pairs: one conversion instruction packs two of them)
template <typename T, int VW>
__device__ __forceinline__ void widen_all(const Vec<T, VW> &x, Acc<T> (&y)[VW]) {
    if constexpr (__is_same(T, __nv_bfloat16) && VW % 2 == 0) {
        const uint32_t *pairs = reinterpret_cast<const uint32_t *>(&x);
#pragma unroll
        for (int k = 0; k < VW; k += 2) {  // a bf16 is the upper half of the same number in fp32
            y[k] = __uint_as_float(pairs[k / 2] << 16);
            y[k + 1] = __uint_as_float(pairs[k / 2] & 0xffff0000u);
        }
    } else if constexpr (__is_same(T, __half) && VW % 2 == 0) {
        const __half2 *pairs = reinterpret_cast<const __half2 *>(&x);
#pragma unroll
        for (int k = 0; k < VW; k += 2) {
            const float2 two = __half22float2(pairs[k / 2]);
            y[k] = two.x;
            y[k + 1] = two.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) y[k] = widen(x.v[k]);
    }
}

template <typename T, int VW>
__device__ __forceinline__ Vec<T, VW> narrow_all(const Acc<T> (&y)[VW]) {
    Vec<T, VW> r;
    if constexpr (__is_same(T, __nv_bfloat16) && VW % 2 == 0) {
#pragma unroll
        for (int k = 0; k < VW; k += 2)
            *reinterpret_cast<__nv_bfloat162 *>(&r.v[k]) = __floats2bfloat162_rn(y[k], y[k + 1]);
    } else if constexpr (__is_same(T, __half) && VW % 2 == 0) {
#pragma unroll
        for (int k = 0; k < VW; k += 2) *reinterpret_cast<__half2 *>(&r.v[k]) = __floats2half2_rn(y[k], y[k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) r.v[k] = narrow<T>(y[k]);
    }
    return r;
}

// VW parameters (weight or bias) from `at` on, of the matrix' type or, beside 16-bit matrices, fp32.
template <typename T, int VW>
__device__ __forceinline__ void load_params(const void *params, bool wide, int64_t at, Acc<T> (&y)[VW]) {
    if (sizeof(T) == 2 && wide) {
        const float *p = static_cast<const float *>(params) + at;
#pragma unroll
        for (int k = 0; k < VW; ++k) y[k] = (Acc<T>)__ldg(p + k);
    } else {
        const T *p = static_cast<const T *>(params) + at;
#pragma unroll
        for (int k = 0; k < VW; ++k) y[k] = widen(p[k]);
    }
}

__device__ __forceinline__ float inverse_root(float x) { return rsqrtf(x); }
__device__ __forceinline__ double inverse_root(double x) { return 1.0 / sqrt(x); }
__device__ __forceinline__ float fused(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return fma(a, b, c); }

// Lanes of the caller's team.
template <int TEAM>
__device__ __forceinline__ unsigned team_mask() {
    if constexpr (TEAM >= 32) return 0xffffffffu;
    else return ((1u << TEAM) - 1u) << ((threadIdx.x & 31) & ~(TEAM - 1));
}

// The sums of N values over the team, on every lane, in a fixed order.  `shared` holds 2 * N * TEAM / 32 values for a
// team of more than a warp, and `turn` counts its calls: two buffers in turn, so that one barrier a call is enough.
template <typename A, int TEAM, int N>
__device__ __forceinline__ void team_sum(A (&s)[N], A *shared, int &turn) {
    const unsigned mask = team_mask<TEAM>();
#pragma unroll
    for (int off = (TEAM < 32 ? TEAM : 32) / 2; off > 0; off >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n) s[n] += __shfl_xor_sync(mask, s[n], off);
    if constexpr (TEAM > 32) {
        constexpr int WARPS = TEAM / 32;
        A *mine = shared + (turn & 1) * N * WARPS;
        ++turn;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) mine[n * WARPS + (threadIdx.x >> 5)] = s[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            s[n] = A(0);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) s[n] += mine[n * WARPS + w];
        }
    }
}

}  // namespace cgnn
