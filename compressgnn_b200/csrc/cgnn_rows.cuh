// Rows of a matrix held by teams of lanes: what the row operators of a training step (normalisation, loss) share.
//
// A team of TEAM lanes holds one row in registers, VPL vectors of VW elements a lane; lane l has the vectors
// l, l + TEAM, ...  Teams of up to 32 lanes lie inside a warp and meet by shuffles, larger ones are a whole block.
// Elements are widened on arrival: sums and statistics are fp32 for the 16-bit types and fp32, fp64 for fp64.
#pragma once

#include <algorithm>

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

// VW parameters (weight or bias) from `at` on, of the matrix' type or, beside 16-bit matrices, fp32.  whole: they begin on
// a 32-byte boundary.
template <typename T, int VW>
__device__ __forceinline__ void load_params(const void *params, bool wide, bool whole, int64_t at, Acc<T> (&y)[VW]) {
    if constexpr (sizeof(T) == 2) {
        if (wide) {
            const float *p = static_cast<const float *>(params) + at;
            if constexpr (VW == 8) {
                if (whole) {
                    // In one instruction: two of 16 bytes would each touch every other half line.  (volatile: an address may
                    // be good under the caller's conditions only, and a plain asm may be moved before them)
                    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                        : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]), "=f"(y[4]), "=f"(y[5]), "=f"(y[6]), "=f"(y[7])
                        : "l"(p));
                    return;
                }
            }
#pragma unroll
            for (int k = 0; k < VW; ++k) y[k] = p[k];
            return;
        }
    }
    const T *p = static_cast<const T *>(params) + at;
    if (whole) {
        widen_all<T, VW>(vec_load<T, VW>(p), y);
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) y[k] = widen(p[k]);
    }
}

// Arithmetic on a lane's vector.  fp32 has instructions for two numbers at once, which round like the single ones.
template <int VW>
__device__ __forceinline__ void add_to_all(float (&v)[VW], float a) {
    if constexpr (VW % 2 == 0) {
#pragma unroll
        for (int k = 0; k < VW; k += 2) {
            const float2 d = __fadd2_rn(make_float2(v[k], v[k + 1]), make_float2(a, a));
            v[k] = d.x;
            v[k + 1] = d.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) v[k] += a;
    }
}
template <int VW>
__device__ __forceinline__ void add_to_all(double (&v)[VW], double a) {
#pragma unroll
    for (int k = 0; k < VW; ++k) v[k] += a;
}
template <int VW>
__device__ __forceinline__ void multiply_all(float (&v)[VW], float a) {
    if constexpr (VW % 2 == 0) {
#pragma unroll
        for (int k = 0; k < VW; k += 2) {
            const float2 d = __fmul2_rn(make_float2(v[k], v[k + 1]), make_float2(a, a));
            v[k] = d.x;
            v[k + 1] = d.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) v[k] *= a;
    }
}
template <int VW>
__device__ __forceinline__ void multiply_all(double (&v)[VW], double a) {
#pragma unroll
    for (int k = 0; k < VW; ++k) v[k] *= a;
}
template <int VW>
__device__ __forceinline__ void multiply_pairwise(float (&v)[VW], const float (&w)[VW]) {
    if constexpr (VW % 2 == 0) {
#pragma unroll
        for (int k = 0; k < VW; k += 2) {
            const float2 d = __fmul2_rn(make_float2(v[k], v[k + 1]), make_float2(w[k], w[k + 1]));
            v[k] = d.x;
            v[k + 1] = d.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) v[k] *= w[k];
    }
}
template <int VW>
__device__ __forceinline__ void multiply_pairwise(double (&v)[VW], const double (&w)[VW]) {
#pragma unroll
    for (int k = 0; k < VW; ++k) v[k] *= w[k];
}
// s += a * b, element by element, a vector's elements by turns into the SUMS places of s (SUMS == VW: each its own).
template <int VW, int SUMS>
__device__ __forceinline__ void multiply_add(const float (&a)[VW], const float (&b)[VW], float (&s)[SUMS]) {
    if constexpr (VW % 2 == 0 && SUMS % 2 == 0) {
#pragma unroll
        for (int k = 0; k < VW; k += 2) {
            const float2 d = __ffma2_rn(make_float2(a[k], a[k + 1]), make_float2(b[k], b[k + 1]),
                                        make_float2(s[k % SUMS], s[k % SUMS + 1]));
            s[k % SUMS] = d.x;
            s[k % SUMS + 1] = d.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) s[k % SUMS] = fmaf(a[k], b[k], s[k % SUMS]);
    }
}
template <int VW, int SUMS>
__device__ __forceinline__ void multiply_add(const double (&a)[VW], const double (&b)[VW], double (&s)[SUMS]) {
#pragma unroll
    for (int k = 0; k < VW; ++k) s[k % SUMS] = fma(a[k], b[k], s[k % SUMS]);
}
template <int VW, int SUMS>
__device__ __forceinline__ void add(const float (&a)[VW], float (&s)[SUMS]) {
    if constexpr (VW % 2 == 0 && SUMS % 2 == 0) {
#pragma unroll
        for (int k = 0; k < VW; k += 2) {
            const float2 d = __fadd2_rn(make_float2(a[k], a[k + 1]), make_float2(s[k % SUMS], s[k % SUMS + 1]));
            s[k % SUMS] = d.x;
            s[k % SUMS + 1] = d.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) s[k % SUMS] += a[k];
    }
}
template <int VW, int SUMS>
__device__ __forceinline__ void add(const double (&a)[VW], double (&s)[SUMS]) {
#pragma unroll
    for (int k = 0; k < VW; ++k) s[k % SUMS] += a[k];
}
// z = h * w + b
template <int VW>
__device__ __forceinline__ void multiply_add_to(const float (&h)[VW], const float (&w)[VW], const float (&b)[VW], float (&z)[VW]) {
    if constexpr (VW % 2 == 0) {
#pragma unroll
        for (int k = 0; k < VW; k += 2) {
            const float2 d = __ffma2_rn(make_float2(h[k], h[k + 1]), make_float2(w[k], w[k + 1]), make_float2(b[k], b[k + 1]));
            z[k] = d.x;
            z[k + 1] = d.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) z[k] = fmaf(h[k], w[k], b[k]);
    }
}
template <int VW>
__device__ __forceinline__ void multiply_add_to(const double (&h)[VW], const double (&w)[VW], const double (&b)[VW], double (&z)[VW]) {
#pragma unroll
    for (int k = 0; k < VW; ++k) z[k] = fma(h[k], w[k], b[k]);
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

// Blocks of a kernel that run at once on a multiprocessor, for launches that walk their work in strides: blocks that begin
// when others end would double the time.
template <typename Kernel>
static int resident_blocks(Kernel *kernel, int threads) {
    int blocks = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, threads, 0) != cudaSuccess) {
        cudaGetLastError();
        return 1;
    }
    return std::max(1, blocks);
}

}  // namespace cgnn
