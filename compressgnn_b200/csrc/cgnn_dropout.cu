// Dropout whose mask is never stored: out = residual + x * keep / (1 - p), where keep is a function of (key, element).
//
// The backward pass is the same pass over the incoming gradient, so nothing is saved between the two.
#include "cgnn_dropout.cuh"
#include "cgnn_rows.cuh"

namespace cgnn {

template <typename T>
struct DropArgs {
    const T *x, *residual;  // residual: optional
    T *out;
    int64_t n;
    Drop drop;
};

// A thread takes UNITS of VW elements (whole blocks of four random words), a block's threads side by side.  WIDE: the
// arrays lie on 16-byte boundaries and move by vectors; otherwise element by element, with the same words.
template <typename T, int VW, int UNITS, bool WIDE>
__global__ void __launch_bounds__(256) dropout_kernel(const DropArgs<T> a) {
    using A = Acc<T>;
    const uint64_t key = a.drop.key();
    const A scale = (A)a.drop.scale;
    const int64_t step = (int64_t)blockDim.x * VW;
    for (int64_t base = (int64_t)blockIdx.x * step * UNITS; base < a.n; base += (int64_t)gridDim.x * step * UNITS) {
        const int64_t first = base + threadIdx.x * VW;
        Vec<T, VW> x[UNITS], r[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int64_t at = first + u * step;
            x[u] = r[u] = vec_zero<T, VW>();
            if (WIDE && at + VW <= a.n) {
                x[u] = vec_load<T, VW>(a.x + at);
                if (a.residual) r[u] = vec_load<T, VW>(a.residual + at);
            } else {
#pragma unroll
                for (int k = 0; k < VW; ++k)
                    if (at + k < a.n) {
                        x[u].v[k] = a.x[at + k];
                        if (a.residual) r[u].v[k] = a.residual[at + k];
                    }
            }
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int64_t at = first + u * step;
            if (at >= a.n) break;
            A y[VW];
            widen_all<T, VW>(x[u], y);
            drop_values<A, VW>(y, at, a.drop.threshold, scale, key);
            if (a.residual)
#pragma unroll
                for (int k = 0; k < VW; ++k) y[k] += widen(r[u].v[k]);
            const Vec<T, VW> out = narrow_all<T, VW>(y);
            if (WIDE && at + VW <= a.n) {
                vec_store<T, VW>(a.out + at, out);
            } else {
#pragma unroll
                for (int k = 0; k < VW; ++k)
                    if (at + k < a.n) a.out[at + k] = out.v[k];
            }
        }
    }
}

template <typename T>
static int dropout(int64_t n, const void *x, const void *residual, const Drop &drop, void *out, cudaStream_t stream) {
    constexpr int VW = sizeof(T) == 2 ? 8 : 4, UNITS = 2;
    const DropArgs<T> a{(const T *)x, (const T *)residual, (T *)out, n, drop};
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(n, 256 * VW * UNITS), 148 * 8);
    if ((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)out) & (sizeof(T) * VW - 1)) == 0)
        dropout_kernel<T, VW, UNITS, true><<<blocks, 256, 0, stream>>>(a);
    else
        dropout_kernel<T, VW, UNITS, false><<<blocks, 256, 0, stream>>>(a);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

}  // namespace cgnn

using namespace cgnn;

extern "C" int cgnn_dropout(int dtype, int64_t n, const void *x, const void *residual, double p, uint64_t seed,
                            const int64_t *device_seed, void *out, cgnn_stream_t stream) {
    CGNN_REQUIRE(dtype >= CGNN_F32 && dtype <= CGNN_F16, "dropout: unknown dtype %d", dtype);
    CGNN_REQUIRE(n >= 0, "dropout: negative size");
    CGNN_REQUIRE(p >= 0.0 && p < 1.0, "dropout: the drop probability must lie in [0, 1)");
    if (n == 0) return CGNN_OK;
    CGNN_REQUIRE(x != nullptr && out != nullptr, "dropout: null pointer");
    const Drop drop = Drop::of(p, seed, device_seed);
    const cudaStream_t s = (cudaStream_t)stream;
    switch (dtype) {
        case CGNN_F32: return dropout<float>(n, x, residual, drop, out, s);
        case CGNN_F64: return dropout<double>(n, x, residual, drop, out, s);
        case CGNN_BF16: return dropout<__nv_bfloat16>(n, x, residual, drop, out, s);
        default: return dropout<__half>(n, x, residual, drop, out, s);
    }
}
