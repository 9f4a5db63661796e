// Dropout whose mask is never stored: out = residual + x * keep / (1 - p), where keep is a function of (key, element).
//
// The backward pass is the same pass over the incoming gradient, so nothing is saved between the two.
#include "cgnn_dropout.cuh"
#include "cgnn_rows.cuh"

namespace cgnn {

constexpr int SMS = 148;

template <typename T>
struct DropArgs {
    const T *x, *residual;  // residual: optional
    T *out;
    int64_t n;
    Drop drop;
};

// A block takes tiles of whole vectors, UNITS a thread, side by side; the elements behind the last tile and arrays that
// do not lie on vector boundaries go element by element, a thread per block of four random words.
// Memory bounds it in fp32: 325,557 x 256 with a residual 144 us for 1.0 GB (two units a thread: 154).
// In bf16, 63 us for 333 MB (51 us) and 84 us with a residual (76 us).
template <typename T, int VW, int UNITS, bool ADDED>
__global__ void __launch_bounds__(256) dropout_kernel(const DropArgs<T> a, int64_t tiles) {
    using A = Acc<T>;
    Philox words(a.drop.key());
    const A scale = (A)a.drop.scale;
    constexpr int TILE = 256 * VW * UNITS;
    for (int64_t i = blockIdx.x; i < tiles; i += gridDim.x) {
        const T *const x = a.x + i * TILE, *const residual = ADDED ? a.residual + i * TILE : nullptr;
        T *const out = a.out + i * TILE;
        Vec<T, VW> v[UNITS], r[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int at = (u * 256 + threadIdx.x) * VW;
            v[u] = vec_load<T, VW>(x + at);
            if (ADDED) r[u] = vec_load<T, VW>(residual + at);
        }
        PhiloxRun run(words, (uint64_t)(i * (TILE / 4)), TILE / 4);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int at = (u * 256 + threadIdx.x) * VW;
            A y[VW];
            widen_all<T, VW>(v[u], y);
            drop_blocks<A, VW>(y, (uint32_t)at / 4, a.drop.threshold, scale, run);
            if (ADDED) {
                A z[VW];
                widen_all<T, VW>(r[u], z);
                add(z, y);
            }
            vec_store<T, VW>(out + at, narrow_all<T, VW>(y));
        }
    }
    const int64_t done = tiles * TILE;
    for (int64_t first = done + ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; first < a.n; first += (int64_t)gridDim.x * 256 * 4) {
        const uint4 q = words((uint64_t)first >> 2);
        const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (first + k < a.n) {
                A y = word[k] < a.drop.threshold ? A(0) : widen(a.x[first + k]) * scale;
                if (ADDED) y += widen(a.residual[first + k]);
                a.out[first + k] = narrow<T>(y);
            }
    }
}

template <typename T, bool ADDED>
static int dropout_typed(const DropArgs<T> &a, cudaStream_t stream) {
    constexpr int VW = sizeof(T) == 2 ? 8 : 4, UNITS = 4, TILE = 256 * VW * UNITS;
    const bool vectors = (((uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.out) & (sizeof(T) * VW - 1)) == 0;
    const int64_t tiles = vectors ? a.n / TILE : 0, rest = ceil_div(a.n - tiles * TILE, 1024);
    static const int resident = resident_blocks(dropout_kernel<T, VW, UNITS, ADDED>, 256);
    const unsigned blocks = (unsigned)std::min<int64_t>(std::max(tiles, rest), SMS * resident);
    dropout_kernel<T, VW, UNITS, ADDED><<<blocks, 256, 0, stream>>>(a, tiles);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

template <typename T>
static int dropout(int64_t n, const void *x, const void *residual, const Drop &drop, void *out, cudaStream_t stream) {
    const DropArgs<T> a{(const T *)x, (const T *)residual, (T *)out, n, drop};
    return residual ? dropout_typed<T, true>(a, stream) : dropout_typed<T, false>(a, stream);
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
