// What the kernels of a dense layer share.
#pragma once

#include <type_traits>

#include "cgnn_dropout.cuh"
#include "cgnn_rows.cuh"

namespace cgnn {

// y = x W^T, dx = z W, dW = z^T x.
enum Form : int { FORWARD, INPUT, WEIGHT };

constexpr int64_t WIDEST = (int64_t)1 << 28;  // a matrix has fewer columns
constexpr int WAIT_LIMIT = 1 << 20;           // polls of a barrier in shared memory

struct Call {
    int64_t rows, in, out, stride;
    const void *x;
};

// Bytes of a row of the mask: whole 64-bit words.
__host__ __device__ __forceinline__ int64_t mask_pitch(int64_t out) { return (out + 63) / 64 * 8; }

// What follows the product of a forward pass.
template <typename T>
struct Epilogue {
    const T *bias, *residual;  // both optional
    uint8_t *mask;             // optional
    int64_t mask_pitch, width;
    int relu;
    Drop drop;

    // Element (m, n) of the output from its product; whether the ReLU and the dropout let it through.
    __device__ __forceinline__ bool element(Acc<T> &y, int64_t m, int64_t n, Philox &words) const {
        using A = Acc<T>;
        if (bias != nullptr) y += widen(bias[n]);
        bool passed = true;
        if (relu && !(y > A(0))) {
            passed = y != y;  // (a NaN stays one)
            if (!passed) y = A(0);
        }
        if (drop.threshold) {
            const int64_t e = m * width + n;
            const uint4 r = words((uint64_t)e >> 2);
            const int at = (int)(e & 3);
            const uint32_t w = at == 0 ? r.x : at == 1 ? r.y : at == 2 ? r.z : r.w;
            const bool kept = w >= drop.threshold;
            y = kept ? y * (A)drop.scale : A(0);
            passed = passed && kept;
        }
        if (residual != nullptr) y += widen(residual[m * width + n]);
        return passed;
    }
};

// out[i] = scale * the sum over the splits, in their order.
template <typename T>
static __global__ void __launch_bounds__(256) join_kernel(const Acc<T> *parts, int64_t splits, int64_t n, double scale, T *out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    Acc<T> sum = parts[i];
    for (int64_t s = 1; s < splits; ++s) sum += parts[s * n + i];
    out[i] = narrow<T>(sum * (Acc<T>)scale);
}

template <typename T>
static int join(const Acc<T> *parts, int64_t splits, int64_t n, double scale, T *out, cudaStream_t stream) {
    join_kernel<T><<<(unsigned)ceil_div(n, 256), 256, 0, stream>>>(parts, splits, n, scale, out);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

// A long sum of fp32 numbers in two of them: what the first loses by rounding goes to the second (Knuth's two-sum), which makes it as
// good as an fp64 sum of some ten thousand terms at a fraction of its time.
template <typename A>
struct LongSum {
    A high = A(0), low = A(0);
    __device__ __forceinline__ void add(A x) {
        const A s = high + x, part = s - high;
        low += (high - (s - part)) + (x - part);
        high = s;
    }
    // (Of an infinity nothing is lost, but the second number says NaN.  A sum beyond fp32's range on the way is infinite, as in fp32.)
    __device__ __forceinline__ double value() const { return isfinite(high) ? (double)high + (double)low : (double)high; }
};
template <>
struct LongSum<double> {
    double sum = 0.0;
    __device__ __forceinline__ void add(double x) { sum += x; }
    __device__ __forceinline__ double value() const { return sum; }
};

// Column sums of x [rows, width], of the elements that `mask` has a bit for (null: all).  A thread has VW neighbouring columns, 2^across
// neighbouring threads a row, each of them COLUMN_UNROLL rows on their way; the grid's second dimension splits the rows:
// parts[blockIdx.y, column], or, of one split, scale times the sums themselves.  (16-bit types: eight rows in fp32 first, which lose nothing that
// their result would keep.)  By vectors of 16 bytes HBM bounds it: 2.45 M x 256 bf16 216 us (floor 192; by a column a lane, two bytes an
// access, 1072), 325,557 x 256 fp32 78 (51).
constexpr int COLUMN_THREADS = 256, COLUMN_UNROLL = 8;

template <typename T, typename X, int VW>
static __global__ void __launch_bounds__(COLUMN_THREADS) columns_kernel(const X *x, const uint8_t *mask, int64_t mask_pitch, int64_t rows,
                                                                        int64_t rows_per_split, int64_t width, int across, double scale,
                                                                        double *parts, T *out) {
    __shared__ double sums[COLUMN_THREADS * VW];
    const int down = threadIdx.x >> across, step = COLUMN_THREADS >> across;
    const int64_t first = ((int64_t)blockIdx.x << across) * VW, c = first + (threadIdx.x & ((1 << across) - 1)) * VW;
    const int64_t end = min(rows, ((int64_t)blockIdx.y + 1) * rows_per_split);
    LongSum<Acc<X>> sum[VW];
    // (The last rows by a loop of their own: with a test at each load the compiler has them wait for each other.)
    const auto take = [&](int64_t row, [[maybe_unused]] auto all) {
        Vec<X, VW> v[COLUMN_UNROLL];
        uint32_t keep[COLUMN_UNROLL];
#pragma unroll
        for (int u = 0; u < COLUMN_UNROLL; ++u) {
            const int64_t r = row + u * step;
            v[u] = decltype(all)::value || r < end ? vec_load<X, VW>(x + r * width + c) : vec_zero<X, VW>();
            keep[u] = 0xffu;
        }
        if (mask != nullptr)
#pragma unroll
            for (int u = 0; u < COLUMN_UNROLL; ++u) {
                const int64_t r = row + u * step;
                if (decltype(all)::value || r < end) keep[u] = mask[r * mask_pitch + c / 8] >> (c % 8);  // (VW divides 8)
            }
        [[maybe_unused]] Acc<X> of_eight[VW];
#pragma unroll
        for (int u = 0; u < COLUMN_UNROLL; ++u) {
            Acc<X> y[VW];
            widen_all<X, VW>(v[u], y);
#pragma unroll
            for (int k = 0; k < VW; ++k) {
                if (!(keep[u] >> k & 1)) y[k] = Acc<X>(0);
                if constexpr (sizeof(X) == 2) of_eight[k] = u == 0 ? y[k] : of_eight[k] + y[k];
                else sum[k].add(y[k]);
            }
        }
        if constexpr (sizeof(X) == 2)
#pragma unroll
            for (int k = 0; k < VW; ++k) sum[k].add(of_eight[k]);
    };
    if (c < width) {
        int64_t row = (int64_t)blockIdx.y * rows_per_split + down;
        for (; row + (COLUMN_UNROLL - 1) * step < end; row += step * COLUMN_UNROLL) take(row, std::true_type());
        if (row < end) take(row, std::false_type());
    }
#pragma unroll
    for (int k = 0; k < VW; ++k) sums[threadIdx.x * VW + k] = sum[k].value();
    __syncthreads();
    const int columns = VW << across;  // of the block, a thread each (256 at most)
    if (threadIdx.x >= columns || first + threadIdx.x >= width) return;
    double s = 0.0;
    for (int d = 0; d < step; ++d) s += sums[d * columns + threadIdx.x];
    if (gridDim.y == 1) out[first + threadIdx.x] = narrow<T>((Acc<T>)(s * scale));
    else parts[blockIdx.y * width + first + threadIdx.x] = s;
}

// Threads for a row of the matrix, 8 to 32 (as a power of two).
__host__ __forceinline__ int columns_across(int64_t vectors) { return vectors > 16 ? 5 : vectors > 8 ? 4 : 3; }

// out[c] = scale * the sum of column c over the splits, in a fixed order.
template <typename T>
static int join_columns(const double *parts, int64_t splits, int64_t width, double scale, T *out, cudaStream_t stream) {
    constexpr int across = 3;  // (few rows: as many of them at once as there can be)
    columns_kernel<T, double, 1><<<(unsigned)ceil_div(width, 1 << across), COLUMN_THREADS, 0, stream>>>(
        parts, nullptr, 0, splits, splits, width, across, scale, nullptr, out);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

// The products on the tensor cores (fp32, bf16, fp16).
template <typename T>
size_t tiles_forward_bytes(int64_t rows, int64_t in, int64_t out);
template <typename T>
int tiles_forward(const Call &c, const T *weight, const Epilogue<T> &epilogue, T *y, void *scratch, int polls, cudaStream_t stream);
template <typename T>
size_t tiles_backward_bytes(int64_t rows, int64_t in, int64_t out);
template <typename T>
int tiles_backward(const Call &c, const T *weight, const T *grad, const uint8_t *mask, double scale, T *dx, T *dweight, T *dbias,
                   void *scratch, int polls, cudaStream_t stream);

}  // namespace cgnn
