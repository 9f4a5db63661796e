// What the kernels of a dense layer share.
#pragma once

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
    // (of an infinity nothing is lost, but the second number says NaN)
    __device__ __forceinline__ double value() const { return isfinite(high) ? (double)high + (double)low : (double)high; }
};
template <>
struct LongSum<double> {
    double sum = 0.0;
    __device__ __forceinline__ void add(double x) { sum += x; }
    __device__ __forceinline__ double value() const { return sum; }
};

// Column sums of x [rows, width], of the elements that `mask` has a bit for (null: all).  A lane has a column, a warp every eighth row
// with COLUMN_UNROLL of them on their way; the grid's second dimension splits the rows: parts[blockIdx.y, column], or, of one
// split, scale times the sums themselves.
constexpr int COLUMN_WARPS = 8, COLUMN_UNROLL = 8;
constexpr int64_t COLUMN_ROWS = COLUMN_WARPS * COLUMN_UNROLL;

template <typename T, typename X>
static __global__ void __launch_bounds__(COLUMN_WARPS * 32) columns_kernel(const X *x, const uint8_t *mask, int64_t mask_pitch, int64_t rows,
                                                                           int64_t rows_per_split, int64_t width, double scale,
                                                                           double *parts, T *out) {
    __shared__ double sums[COLUMN_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c0 = (int64_t)blockIdx.x * 32, c = c0 + lane;
    const int64_t end = min(rows, ((int64_t)blockIdx.y + 1) * rows_per_split);
    LongSum<Acc<X>> sum;
    if (c < width) {
        for (int64_t row = (int64_t)blockIdx.y * rows_per_split + warp; row < end; row += COLUMN_ROWS) {
            Acc<X> v[COLUMN_UNROLL];
            uint32_t keep[COLUMN_UNROLL];
#pragma unroll
            for (int u = 0; u < COLUMN_UNROLL; ++u) {
                const int64_t r = row + u * COLUMN_WARPS;
                v[u] = r < end ? widen(x[r * width + c]) : Acc<X>(0);
                // (a row of the mask is whole 64-bit words)
                keep[u] = mask != nullptr && r < end ? *reinterpret_cast<const uint32_t *>(mask + r * mask_pitch + c0 / 8) : 0xffffffffu;
            }
#pragma unroll
            for (int u = 0; u < COLUMN_UNROLL; ++u) sum.add(keep[u] >> lane & 1 ? v[u] : Acc<X>(0));
        }
    }
    double s = sum.value();
    sums[warp][lane] = s;
    __syncthreads();
    if (warp > 0 || c >= width) return;
#pragma unroll
    for (int w = 1; w < COLUMN_WARPS; ++w) s += sums[w][lane];
    if (gridDim.y == 1) out[c] = narrow<T>((Acc<T>)(s * scale));
    else parts[blockIdx.y * width + c] = s;
}

// out[c] = scale * the sum of column c over the splits, in a fixed order.
template <typename T>
static int join_columns(const double *parts, int64_t splits, int64_t width, double scale, T *out, cudaStream_t stream) {
    columns_kernel<T, double><<<(unsigned)ceil_div(width, 32), COLUMN_WARPS * 32, 0, stream>>>(parts, nullptr, 0, splits, splits, width, scale,
                                                                                                  nullptr, out);
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
