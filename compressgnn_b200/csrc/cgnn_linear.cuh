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
template <typename T, typename P>
static __global__ void __launch_bounds__(256) join_kernel(const P *parts, int64_t splits, int64_t n, double scale, T *out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    P sum = parts[i];
    for (int64_t s = 1; s < splits; ++s) sum += parts[s * n + i];
    out[i] = narrow<T>((Acc<T>)(sum * (P)scale));
}

template <typename T, typename P>
static int join(const P *parts, int64_t splits, int64_t n, double scale, T *out, cudaStream_t stream) {
    join_kernel<T, P><<<(unsigned)ceil_div(n, 256), 256, 0, stream>>>(parts, splits, n, scale, out);
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
