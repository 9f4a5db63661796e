// What the kernels of a dense layer share.
#pragma once

#include "cgnn_dropout.cuh"
#include "cgnn_rows.cuh"

namespace cgnn {

// y = x W^T, dx = z W, dW = z^T x.
enum Form : int { FORWARD, INPUT, WEIGHT };

constexpr int64_t WIDEST = (int64_t)1 << 30;  // most columns of a matrix
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

}  // namespace cgnn
