// Softmax cross entropy of class scores over the labelled nodes, with the gradient of the scores.
//
// Row i with label t:  loss_i = lse(z_i) - z_i[t],  dz_i = (softmax(z_i) - onehot(t)) * share_i.  A row whose label is
// `ignore_index` has no loss and a gradient of zeros, and its scores are not read; a label that is no class is treated
// the same and sets a status bit.  share_i is the incoming gradient, for a mean over the number of labelled rows.
//
// Memory bounds it.  For a sum or a mean the forward pass writes the gradient for an incoming gradient of one beside the
// loss, from the row it holds anyway: the scores are read once a step, not twice.  Losses are added up in fp64 and in a
// fixed order.
#include <algorithm>

#include "cgnn_rows.cuh"

namespace cgnn {

static __device__ int g_loss_status = 0;

int loss_status(int *out) {
    int zero = 0;
    CGNN_CUDA(cudaMemcpyFromSymbol(out, g_loss_status, sizeof(int)));
    CGNN_CUDA(cudaMemcpyToSymbol(g_loss_status, &zero, sizeof(int)));
    return CGNN_OK;
}

constexpr int SMS = 148;
constexpr int LOSS_THREADS = 256;
constexpr int LOSS_BLOCKS = SMS * 8;  // most blocks of a launch, each of which leaves a partial sum
constexpr int COUNT_THREADS = 1024;

template <typename T>
struct LossArgs {
    using A = Acc<T>;
    const T *logits;
    int64_t rows, classes, stride;
    const int64_t *target;
    int64_t ignore_index;
    int reduction;
    const int64_t *labelled;  // number of labelled rows (a mean's divisor), on the device
    A *stats;                 // [rows, 2]: a row's largest score, 1 / sum exp(z - it); forward: written unless null
    A *row_loss;              // forward without reduction: [rows]
    double *partial;          // forward with reduction: [blocks]
    T *grad;                  // optional in the forward pass
    const A *upstream;        // backward: one value, or one per row without reduction
    int skip_one;             // backward: `grad` holds the gradient for an incoming one already
};

// The class of a row, or -1 for a row without one.
__device__ __forceinline__ int64_t class_of(int64_t t, int64_t classes, int64_t ignore_index, bool report) {
    if (t == ignore_index) return -1;
    if (t < 0 || t >= classes) {
        if (report) atomicOr(&g_loss_status, STATUS_BAD_INDEX);
        return -1;
    }
    return t;
}

__device__ __forceinline__ float exponential(float x) { return __expf(x); }
__device__ __forceinline__ double exponential(double x) { return exp(x); }
__device__ __forceinline__ float logarithm(float x) { return logf(x); }
__device__ __forceinline__ double logarithm(double x) { return log(x); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

// What a row's gradient is multiplied by before the incoming gradient: a mean's share is rounded once.
template <typename T>
__device__ __forceinline__ Acc<T> share_of(const LossArgs<T> &a, double upstream) {
    return (Acc<T>)(a.reduction == CGNN_MEAN ? upstream / (double)*a.labelled : upstream);
}

// Adds the threads' sums up in thread order (tree), on thread 0.
template <int THREADS>
__device__ __forceinline__ double block_sum(double s) {
    __shared__ double sums[THREADS / 32];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0)
#pragma unroll
        for (int w = 1; w < THREADS / 32; ++w) s += sums[w];
    return s;
}

// The number of labelled rows (one block per range; whole numbers, so the order of the additions does not matter).
__global__ void __launch_bounds__(COUNT_THREADS) loss_count_kernel(const int64_t *target, int64_t rows, int64_t classes,
                                                                   int64_t ignore_index, int64_t *labelled) {
    int mine = 0;
    for (int64_t r = (int64_t)blockIdx.x * COUNT_THREADS + threadIdx.x; r < rows; r += (int64_t)gridDim.x * COUNT_THREADS)
        mine += class_of(target[r], classes, ignore_index, false) >= 0;
    mine = __reduce_add_sync(0xffffffffu, mine);
    __shared__ int sums[COUNT_THREADS / 32];
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t all = 0;
        for (int w = 0; w < COUNT_THREADS / 32; ++w) all += sums[w];
        atomicAdd(reinterpret_cast<unsigned long long *>(labelled), (unsigned long long)all);
    }
}

// Rows in the registers of a team.  FORWARD: losses, and the gradient for an incoming one where wanted; otherwise the
// gradient from the saved statistics.
template <typename T, int VW, int TEAM, int VPL, bool FORWARD>
__global__ void __launch_bounds__(LOSS_THREADS) loss_kernel(const LossArgs<T> a) {
    using A = Acc<T>;
    if (!FORWARD && a.skip_one && *a.upstream == A(1)) return;
    constexpr int TEAMS = LOSS_THREADS / TEAM;
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
    const unsigned mask = team_mask<TEAM>();
    double total = 0.0;
    A share = A(0);
    if (a.grad && !(!FORWARD && a.reduction == CGNN_NONE)) share = share_of(a, FORWARD ? 1.0 : (double)*a.upstream);
    for (int64_t r = (int64_t)blockIdx.x * TEAMS + team; r < a.rows; r += (int64_t)gridDim.x * TEAMS) {
        const int64_t t = class_of(a.target[r], a.classes, a.ignore_index, FORWARD && lane == 0);
        A v[VPL][VW];
        if (t >= 0) {
            const T *row = a.logits + r * a.stride;
            Vec<T, VW> raw[VPL];
#pragma unroll
            for (int p = 0; p < VPL; ++p) {
                const int col = (p * TEAM + lane) * VW;
                if (col < a.classes) raw[p] = vec_load<T, VW>(row + col);
            }
#pragma unroll
            for (int p = 0; p < VPL; ++p) widen_all<T, VW>(raw[p], v[p]);
            A m = -(A)INFINITY, inv;
            if constexpr (FORWARD) {
#pragma unroll
                for (int p = 0; p < VPL; ++p)
                    if ((p * TEAM + lane) * VW < a.classes)
#pragma unroll
                        for (int k = 0; k < VW; ++k) m = larger(m, v[p][k]);
#pragma unroll
                for (int off = TEAM / 2; off > 0; off >>= 1) m = larger(m, __shfl_xor_sync(mask, m, off));
                A s = A(0);
#pragma unroll
                for (int p = 0; p < VPL; ++p)
                    if ((p * TEAM + lane) * VW < a.classes)
#pragma unroll
                        for (int k = 0; k < VW; ++k) s += exponential(v[p][k] - m);
#pragma unroll
                for (int off = TEAM / 2; off > 0; off >>= 1) s += __shfl_xor_sync(mask, s, off);
                inv = A(1) / s;
                if (lane == 0) {
                    // (the label's score and the largest one first: both may be large beside their difference)
                    const A loss = logarithm(s) + (m - widen(row[t]));
                    if (a.row_loss) a.row_loss[r] = loss;
                    total += (double)loss;
                    if (a.stats) {
                        a.stats[2 * r] = m;
                        a.stats[2 * r + 1] = inv;
                    }
                }
            } else {
                m = a.stats[2 * r];
                inv = a.stats[2 * r + 1];
                if (a.reduction == CGNN_NONE) share = a.upstream[r];
            }
            if (a.grad)
#pragma unroll
                for (int p = 0; p < VPL; ++p)
#pragma unroll
                    for (int k = 0; k < VW; ++k) v[p][k] = exponential(v[p][k] - m) * inv;
        } else if (FORWARD && lane == 0) {
            if (a.row_loss) a.row_loss[r] = A(0);
        }
        if (!a.grad) continue;
#pragma unroll
        for (int p = 0; p < VPL; ++p) {
            const int col = (p * TEAM + lane) * VW;
            if (col >= a.classes) continue;
            A d[VW];
#pragma unroll
            for (int k = 0; k < VW; ++k) d[k] = t >= 0 ? (v[p][k] - (col + k == t ? A(1) : A(0))) * share : A(0);
            vec_store<T, VW>(a.grad + r * a.classes + col, narrow_all<T, VW>(d));
        }
    }
    if constexpr (FORWARD) {
        if (!a.partial) return;
        const double s = block_sum<LOSS_THREADS>(total);
        if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
    }
}

// Rows too long for registers: a block per row, which passes over it twice (the second time out of L2).
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(LOSS_THREADS) loss_long_kernel(const LossArgs<T> a) {
    using A = Acc<T>;
    if (!FORWARD && a.skip_one && *a.upstream == A(1)) return;
    __shared__ A maxima[LOSS_THREADS / 32], sums[LOSS_THREADS / 32];
    double total = 0.0;
    A share = A(0);
    if (a.grad && !(!FORWARD && a.reduction == CGNN_NONE)) share = share_of(a, FORWARD ? 1.0 : (double)*a.upstream);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int64_t t = class_of(a.target[r], a.classes, a.ignore_index, FORWARD && threadIdx.x == 0);
        const T *row = a.logits + r * a.stride;
        A m = A(0), scale = A(1);
        if (t >= 0) {
            if constexpr (FORWARD) {
                m = -(A)INFINITY;
                for (int64_t c = threadIdx.x; c < a.classes; c += LOSS_THREADS) m = larger(m, widen(row[c]));
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, off));
                if ((threadIdx.x & 31) == 0) maxima[threadIdx.x >> 5] = m;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < LOSS_THREADS / 32; ++w) m = larger(m, maxima[w]);
                A s = A(0);
                for (int64_t c = threadIdx.x; c < a.classes; c += LOSS_THREADS) s += exponential(widen(row[c]) - m);
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
                if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
                __syncthreads();
                s = A(0);
#pragma unroll
                for (int w = 0; w < LOSS_THREADS / 32; ++w) s += sums[w];
                if (threadIdx.x == 0) {
                    const A loss = logarithm(s) + (m - widen(row[t]));
                    if (a.row_loss) a.row_loss[r] = loss;
                    total += (double)loss;
                    if (a.stats) {
                        a.stats[2 * r] = m;
                        a.stats[2 * r + 1] = A(1) / s;
                    }
                }
                scale = A(1) / s;
            } else {
                m = a.stats[2 * r];
                scale = a.stats[2 * r + 1];
                if (a.reduction == CGNN_NONE) share = a.upstream[r];
            }
        } else if (FORWARD && threadIdx.x == 0) {
            if (a.row_loss) a.row_loss[r] = A(0);
        }
        if (!a.grad) continue;
        T *out = a.grad + r * a.classes;
        for (int64_t c = threadIdx.x; c < a.classes; c += LOSS_THREADS)
            out[c] = narrow<T>(t >= 0 ? (exponential(widen(row[c]) - m) * scale - (c == t ? A(1) : A(0))) * share : A(0));
    }
    if constexpr (FORWARD) {
        if (!a.partial) return;
        if (threadIdx.x == 0) a.partial[blockIdx.x] = total;
    }
}

template <typename A>
__global__ void __launch_bounds__(256) loss_sum_kernel(const double *partial, int blocks, int reduction, const int64_t *labelled,
                                                       A *loss) {
    double s = 0.0;
    for (int b = threadIdx.x; b < blocks; b += 256) s += partial[b];
    s = block_sum<256>(s);
    if (threadIdx.x == 0) *loss = (A)(reduction == CGNN_MEAN ? s / (double)*labelled : s);
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
template <typename T, int VW, int TEAM, int VPL, bool FORWARD>
static int launch_team(const LossArgs<T> &a, int64_t *blocks, cudaStream_t stream) {
    *blocks = std::min<int64_t>(ceil_div(a.rows, LOSS_THREADS / TEAM), LOSS_BLOCKS);
    loss_kernel<T, VW, TEAM, VPL, FORWARD><<<(unsigned)*blocks, LOSS_THREADS, 0, stream>>>(a);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

template <typename T, int VW, bool FORWARD>
static int launch_rows(const LossArgs<T> &a, int64_t *blocks, cudaStream_t stream) {
    const int64_t vectors = a.classes / VW;
    if (vectors <= 4) return launch_team<T, VW, 4, 1, FORWARD>(a, blocks, stream);
    if (vectors <= 8) return launch_team<T, VW, 4, 2, FORWARD>(a, blocks, stream);
    if (vectors <= 16) return launch_team<T, VW, 8, 2, FORWARD>(a, blocks, stream);
    if (vectors <= 48) return launch_team<T, VW, 16, 3, FORWARD>(a, blocks, stream);
    if (vectors <= 128) return launch_team<T, VW, 32, 4, FORWARD>(a, blocks, stream);
    if (VW == 1 && vectors <= 512) return launch_team<T, VW, 32, VW == 1 ? 16 : 4, FORWARD>(a, blocks, stream);
    *blocks = std::min<int64_t>(a.rows, LOSS_BLOCKS);
    loss_long_kernel<T, FORWARD><<<(unsigned)*blocks, LOSS_THREADS, 0, stream>>>(a);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

template <typename T, bool FORWARD>
static int launch(const LossArgs<T> &a, int64_t *blocks, cudaStream_t stream) {
    constexpr int VW = 16 / (int)sizeof(T);
    const uintptr_t bits = (uintptr_t)a.logits | (uintptr_t)a.grad;
    if (a.classes % VW == 0 && a.stride % VW == 0 && (bits & 15) == 0) return launch_rows<T, VW, FORWARD>(a, blocks, stream);
    return launch_rows<T, 1, FORWARD>(a, blocks, stream);
}

static int check_call(const char *what, int dtype, int64_t rows, int64_t classes, int64_t stride, int reduction) {
    CGNN_REQUIRE(dtype >= CGNN_F32 && dtype <= CGNN_F16, "%s: unknown dtype %d", what, dtype);
    CGNN_REQUIRE(reduction >= CGNN_NONE && reduction <= CGNN_MEAN, "%s: unknown reduction %d", what, reduction);
    CGNN_REQUIRE(rows >= 0 && stride >= 0, "%s: negative size", what);
    CGNN_REQUIRE(classes >= 1 && classes <= INT32_MAX / 2, "%s: %lld classes are not supported", what, (long long)classes);
    return CGNN_OK;
}

}  // namespace cgnn

using namespace cgnn;

extern "C" {

size_t cgnn_cross_entropy_scratch_bytes(void) { return LOSS_BLOCKS * sizeof(double); }

int cgnn_cross_entropy(int dtype, int64_t rows, int64_t classes, int64_t stride, const void *logits, const int64_t *target,
                       int64_t ignore_index, int reduction, void *loss, void *stats, void *grad, int64_t *labelled, void *scratch,
                       size_t scratch_bytes, cgnn_stream_t stream_) {
    if (int rc = check_call("cross_entropy", dtype, rows, classes, stride, reduction)) return rc;
    const cudaStream_t stream = (cudaStream_t)stream_;
    CGNN_REQUIRE(reduction != CGNN_NONE || grad == nullptr, "cross_entropy: the gradient of unreduced losses takes their gradients");
    CGNN_REQUIRE(loss != nullptr || (reduction == CGNN_NONE && rows == 0), "cross_entropy: null loss");
    CGNN_REQUIRE(rows == 0 || (logits != nullptr && target != nullptr), "cross_entropy: null pointer");
    if (reduction != CGNN_NONE)
        CGNN_REQUIRE(labelled != nullptr && scratch != nullptr && scratch_bytes >= cgnn_cross_entropy_scratch_bytes() &&
                         ((uintptr_t)scratch & 7) == 0,
                     "cross_entropy: no place for the count, or the scratch is too small or not 8-byte aligned");
    if (reduction == CGNN_MEAN) {
        CGNN_CUDA(cudaMemsetAsync(labelled, 0, sizeof(int64_t), stream));
        if (rows) {
            loss_count_kernel<<<(unsigned)std::min<int64_t>(ceil_div(rows, COUNT_THREADS), SMS), COUNT_THREADS, 0, stream>>>(
                target, rows, classes, ignore_index, labelled);
            CGNN_LAUNCH_CHECK();
        }
    }
    const auto run = [&](auto zero) -> int {
        using T = decltype(zero);
        using A = Acc<T>;
        LossArgs<T> a{};
        a.logits = (const T *)logits;
        a.rows = rows;
        a.classes = classes;
        a.stride = stride;
        a.target = target;
        a.ignore_index = ignore_index;
        a.reduction = reduction;
        a.labelled = labelled;
        a.stats = (A *)stats;
        a.row_loss = reduction == CGNN_NONE ? (A *)loss : nullptr;
        a.partial = reduction == CGNN_NONE ? nullptr : (double *)scratch;
        a.grad = (T *)grad;
        int64_t blocks = 0;
        if (rows)
            if (int rc = launch<T, true>(a, &blocks, stream)) return rc;
        if (reduction == CGNN_NONE) return CGNN_OK;
        loss_sum_kernel<A><<<1, 256, 0, stream>>>(a.partial, (int)blocks, reduction, labelled, (A *)loss);
        CGNN_LAUNCH_CHECK();
        return CGNN_OK;
    };
    switch (dtype) {
        case CGNN_F32: return run(0.0f);
        case CGNN_F64: return run(0.0);
        case CGNN_BF16: return run(__nv_bfloat16());
        default: return run(__half());
    }
}

int cgnn_cross_entropy_backward(int dtype, int64_t rows, int64_t classes, int64_t stride, const void *logits,
                                const int64_t *target, int64_t ignore_index, int reduction, const void *stats,
                                const int64_t *labelled, const void *upstream, int holds_unit_gradient, void *grad,
                                cgnn_stream_t stream) {
    if (int rc = check_call("cross_entropy_backward", dtype, rows, classes, stride, reduction)) return rc;
    if (rows == 0) return CGNN_OK;
    CGNN_REQUIRE(logits != nullptr && target != nullptr && stats != nullptr && upstream != nullptr && grad != nullptr &&
                     (reduction != CGNN_MEAN || labelled != nullptr),
                 "cross_entropy_backward: null pointer");
    const auto run = [&](auto zero) -> int {
        using T = decltype(zero);
        using A = Acc<T>;
        LossArgs<T> a{};
        a.logits = (const T *)logits;
        a.rows = rows;
        a.classes = classes;
        a.stride = stride;
        a.target = target;
        a.ignore_index = ignore_index;
        a.reduction = reduction;
        a.labelled = labelled;
        a.stats = (A *)const_cast<void *>(stats);
        a.upstream = (const A *)upstream;
        a.skip_one = reduction != CGNN_NONE && holds_unit_gradient;
        a.grad = (T *)grad;
        int64_t blocks = 0;
        return launch<T, false>(a, &blocks, (cudaStream_t)stream);
    };
    switch (dtype) {
        case CGNN_F32: return run(0.0f);
        case CGNN_F64: return run(0.0);
        case CGNN_BF16: return run(__nv_bfloat16());
        default: return run(__half());
    }
}

}  // extern "C"
