// Softmax cross entropy of class scores over the labelled nodes, with the gradient of the scores.
//
// Row i with label t:  loss_i = lse(z_i) - z_i[t],  dz_i = (softmax(z_i) - onehot(t)) * share_i.  A row whose label is
// `ignore_index` has no loss and a gradient of zeros, and its scores are not read; a label that is no class is treated
// the same and sets a status bit.  share_i is the incoming gradient, for a mean over the number of labelled rows.
//
// Memory bounds it.  For a sum or a mean the forward pass writes the gradient for an incoming gradient of one beside the
// loss, from the copy of the row it holds anyway: the scores are read once a step, not twice.  Losses are added up in
// fp64 and in a fixed order.
#include <algorithm>

#include <cooperative_groups.h>

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
constexpr int LOSS_BLOCKS = SMS * 16;       // most blocks of a launch, each of which leaves a partial sum
constexpr int COUNT_THREADS = 1024;
constexpr int CLUSTER = 8;                  // blocks of the launch that does a small case alone
constexpr int64_t CLUSTER_ROWS = 4096;
constexpr size_t SHARED_MOST = 227 * 1024;  // of a block
constexpr int LONG_THREADS = 512;

// What the launches of one call hand each other.
struct LossScratch {
    double partial[LOSS_BLOCKS];
    int64_t counts[SMS];
    unsigned ticket;
};

template <typename T>
struct LossArgs {
    using A = Acc<T>;
    const T *logits;
    int64_t rows, classes, stride;
    const int64_t *target;
    int64_t ignore_index;
    int reduction;
    int64_t *labelled;     // the number of labelled rows (a mean's divisor): written by the forward pass, read by the backward
    A *stats;              // [rows, 2]: a row's largest score, 1 / sum exp(z - it); forward: written unless null
    A *loss;               // forward: [rows] without reduction, else one value
    LossScratch *scratch;  // forward with reduction
    int count_blocks;      // forward, mean: entries of scratch->counts
    T *grad;               // optional in the forward pass
    const A *upstream;     // backward: one value, or one per row without reduction
    int skip_one;          // backward: `grad` holds the gradient for an incoming one already
    int dense;             // rows lie one behind the other from a 16-byte boundary on, in the scores and the gradient
    uint32_t per_class;    // ceil(2^32 / classes): e / classes == umulhi(e, it) for the elements of a tile
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

// e^x for x <= 0: 2^(x * log2(e)) by the special function unit; what lies below the normal numbers is zero.
__device__ __forceinline__ float exponential(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}
__device__ __forceinline__ double exponential(double x) { return exp(x); }
__device__ __forceinline__ float logarithm(float x) { return logf(x); }
__device__ __forceinline__ double logarithm(double x) { return log(x); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

// One element of the gradient, the same arithmetic in every kernel.
template <typename A>
__device__ __forceinline__ A slope(A z, A m, A inv, bool label, A share) {
    return fused(exponential(z - m), inv, label ? A(-1) : A(0)) * share;
}

// What a row's gradient is multiplied by: a mean's share is rounded once.
template <typename T>
__device__ __forceinline__ Acc<T> share_of(const LossArgs<T> &a, double upstream, int64_t labelled) {
    return (Acc<T>)(a.reduction == CGNN_MEAN ? upstream / (double)labelled : upstream);
}

__device__ __forceinline__ void copy16(void *shared, const void *global, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(global),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The threads' values added up in a fixed order, on thread 0.
template <int THREADS, typename N>
__device__ __forceinline__ N block_sum(N s) {
    __shared__ N sums[THREADS / 32];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0)
#pragma unroll
        for (int w = 1; w < THREADS / 32; ++w) s += sums[w];
    __syncthreads();
    return s;
}

// First launch of a reduced loss: every block counts the labelled rows of its share.
__global__ void __launch_bounds__(COUNT_THREADS) loss_count_kernel(const int64_t *target, int64_t rows, int64_t classes,
                                                                   int64_t ignore_index, LossScratch *scratch) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int64_t mine = 0;
    for (int64_t r = (int64_t)blockIdx.x * COUNT_THREADS + threadIdx.x; r < rows; r += (int64_t)gridDim.x * COUNT_THREADS)
        mine += class_of(target[r], classes, ignore_index, false) >= 0;
    mine = block_sum<COUNT_THREADS>(mine);
    if (threadIdx.x) return;
    scratch->counts[blockIdx.x] = mine;
    if (blockIdx.x == 0) scratch->ticket = 0;
}

// The number of labelled rows, on every thread of a block of the launch behind that one.
template <typename T, int THREADS>
__device__ __forceinline__ int64_t labelled_rows(const LossArgs<T> &a) {
    __shared__ int64_t all;
    if (a.reduction != CGNN_MEAN) return 0;
    int64_t mine = 0;
    for (int b = threadIdx.x; b < a.count_blocks; b += THREADS) mine += a.scratch->counts[b];
    mine = block_sum<THREADS>(mine);
    if (threadIdx.x == 0) all = mine;
    __syncthreads();
    return all;
}

// The end of a reduced loss: a block leaves its sum, and the last one to do so adds all of them up in block order.
template <typename T, int THREADS>
__device__ __forceinline__ void finish(const LossArgs<T> &a, double total, int64_t labelled) {
    __shared__ bool last;
    total = block_sum<THREADS>(total);
    if (threadIdx.x == 0) {
        a.scratch->partial[blockIdx.x] = total;
        __threadfence();
        last = atomicAdd(&a.scratch->ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double s = 0.0;
    for (int b = threadIdx.x; b < (int)gridDim.x; b += THREADS) s += __ldcg(&a.scratch->partial[b]);
    s = block_sum<THREADS>(s);
    if (threadIdx.x) return;
    *a.loss = (Acc<T>)(a.reduction == CGNN_MEAN ? s / (double)labelled : s);
    *a.labelled = labelled;
}

// Columns lane, lane + LANES, ... of a row, beginning at `start` (a multiple of LANES) and around.
template <int LANES, typename F>
__device__ __forceinline__ void for_columns(int classes, int lane, int start, F &&f) {
#pragma unroll 4
    for (int c = lane + start; c < classes; c += LANES) f(c);
    const int end = min(lane + start, classes);
#pragma unroll 4
    for (int c = lane; c < end; c += LANES) f(c);
}

// Rows of up to 1024 classes.  A block copies ROWS whole rows into shared memory as the 16-byte vectors they lie in, in
// whatever way rows and vectors meet (47 classes: 188 bytes a row), leaving out vectors of unlabelled rows alone; LANES lanes
// a row then pass over it three times (maximum, sum, gradient in place), and the gradient leaves by whole vectors.
// The lanes of a warp begin at different columns, or rows of an even length would meet in the same banks.
// CLUSTERED: the launch is one cluster, which counts the labelled rows and adds up the losses itself.
template <typename T, int LANES, int ROWS, bool FORWARD, bool CLUSTERED>
__global__ void __launch_bounds__(LANES *ROWS) loss_tile_kernel(const LossArgs<T> a) {
    using A = Acc<T>;
    constexpr int THREADS = LANES * ROWS, VW = 16 / sizeof(T);
    extern __shared__ uint4 tile_vectors[];
    __shared__ bool labelled_row[ROWS];
    __shared__ double cluster_sum;
    __shared__ int cluster_count;
    if constexpr (!FORWARD) {
        if (a.skip_one && *a.upstream == A(1)) return;
    }
    if constexpr (FORWARD && !CLUSTERED) asm volatile("griddepcontrol.wait;" ::: "memory");
    T *tile = reinterpret_cast<T *>(tile_vectors);
    const int team = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const int classes = (int)a.classes;
    const unsigned mask = team_mask<LANES>();
    int64_t labelled = 0;
    if constexpr (CLUSTERED) {
        namespace cg = cooperative_groups;
        if (a.reduction == CGNN_MEAN) {
            int mine = 0;
            for (int64_t r = (int64_t)blockIdx.x * THREADS + threadIdx.x; r < a.rows; r += CLUSTER * THREADS)
                mine += class_of(a.target[r], a.classes, a.ignore_index, false) >= 0;
            mine = block_sum<THREADS>(mine);
            if (threadIdx.x == 0) cluster_count = mine;
            cg::this_cluster().sync();
            for (int b = 0; b < CLUSTER; ++b) labelled += *cg::this_cluster().map_shared_rank(&cluster_count, b);
        }
    } else if (FORWARD && a.reduction != CGNN_NONE) {
        labelled = labelled_rows<T, THREADS>(a);
    } else if (!FORWARD && a.reduction == CGNN_MEAN) {
        labelled = *a.labelled;
    }
    A share = A(0);
    if (a.grad && (FORWARD || a.reduction != CGNN_NONE)) share = share_of(a, FORWARD ? 1.0 : (double)*a.upstream, labelled);
    double total = 0.0;
    int start = 0;
    if (LANES < 32 && (LANES > 1 || classes % 2 == 0)) start = team % ((classes + LANES - 1) / LANES) * LANES;
    const auto row_of = [&](int e) { return classes == 1 ? e : (int)__umulhi((uint32_t)e, a.per_class); };
    const int64_t tiles = (a.rows + ROWS - 1) / ROWS;
    for (int64_t i = blockIdx.x; i < tiles; i += gridDim.x) {
        const int64_t r0 = i * ROWS, r = r0 + team;
        const int n = (int)min((int64_t)ROWS, a.rows - r0) * classes;  // elements of the tile
        const int64_t label = r < a.rows ? class_of(a.target[r], a.classes, a.ignore_index, FORWARD && lane == 0) : -1;
        const int t = (int)label;
        if (lane == 0) labelled_row[team] = t >= 0;
        __syncthreads();
        if (a.dense) {
            const T *from = a.logits + r0 * a.classes;
            for (int e = threadIdx.x * VW; e < n; e += THREADS * VW) {
                const int last = row_of(min(e + VW, n) - 1);
                bool any = false;
                for (int row = row_of(e); row <= last; ++row) any |= labelled_row[row];
                if (any) copy16(tile + e, from + e, min(16, (n - e) * (int)sizeof(T)));
            }
            copies_done();
        } else {
            for (int e = threadIdx.x; e < n; e += THREADS) {
                const int row = row_of(e);
                if (labelled_row[row]) tile[e] = a.logits[(r0 + row) * a.stride + (e - row * classes)];
            }
        }
        __syncthreads();
        T *z = tile + team * classes;
        if (t >= 0) {
            A m = -(A)INFINITY, inv;
            if constexpr (FORWARD) {
                for_columns<LANES>(classes, lane, start, [&](int c) { m = larger(m, widen(z[c])); });
#pragma unroll
                for (int off = LANES / 2; off > 0; off >>= 1) m = larger(m, __shfl_xor_sync(mask, m, off));
                A s = A(0);
                for_columns<LANES>(classes, lane, start, [&](int c) { s += exponential(widen(z[c]) - m); });
#pragma unroll
                for (int off = LANES / 2; off > 0; off >>= 1) s += __shfl_xor_sync(mask, s, off);
                inv = A(1) / s;
                if (lane == 0) {
                    // (the label's score and the largest one first: both may be large beside their difference)
                    const A loss = logarithm(s) + (m - widen(z[t]));
                    if (a.reduction == CGNN_NONE) a.loss[r] = loss;
                    total += (double)loss;
                    if (a.stats) {
                        a.stats[2 * r] = m;
                        a.stats[2 * r + 1] = inv;
                    }
                }
                __syncwarp(mask);
            } else {
                m = a.stats[2 * r];
                inv = a.stats[2 * r + 1];
                if (a.reduction == CGNN_NONE) share = a.upstream[r];
            }
            if (a.grad)
                for_columns<LANES>(classes, lane, start, [&](int c) { z[c] = narrow<T>(slope<A>(widen(z[c]), m, inv, c == t, share)); });
        } else if (r < a.rows) {
            if (FORWARD && a.reduction == CGNN_NONE && lane == 0) a.loss[r] = A(0);
            if (a.grad) for_columns<LANES>(classes, lane, start, [&](int c) { z[c] = narrow<T>(A(0)); });
        }
        if (!a.grad) continue;
        __syncthreads();
        T *to = a.grad + r0 * a.classes;
        if (a.dense) {
            for (int e = threadIdx.x * VW; e < n; e += THREADS * VW) {
                if (e + VW <= n) vec_store<T, VW>(to + e, vec_load<T, VW>(tile + e));
                else
                    for (int k = e; k < n; ++k) to[k] = tile[k];
            }
        } else {
            for (int e = threadIdx.x; e < n; e += THREADS) to[e] = tile[e];
        }
    }
    if constexpr (FORWARD) {
        if (a.reduction == CGNN_NONE) return;
        if constexpr (CLUSTERED) {
            namespace cg = cooperative_groups;
            total = block_sum<THREADS>(total);
            if (threadIdx.x == 0) cluster_sum = total;
            cg::this_cluster().sync();
            if (blockIdx.x == 0 && threadIdx.x == 0) {
                double s = 0.0;
                for (int b = 0; b < CLUSTER; ++b) s += *cg::this_cluster().map_shared_rank(&cluster_sum, b);
                *a.loss = (A)(a.reduction == CGNN_MEAN ? s / (double)labelled : s);
                *a.labelled = labelled;
            }
            cg::this_cluster().sync();  // a block's shared memory is read until here
        } else {
            finish<T, THREADS>(a, total, labelled);
        }
    }
}

// The 16-byte vectors that cover a row, wherever it begins.  The bytes in front of a row that the first one holds lie in
// the same aligned 16 bytes as the row's own; behind the row nothing is read.
template <typename T>
struct Cover {
    const char *base;
    int shift, vectors, classes;  // elements of the first vector in front of the row; vectors; elements of the row
    __device__ __forceinline__ Cover(const T *row, int64_t classes_)
        : base(reinterpret_cast<const char *>((uintptr_t)row & ~(uintptr_t)15)),
          shift((int)((uintptr_t)row & 15) / (int)sizeof(T)),
          vectors((int)((shift + classes_ + 16 / (int)sizeof(T) - 1) / (16 / (int)sizeof(T)))),
          classes((int)classes_) {}
    __device__ __forceinline__ void copy(uint4 *to, int q) const {
        copy16(to + q, base + (int64_t)q * 16, min(16, (shift + classes) * (int)sizeof(T) - q * 16));
    }
    __device__ __forceinline__ int first(int q) const { return q * (16 / (int)sizeof(T)) - shift; }
};

// Rows of more classes: a block holds one row in shared memory.  A thread copies, reads and writes the same vectors
// throughout, so that only the two sums over the block need barriers, and it fetches the next row's vector as soon as it is
// done with this row's: one row is read while the other is written.
template <typename T, int THREADS, bool FORWARD>
__global__ void __launch_bounds__(THREADS) loss_row_kernel(const LossArgs<T> a) {
    using A = Acc<T>;
    constexpr int VW = 16 / sizeof(T), WARPS = THREADS / 32;
    extern __shared__ uint4 row_vectors[];
    __shared__ A maxima[WARPS], sums[WARPS];
    if constexpr (!FORWARD) {
        if (a.skip_one && *a.upstream == A(1)) return;
    }
    if constexpr (FORWARD) asm volatile("griddepcontrol.wait;" ::: "memory");
    int64_t labelled = 0;
    if (FORWARD && a.reduction != CGNN_NONE) labelled = labelled_rows<T, THREADS>(a);
    if (!FORWARD && a.reduction == CGNN_MEAN) labelled = *a.labelled;
    A share = A(0);
    if (a.grad && (FORWARD || a.reduction != CGNN_NONE)) share = share_of(a, FORWARD ? 1.0 : (double)*a.upstream, labelled);
    double total = 0.0;
    const int classes = (int)a.classes;
    const auto label_of = [&](int64_t r) {
        return r < a.rows ? (int)class_of(a.target[r], a.classes, a.ignore_index, FORWARD && threadIdx.x == 0) : -1;
    };
    int64_t r = blockIdx.x;
    int t = label_of(r);
    A at_label = A(0);
    if (t >= 0) {
        const Cover<T> row(a.logits + r * a.stride, a.classes);
        for (int q = threadIdx.x; q < row.vectors; q += THREADS) row.copy(row_vectors, q);
        if (FORWARD && threadIdx.x == 0) at_label = widen(a.logits[r * a.stride + t]);
    }
    while (r < a.rows) {
        const int64_t next = r + gridDim.x;
        const int t_next = label_of(next);
        const Cover<T> row(a.logits + r * a.stride, a.classes), row_next(a.logits + (t_next >= 0 ? next : r) * a.stride, a.classes);
        A at_next = A(0);
        if (FORWARD && t_next >= 0 && threadIdx.x == 0) at_next = widen(a.logits[next * a.stride + t_next]);
        A m = -(A)INFINITY, inv = A(0);
        if (t >= 0) {
            copies_done();
            if constexpr (FORWARD) {
                for (int q = threadIdx.x; q < row.vectors; q += THREADS) {
                    A v[VW];
                    widen_all<T, VW>(vec_load<T, VW>(reinterpret_cast<const T *>(row_vectors + q)), v);
                    const int e = row.first(q);
                    if (e >= 0 && e + VW <= classes) {
#pragma unroll
                        for (int k = 0; k < VW; ++k) m = larger(m, v[k]);
                    } else {
#pragma unroll
                        for (int k = 0; k < VW; ++k)
                            if ((unsigned)(e + k) < (unsigned)classes) m = larger(m, v[k]);
                    }
                }
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, off));
                if ((threadIdx.x & 31) == 0) maxima[threadIdx.x >> 5] = m;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WARPS; ++w) m = larger(m, maxima[w]);
                A s = A(0);
                for (int q = threadIdx.x; q < row.vectors; q += THREADS) {
                    A v[VW];
                    widen_all<T, VW>(vec_load<T, VW>(reinterpret_cast<const T *>(row_vectors + q)), v);
                    const int e = row.first(q);
                    if (e >= 0 && e + VW <= classes) {
#pragma unroll
                        for (int k = 0; k < VW; ++k) s += exponential(v[k] - m);
                    } else {
#pragma unroll
                        for (int k = 0; k < VW; ++k)
                            if ((unsigned)(e + k) < (unsigned)classes) s += exponential(v[k] - m);
                    }
                }
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
                if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
                __syncthreads();
                s = A(0);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) s += sums[w];
                inv = A(1) / s;
                if (threadIdx.x == 0) {
                    const A loss = logarithm(s) + (m - at_label);
                    if (a.reduction == CGNN_NONE) a.loss[r] = loss;
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
        } else if (FORWARD && a.reduction == CGNN_NONE && threadIdx.x == 0) {
            a.loss[r] = A(0);
        }
        // Out with this row, in with the next: the same vectors by the same thread.
        T *out = a.grad + r * a.classes;
        const bool aligned = ((uintptr_t)out & 15) == (uintptr_t)(row.shift * sizeof(T));
        const int most = max(row.vectors, t_next >= 0 ? row_next.vectors : 0);
        for (int q = threadIdx.x; q < most; q += THREADS) {
            if (a.grad && q < row.vectors) {
                A d[VW];
                const int e = row.first(q);
                if (t >= 0) {
                    A v[VW];
                    widen_all<T, VW>(vec_load<T, VW>(reinterpret_cast<const T *>(row_vectors + q)), v);
#pragma unroll
                    for (int k = 0; k < VW; ++k) d[k] = slope<A>(v[k], m, inv, e + k == t, share);
                } else {
#pragma unroll
                    for (int k = 0; k < VW; ++k) d[k] = A(0);
                }
                const Vec<T, VW> y = narrow_all<T, VW>(d);
                if (aligned && e >= 0 && e + VW <= classes) {
                    vec_store<T, VW>(out + e, y);
                } else {
#pragma unroll
                    for (int k = 0; k < VW; ++k)
                        if ((unsigned)(e + k) < (unsigned)classes) out[e + k] = y.v[k];
                }
            }
            if (t_next >= 0 && q < row_next.vectors) row_next.copy(row_vectors, q);
        }
        r = next;
        t = t_next;
        at_label = at_next;
    }
    if constexpr (FORWARD) {
        if (a.reduction != CGNN_NONE) finish<T, THREADS>(a, total, labelled);
    }
}

// Rows that shared memory does not hold: a block passes over its row again instead (the later times out of L2).
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(LONG_THREADS) loss_long_kernel(const LossArgs<T> a) {
    using A = Acc<T>;
    constexpr int WARPS = LONG_THREADS / 32;
    __shared__ A maxima[WARPS], sums[WARPS];
    if constexpr (!FORWARD) {
        if (a.skip_one && *a.upstream == A(1)) return;
    }
    if constexpr (FORWARD) asm volatile("griddepcontrol.wait;" ::: "memory");
    int64_t labelled = 0;
    if (FORWARD && a.reduction != CGNN_NONE) labelled = labelled_rows<T, LONG_THREADS>(a);
    if (!FORWARD && a.reduction == CGNN_MEAN) labelled = *a.labelled;
    A share = A(0);
    if (a.grad && (FORWARD || a.reduction != CGNN_NONE)) share = share_of(a, FORWARD ? 1.0 : (double)*a.upstream, labelled);
    double total = 0.0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int64_t t = class_of(a.target[r], a.classes, a.ignore_index, FORWARD && threadIdx.x == 0);
        const T *row = a.logits + r * a.stride;
        A m = -(A)INFINITY, inv = A(0);
        if (t >= 0) {
            if constexpr (FORWARD) {
#pragma unroll 8
                for (int64_t c = threadIdx.x; c < a.classes; c += LONG_THREADS) m = larger(m, widen(row[c]));
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, off));
                if ((threadIdx.x & 31) == 0) maxima[threadIdx.x >> 5] = m;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WARPS; ++w) m = larger(m, maxima[w]);
                A s = A(0);
#pragma unroll 8
                for (int64_t c = threadIdx.x; c < a.classes; c += LONG_THREADS) s += exponential(widen(row[c]) - m);
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
                if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
                __syncthreads();
                s = A(0);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) s += sums[w];
                inv = A(1) / s;
                if (threadIdx.x == 0) {
                    const A loss = logarithm(s) + (m - widen(row[t]));
                    if (a.reduction == CGNN_NONE) a.loss[r] = loss;
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
        } else if (FORWARD && a.reduction == CGNN_NONE && threadIdx.x == 0) {
            a.loss[r] = A(0);
        }
        if (!a.grad) continue;
        T *out = a.grad + r * a.classes;
#pragma unroll 8
        for (int64_t c = threadIdx.x; c < a.classes; c += LONG_THREADS)
            out[c] = narrow<T>(t >= 0 ? slope<A>(widen(row[c]), m, inv, c == t, share) : A(0));
    }
    if constexpr (FORWARD) {
        if (a.reduction != CGNN_NONE) finish<T, LONG_THREADS>(a, total, labelled);
    }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
// follows: behind the launch that counts, which it may overlap until it waits; cluster: blocks of one cluster, or 1.
template <typename T>
static int launch(void (*kernel)(const LossArgs<T>), const LossArgs<T> &a, int64_t units, int threads, size_t shared, bool follows,
                  int cluster, cudaStream_t stream) {
    if (shared > 44 * 1024)  // (with the kernels' own variables no more than the 48 KB that need no leave)
        CGNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared));
    const int64_t resident = std::min<int64_t>({16, (int64_t)(SHARED_MOST / (shared + 2048)), 2048 / threads});
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(cluster > 1 ? (unsigned)cluster
                                      : (unsigned)std::max<int64_t>(1, std::min<int64_t>(units, SMS * std::max<int64_t>(1, resident))));
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    if (cluster > 1) {
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = (unsigned)cluster;
        attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    } else {
        attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attribute.val.programmaticStreamSerializationAllowed = 1;
    }
    config.attrs = &attribute;
    config.numAttrs = follows || cluster > 1 ? 1 : 0;
    CGNN_CUDA(cudaLaunchKernelEx(&config, kernel, a));
    return CGNN_OK;
}

template <typename T, int LANES, int ROWS, bool FORWARD>
static int launch_tiles(const LossArgs<T> &a, bool follows, cudaStream_t stream) {
    const size_t shared = (ROWS * a.classes * sizeof(T) + 15) / 16 * 16;
    return launch<T>(loss_tile_kernel<T, LANES, ROWS, FORWARD, false>, a, ceil_div(a.rows, ROWS), LANES * ROWS, shared, follows, 1,
                     stream);
}

template <typename T, bool FORWARD>
static int launch_rows(const LossArgs<T> &a, bool follows, cudaStream_t stream) {
    if (a.classes <= 64) return launch_tiles<T, 1, 128, FORWARD>(a, follows, stream);
    if (a.classes <= 256) return launch_tiles<T, 4, 32, FORWARD>(a, follows, stream);
    if (a.classes <= 1024) return launch_tiles<T, 32, 8, FORWARD>(a, follows, stream);
    const size_t shared = (a.classes * sizeof(T) + 15) / 16 * 16 + 16;
    if (shared <= 32 * 1024) return launch<T>(loss_row_kernel<T, 256, FORWARD>, a, a.rows, 256, shared, follows, 1, stream);
    if (shared <= SHARED_MOST / 2 - 2048) return launch<T>(loss_row_kernel<T, 512, FORWARD>, a, a.rows, 512, shared, follows, 1, stream);
    if (shared <= SHARED_MOST - 2048) return launch<T>(loss_row_kernel<T, 1024, FORWARD>, a, a.rows, 1024, shared, follows, 1, stream);
    return launch<T>(loss_long_kernel<T, FORWARD>, a, a.rows, LONG_THREADS, 0, follows, 1, stream);
}

// One launch where a cluster does it all, else one that counts and one that computes.
template <typename T>
static int forward(LossArgs<T> a, cudaStream_t stream) {
    if (a.reduction == CGNN_NONE) return a.rows ? launch_rows<T, true>(a, false, stream) : CGNN_OK;
    if (a.rows <= CLUSTER_ROWS && a.classes <= 64)
        return launch<T>(loss_tile_kernel<T, 1, 128, true, true>, a, CLUSTER, 128, (128 * a.classes * sizeof(T) + 15) / 16 * 16, false,
                         CLUSTER, stream);
    a.count_blocks = a.reduction == CGNN_MEAN ? (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(a.rows, COUNT_THREADS), SMS)) : 1;
    loss_count_kernel<<<(unsigned)a.count_blocks, COUNT_THREADS, 0, stream>>>(
        a.target, a.reduction == CGNN_MEAN ? a.rows : 0, a.classes, a.ignore_index, a.scratch);
    CGNN_LAUNCH_CHECK();
    return launch_rows<T, true>(a, true, stream);
}

template <typename T>
static LossArgs<T> args_of(int64_t rows, int64_t classes, int64_t stride, const void *logits, const int64_t *target,
                           int64_t ignore_index, int reduction, void *grad) {
    LossArgs<T> a{};
    a.logits = (const T *)logits;
    a.rows = rows;
    a.classes = classes;
    a.stride = stride;
    a.target = target;
    a.ignore_index = ignore_index;
    a.reduction = reduction;
    a.grad = (T *)grad;
    a.dense = (stride == classes || rows == 1) && (((uintptr_t)logits | (uintptr_t)grad) & 15) == 0;
    a.per_class = (uint32_t)(((uint64_t)1 << 32) / (uint64_t)classes + 1);
    return a;
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

size_t cgnn_cross_entropy_scratch_bytes(void) { return sizeof(LossScratch); }

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
    const auto run = [&](auto zero) -> int {
        using T = decltype(zero);
        LossArgs<T> a = args_of<T>(rows, classes, stride, logits, target, ignore_index, reduction, grad);
        a.labelled = labelled;
        a.stats = (Acc<T> *)stats;
        a.loss = (Acc<T> *)loss;
        a.scratch = (LossScratch *)scratch;
        return forward<T>(a, stream);
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
        LossArgs<T> a = args_of<T>(rows, classes, stride, logits, target, ignore_index, reduction, grad);
        a.labelled = const_cast<int64_t *>(labelled);
        a.stats = (Acc<T> *)const_cast<void *>(stats);
        a.upstream = (const Acc<T> *)upstream;
        a.skip_one = reduction != CGNN_NONE && holds_unit_gradient;
        return launch_rows<T, false>(a, false, (cudaStream_t)stream);
    };
    switch (dtype) {
        case CGNN_F32: return run(0.0f);
        case CGNN_F64: return run(0.0);
        case CGNN_BF16: return run(__nv_bfloat16());
        default: return run(__half());
    }
}

}  // extern "C"
