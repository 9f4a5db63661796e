// Softmax cross entropy of class scores over the labelled nodes, with the gradient of the scores.
//
// Row i with label t:  loss_i = lse(z_i) - z_i[t],  dz_i = (softmax(z_i) - onehot(t)) * share_i.  A row whose label is
// `ignore_index` has no loss and a gradient of zeros, whatever its scores are; a label that is no class is treated
// the same and sets a status bit.  share_i is the incoming gradient, for a mean over the number of labelled rows.
//
// Memory bounds it.  For a sum or a mean the forward pass writes the gradient for an incoming gradient of one beside the
// loss, from the copy of the row it holds anyway: the scores are read once a step, not twice.  Losses are added up in
// fp64 and in a fixed order.
#include <algorithm>
#include <atomic>
#include <type_traits>

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
constexpr size_t SHARED_MOST = 227 * 1024;  // of a block
constexpr size_t DYNAMIC_MOST = SHARED_MOST - 2048;  // of it beside the kernels' own variables
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
    int clustered;         // forward with reduction: the launch is one cluster, which counts and adds up itself
    T *grad;               // optional in the forward pass
    const A *upstream;     // backward: one value, or one per row without reduction
    int skip_one;          // backward: `grad` holds the gradient for an incoming one already
    int dense;             // rows lie one behind the other from a 16-byte boundary on, in the scores and the gradient
    int whole_tiles;       // dense and narrow: a tile comes in one copy, unlabelled rows and all
    int polls;             // after which a copy is given up
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

constexpr float LOG2_E = 1.4426950408889634f;
// By the special function unit; what lies below the normal numbers is zero.
__device__ __forceinline__ float power_of_two(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// e^x for x <= 0.
__device__ __forceinline__ float exponential(float x) { return power_of_two(x * LOG2_E); }
__device__ __forceinline__ double exponential(double x) { return exp(x); }
__device__ __forceinline__ float logarithm(float x) { return logf(x); }
__device__ __forceinline__ double logarithm(double x) { return log(x); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

// The gradient of a score from its exponential, the same arithmetic in every kernel: scale = inv * share.
template <typename A>
__device__ __forceinline__ A slope(A e, A scale) { return e * scale; }
template <typename A>
__device__ __forceinline__ A slope_at_label(A e, A scale, A share) { return fused(e, scale, -share); }

// The same of two scores at once: fp32 has instructions for pairs.
__device__ __forceinline__ void exponentials(float &a, float &b, float m) {
    const float2 d = __fadd2_rn(make_float2(a, b), make_float2(-m, -m));
    const float2 e = __fmul2_rn(d, make_float2(LOG2_E, LOG2_E));
    a = power_of_two(e.x);
    b = power_of_two(e.y);
}
__device__ __forceinline__ void exponentials(double &a, double &b, double m) {
    a = exponential(a - m);
    b = exponential(b - m);
}
__device__ __forceinline__ void add_pair(float (&s)[2], float a, float b) {
    const float2 two = __fadd2_rn(make_float2(s[0], s[1]), make_float2(a, b));
    s[0] = two.x;
    s[1] = two.y;
}
__device__ __forceinline__ void add_pair(double (&s)[2], double a, double b) {
    s[0] += a;
    s[1] += b;
}
__device__ __forceinline__ void slopes(float &a, float &b, float scale) {
    const float2 two = __fmul2_rn(make_float2(a, b), make_float2(scale, scale));
    a = two.x;
    b = two.y;
}
__device__ __forceinline__ void slopes(double &a, double &b, double scale) {
    a = slope(a, scale);
    b = slope(b, scale);
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
// Bulk copies (whole 16-byte vectors) report to a barrier in shared memory, for which threads wait with a limit of polls.
constexpr int WAIT_LIMIT = 1 << 20;
__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(uint64_t *barrier, int arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(barrier)), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t *barrier, uint32_t bytes) {  // and arrive
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(barrier)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_copy(void *shared, const void *global, uint32_t bytes, uint64_t *barrier) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(shared_address(shared)),
                 "l"(global), "r"(bytes), "r"(shared_address(barrier))
                 : "memory");
}
__device__ __forceinline__ bool barrier_wait(uint64_t *barrier, uint32_t parity, int polls) {
    for (int i = 0; i < polls; ++i) {
        uint32_t done;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done)
                     : "r"(shared_address(barrier)), "r"(parity)
                     : "memory");
        if (done) return true;
    }
    return false;
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

// The number of labelled rows, on every thread of a block: from the launch before, or counted by the cluster that the
// launch is.
template <typename T, int THREADS>
__device__ __forceinline__ int64_t labelled_rows(const LossArgs<T> &a) {
    namespace cg = cooperative_groups;
    __shared__ int64_t all;
    if (a.reduction != CGNN_MEAN) return 0;
    int64_t mine = 0;
    if (a.clustered) {
        for (int64_t r = (int64_t)blockIdx.x * THREADS + threadIdx.x; r < a.rows; r += CLUSTER * THREADS)
            mine += class_of(a.target[r], a.classes, a.ignore_index, false) >= 0;
    } else {
        for (int b = threadIdx.x; b < a.count_blocks; b += THREADS) mine += a.scratch->counts[b];
    }
    mine = block_sum<THREADS>(mine);
    if (threadIdx.x == 0) all = mine;
    if (!a.clustered) {
        __syncthreads();
        return all;
    }
    cg::this_cluster().sync();
    mine = 0;
    for (int b = 0; b < CLUSTER; ++b) mine += *cg::this_cluster().map_shared_rank(&all, b);
    return mine;
}

// The end of a reduced loss: a block leaves its sum, and the last one to do so adds all of them up in block order; the
// blocks of a cluster leave them in their shared memory.
template <typename T, int THREADS>
__device__ __forceinline__ void finish(const LossArgs<T> &a, double total, int64_t labelled) {
    namespace cg = cooperative_groups;
    __shared__ bool last;
    __shared__ double here;
    total = block_sum<THREADS>(total);
    if (a.clustered) {
        if (threadIdx.x == 0) here = total;
        cg::this_cluster().sync();
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            double s = 0.0;
            for (int b = 0; b < CLUSTER; ++b) s += *cg::this_cluster().map_shared_rank(&here, b);
            *a.loss = (Acc<T>)(a.reduction == CGNN_MEAN ? s / (double)labelled : s);
            *a.labelled = labelled;
        }
        cg::this_cluster().sync();  // a block's shared memory is read until here
        return;
    }
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

// Rows of up to 768 classes.  A block copies ROWS whole rows into shared memory as the 16-byte vectors they lie in, in
// whatever way rows and vectors meet (47 classes: 188 bytes a row): one bulk copy for each labelled row, while the tile
// before is worked on.  LANES lanes then hold a row in registers, lane l the columns l, l + LANES, ...; the gradient takes
// the row's place in shared memory and leaves by whole vectors.
// What bounds it is instructions and their latency more than memory: 2.45 M x 47 in fp32 with 0.6 of the rows
// labelled takes 170 us (DRAM 782 MB, 120 us); a lane group of 16 over registers loaded from DRAM took 375, three passes
// over shared memory 301, one tile at a time 237.  Columns a lane, registers and time were tried together: 48 in 102 registers
// 170, 48 in 85 181, 24 in 64 172 to 179, 24 in 80 176, 32 in 80 177, 32 in 64 193, 16 in 51 259.
// AROUND: the lanes of a warp begin at different columns and go around, or rows of an even length would meet in the
// same banks.
constexpr int HELD = 24;  // columns of a lane, or twice as many
template <typename T, int THREADS, int COLUMNS>
constexpr int TILE_BLOCKS = (COLUMNS > HELD ? (sizeof(T) == 8 ? 256 : 640) : sizeof(T) == 8 ? 384 : 1024) / THREADS;  // to a
// multiprocessor, by their registers
template <typename T, int LANES, int ROWS, int COLUMNS, bool AROUND, bool FORWARD>
__global__ void __launch_bounds__(LANES *ROWS, TILE_BLOCKS<T, LANES * ROWS, COLUMNS>) loss_tile_kernel(const LossArgs<T> a) {
    using A = Acc<T>;
    constexpr int THREADS = LANES * ROWS, VW = 16 / sizeof(T);
    extern __shared__ uint4 tile_vectors[];
    __shared__ uint64_t arrived[2];
    if constexpr (!FORWARD) {
        if (a.skip_one && *a.upstream == A(1)) return;
    }
    if constexpr (FORWARD) asm volatile("griddepcontrol.wait;" ::: "memory");
    T *tile = reinterpret_cast<T *>(tile_vectors);
    const int team = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const int classes = (int)a.classes, held = (classes + LANES - 1) / LANES;
    const unsigned mask = team_mask<LANES>();
    int64_t labelled = 0;
    if (FORWARD && a.reduction != CGNN_NONE) labelled = labelled_rows<T, THREADS>(a);
    if (!FORWARD && a.reduction == CGNN_MEAN) labelled = *a.labelled;
    A share = A(0);
    if (a.grad && (FORWARD || a.reduction != CGNN_NONE)) share = share_of(a, FORWARD ? 1.0 : (double)*a.upstream, labelled);
    double total = 0.0;
    // Register j of a lane has the column `lane + LANES * ((j + turn) % held)`, where there is one.
    const int turn = AROUND ? team % held : 0, wrap = held - turn;
    const int missing = lane + LANES * (held - 1) < classes ? -1 : (AROUND ? wrap - 1 : held - 1);
    // (`phase` keeps the compiler from holding the addresses of one pass for the next: they do not fit the registers)
    struct Columns {
        int begin, again, wrap;
        __device__ __forceinline__ int operator()(int j) const { return (AROUND && j >= wrap ? again : begin) + LANES * j; }
    };
    const auto phase = [&] {
        Columns c{lane + LANES * turn, lane - LANES * wrap, wrap};
        if (AROUND) asm volatile("" : "+r"(c.begin), "+r"(c.again), "+r"(c.wrap));
        return c;
    };
    const auto there_is = [&](int j, int count) { return j < count && j != missing; };
    const int tiles = (int)((a.rows + ROWS - 1) / ROWS);  // (below 2^31: the rows of more do not fit any memory)
    // The team's row: the vectors that cover it, in one copy; one that it shares with the next row both may bring.  (The
    // very last row may end inside a vector: its last elements are loaded one by one.)
    const int first = team * classes / VW * VW, behind = (team + 1) * classes, last = (behind + VW - 1) / VW * VW;
    const auto copy = [&](int i, bool wanted, int place, T *to) {
        if (!a.dense) {
            const T *from = a.logits + ((int64_t)i * ROWS + team) * a.stride;
            if (wanted)
                for (int c = lane; c < classes; c += LANES) to[team * classes + c] = from[c];
        } else if (a.whole_tiles) {
            const T *from = a.logits + (int64_t)i * (ROWS * classes);
            const int n = i < tiles - 1 ? ROWS * classes : (int)(a.rows - (int64_t)i * ROWS) * classes, whole = n / VW * VW;
            if (threadIdx.x == 0) {
                barrier_expect(&arrived[place], (uint32_t)(whole * sizeof(T)));
                if (whole) bulk_copy(to, from, (uint32_t)(whole * sizeof(T)), &arrived[place]);
            }
            if (whole + (int)threadIdx.x < n) to[whole + threadIdx.x] = from[whole + threadIdx.x];
        } else if (lane == 0) {
            const T *from = a.logits + (int64_t)i * (ROWS * classes);
            int end = last;
            if (i == tiles - 1) end = min(last, (int)(a.rows - (int64_t)i * ROWS) * classes / VW * VW);
            const uint32_t bytes = wanted && end > first ? (uint32_t)((end - first) * sizeof(T)) : 0u;
            barrier_expect(&arrived[place], bytes);
            if (bytes) bulk_copy(to + first, from + first, bytes, &arrived[place]);
            if (wanted)
                for (int e = max(end, first); e < behind; ++e) to[e] = from[e];
        }
    };
    const auto label_of = [&](int i) {  // of the team's row of a tile
        const int64_t r = (int64_t)i * ROWS + team;
        return i < tiles && r < a.rows ? a.target[r] : a.ignore_index;
    };
    const auto class_or_none = [&](int64_t label) { return (int)class_of(label, a.classes, a.ignore_index, FORWARD && lane == 0); };
    if (threadIdx.x == 0) {
        barrier_init(&arrived[0], a.whole_tiles ? 1 : ROWS);
        barrier_init(&arrived[1], a.whole_tiles ? 1 : ROWS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // While one tile is worked on the next one arrives, and the labels of the one after it.
    T *here = tile, *there = tile + (ROWS * classes + VW - 1) / VW * VW;
    int t = class_or_none(label_of(blockIdx.x)), round = 0;
    int64_t label_next = label_of(blockIdx.x + gridDim.x);
    if ((int)blockIdx.x < tiles) copy(blockIdx.x, t >= 0, 0, here);
    int i = blockIdx.x;
    bool late = false;
    for (; i < tiles; i += gridDim.x, ++round) {
        // (ordinary accesses to the other tile's place come before the copy into it)
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        late = a.dense && !barrier_wait(&arrived[round & 1], (uint32_t)(round >> 1) & 1u, a.polls);
        late = __syncthreads_or(late);  // the tile is here, and the one before it has left; or a copy did not arrive
        if (late) break;
        const int t_next = class_or_none(label_next);
        if (i + (int)gridDim.x < tiles) copy(i + gridDim.x, t_next >= 0, (round & 1) ^ 1, there);
        label_next = label_of(i + 2 * gridDim.x);
        const int64_t r = (int64_t)i * ROWS + team;
        const bool inside = i < tiles - 1 || r < a.rows;
        T *const z = here + team * classes;
        // A row without a label passes as one of scores of minus infinity with a share of zero.
        const int read = t >= 0 ? held : 0, written = inside ? held : 0;
        const Columns column = phase();
        A v[COLUMNS], m = -(A)INFINITY, other = m, inv = A(0), at_label = A(0);
        if (t >= 0) at_label = widen(z[t]);
#pragma unroll
        for (int j = 0; j < COLUMNS; j += 8) {
            if (j >= held) break;
#pragma unroll
            for (int k = j; k < j + 8; ++k) {
                v[k] = -(A)INFINITY;
                if (there_is(k, read)) v[k] = widen(z[column(k)]);
                if (FORWARD) (k & 1 ? other : m) = larger(k & 1 ? other : m, v[k]);
            }
        }
        if constexpr (FORWARD) {
            m = larger(m, other);
#pragma unroll
            for (int off = LANES / 2; off > 0; off >>= 1) m = larger(m, __shfl_xor_sync(mask, m, off));
        } else if (t >= 0) {
            m = a.stats[2 * r];
            inv = a.stats[2 * r + 1];
            if (a.reduction == CGNN_NONE) share = a.upstream[r];
        }
        if (t < 0) m = A(0);
        A parts[2] = {A(0), A(0)};
#pragma unroll
        for (int j = 0; j < COLUMNS; j += 8) {
            if (j >= held) break;
#pragma unroll
            for (int k = j; k < j + 8; k += 2) {
                exponentials(v[k], v[k + 1], m);
                if (FORWARD) add_pair(parts, v[k], v[k + 1]);
            }
        }
        A s = parts[0] + parts[1];
        if constexpr (FORWARD) {
#pragma unroll
            for (int off = LANES / 2; off > 0; off >>= 1) s += __shfl_xor_sync(mask, s, off);
            inv = A(1) / s;
            if (lane == 0 && inside) {
                // (the label's score and the largest one first: both may be large beside their difference)
                const A loss = t >= 0 ? logarithm(s) + (m - at_label) : A(0);
                if (a.reduction == CGNN_NONE) a.loss[r] = loss;
                total += (double)loss;
                if (a.stats) vec_store<A, 2>(a.stats + 2 * r, Vec<A, 2>{{m, inv}});
            }
        }
        T *const now = here;
        here = there;
        there = now;
        if (a.grad) {
            const A scale = t >= 0 ? inv * share : A(0);
            __syncwarp(mask);  // every lane has read its label's score ...
            const Columns column = phase();
#pragma unroll
            for (int j = 0; j < COLUMNS; j += 8) {
                if (j >= held) break;
#pragma unroll
                for (int k = j; k < j + 8; k += 2) {
                    slopes(v[k], v[k + 1], scale);
                    if (there_is(k, written)) z[column(k)] = narrow<T>(v[k]);
                    if (there_is(k + 1, written)) z[column(k + 1)] = narrow<T>(v[k + 1]);
                }
            }
            __syncwarp(mask);  // ... and written its columns
            if (lane == 0 && t >= 0) z[t] = narrow<T>(slope_at_label(exponential(at_label - m), scale, share));
            __syncthreads();
            T *const to = a.grad + (int64_t)i * (ROWS * classes);
            const int n = i < tiles - 1 ? ROWS * classes : (int)(a.rows - (int64_t)i * ROWS) * classes;
            if (a.dense) {
                const int whole = n / VW * VW;
#pragma unroll 4
                for (int e = threadIdx.x * VW; e < whole; e += THREADS * VW) vec_store<T, VW>(to + e, vec_load<T, VW>(now + e));
                if (whole + (int)threadIdx.x < n) to[whole + threadIdx.x] = now[whole + threadIdx.x];
            } else {
                for (int e = threadIdx.x; e < n; e += THREADS) to[e] = now[e];
            }
        }
        t = t_next;
    }
    if (late) {
        // What was not computed is NaN, and the block takes part in the sum like the others, which wait for it.  Its copy
        // comes to its end before the memory is another block's.
        if (threadIdx.x == 0) atomicOr(&g_loss_status, STATUS_WAIT_EXPIRED);
        barrier_wait(&arrived[round & 1], (uint32_t)(round >> 1) & 1u, WAIT_LIMIT);
        const A none = (A)NAN;
        total = NAN;
        for (; i < tiles; i += gridDim.x) {
            const int64_t r = (int64_t)i * ROWS + team;
            if (FORWARD && lane == 0 && r < a.rows) {
                if (a.reduction == CGNN_NONE) a.loss[r] = none;
                if (a.stats) vec_store<A, 2>(a.stats + 2 * r, Vec<A, 2>{{none, none}});
            }
            const int n = i < tiles - 1 ? ROWS * classes : (int)(a.rows - (int64_t)i * ROWS) * classes;
            if (a.grad)
                for (int e = threadIdx.x; e < n; e += THREADS) a.grad[(int64_t)i * (ROWS * classes) + e] = narrow<T>(none);
        }
    }
    if constexpr (FORWARD) {
        if (a.reduction != CGNN_NONE) finish<T, THREADS>(a, total, labelled);
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
    // Elements of a copied vector that are not the row's become minus infinity.
    __device__ __forceinline__ void clear(uint4 *in, int q) const {
        T *v = reinterpret_cast<T *>(in + q);
        for (int k = 0; k < 16 / (int)sizeof(T); ++k)
            if ((unsigned)(first(q) + k) >= (unsigned)classes) v[k] = narrow<T>(-(Acc<T>)INFINITY);
    }
};

// NaN where either is.
__device__ __forceinline__ float larger_or_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ double larger_or_nan(double a, double b) { return a != a || a > b ? a : b; }

// The largest element of a vector, NaN where it holds one (pairs of 16-bit ones are compared as they are).
template <typename T, int VW>
__device__ __forceinline__ Acc<T> largest(const Vec<T, VW> &x) {
    if constexpr (__is_same(T, __nv_bfloat16)) {
        const __nv_bfloat162 *pairs = reinterpret_cast<const __nv_bfloat162 *>(&x);
        const __nv_bfloat162 two = __hmax2_nan(__hmax2_nan(pairs[0], pairs[1]), __hmax2_nan(pairs[2], pairs[3]));
        return larger_or_nan(__low2float(two), __high2float(two));
    } else if constexpr (__is_same(T, __half)) {
        const __half2 *pairs = reinterpret_cast<const __half2 *>(&x);
        const __half2 two = __hmax2_nan(__hmax2_nan(pairs[0], pairs[1]), __hmax2_nan(pairs[2], pairs[3]));
        return larger_or_nan(__low2float(two), __high2float(two));
    } else {
        Acc<T> m = widen(x.v[0]);
#pragma unroll
        for (int k = 1; k < VW; ++k) m = larger_or_nan(m, widen(x.v[k]));
        return m;
    }
}

// e^(x - m) of fp32 sums as 2^(x * log2(e) - c), c = m * log2(e) rounded: one instruction before the special function.  All
// exponentials of one m are off by the same factor of 2^(m * log2(e) - c), which is divided out of their sum and of the scale
// they are multiplied by; a sum goes over to another m by the difference of the two rounded c's, and then has that one's
// factor.  The factor stays near one for |m| below 2^20; other rows subtract first.
__device__ __forceinline__ float from_offset(float m) { return power_of_two(fmaf(-m, LOG2_E, m * LOG2_E)); }  // 1 / that factor
template <typename A>
__device__ __forceinline__ bool is_steep(A m) {
    return sizeof(A) == 8 || !(m < A(1048576) && m > A(-1048576));
}

// A row's largest score and 1 / sum e^(x - it), on every thread of the block.  vector(q) is vector q of the row's cover,
// with minus infinity where it is not the row.  `turn` counts the calls: two sets of places in turn, so that one
// barrier is enough.
template <typename T, int THREADS, int BATCH, typename Vectors>
__device__ __forceinline__ void row_statistics(Vectors &&vector, int vectors, int &turn, Acc<T> &m, Acc<T> &s) {
    using A = Acc<T>;
    constexpr int VW = 16 / sizeof(T), WARPS = THREADS / 32;
    __shared__ A tops_of[2][WARPS], parts_of[2][WARPS];
    A *const tops = tops_of[turn & 1], *const parts = parts_of[turn & 1];
    ++turn;
    m = -(A)INFINITY;
    s = A(0);
    bool steep = sizeof(A) == 8;
    if constexpr (sizeof(A) == 4) {
        // One pass with a running maximum of the thread, a batch of vectors at a time.
        float2 two = make_float2(0.0f, 0.0f);
        float offset = -INFINITY;  // m * log2(e), rounded
        for (int q = threadIdx.x; q < vectors; q += BATCH * THREADS) {
            Vec<T, VW> x[BATCH];
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < BATCH; ++b) x[b] = vector(q + b * THREADS < vectors ? q + b * THREADS : q);  // a thread's own
#pragma unroll
            for (int b = 0; b < BATCH; ++b) top = larger_or_nan(top, largest<T, VW>(x[b]));
            if (top == -INFINITY) continue;  // (nothing to add)
            steep |= is_steep(top);          // (so is a NaN: the passes below carry it into the sum)
            if (top > m) {
                const float raised = __fmul_rn(top, LOG2_E), down = power_of_two(offset - raised);
                two.x *= down;
                two.y *= down;
                m = top;
                offset = raised;
            }
            const float2 base = make_float2(LOG2_E, LOG2_E), c = make_float2(-offset, -offset);
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                if (q + b * THREADS >= vectors) break;
                float v[VW];
                widen_all<T, VW>(x[b], v);
#pragma unroll
                for (int k = 0; k < VW; k += 2) {
                    const float2 e = __ffma2_rn(make_float2(v[k], v[k + 1]), base, c);  // (two of them in one instruction)
                    two = __fadd2_rn(make_float2(power_of_two(e.x), power_of_two(e.y)), two);
                }
            }
        }
        s = two.x + two.y;
    }
    // The threads' sums meet under the largest maximum; they are not used where a maximum is too large for them.
    const A mine = m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, off));
    if constexpr (sizeof(A) == 4)
        if (mine > -INFINITY) s *= from_offset(mine) * exponential(mine - m);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if ((threadIdx.x & 31) == 0) {
        tops[threadIdx.x >> 5] = m;
        parts[threadIdx.x >> 5] = s;
    }
    if (!__syncthreads_or(steep)) {
        m = tops[0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) m = larger(m, tops[w]);
        s = A(0);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const A part = parts[w];  // (a warp without a score has none, and minus infinity for a maximum)
            s += part == A(0) ? part : part * exponential(tops[w] - m);
        }
        return;
    }
    m = -(A)INFINITY;
    for (int q = threadIdx.x; q < vectors; q += THREADS) m = larger(m, largest<T, VW>(vector(q)));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, off));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = larger(m, tops[w]);
    s = A(0);
    for (int q = threadIdx.x; q < vectors; q += THREADS) {
        A v[VW];
        widen_all<T, VW>(vector(q), v);
#pragma unroll
        for (int k = 0; k < VW; ++k) s += exponential(v[k] - m);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = s;
    __syncthreads();
    s = A(0);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += parts[w];
}

// The gradient of a vector of scores: e^(x - m) * scale, the label apart.
template <typename T, bool STEEP>
struct VectorSlope {
    using A = Acc<T>;
    static constexpr int VW = 16 / sizeof(T);
    A m, scale, c;
    __device__ __forceinline__ VectorSlope(A m_, A inv, A share) : m(m_), scale(inv * share), c(A(0)) {
        if constexpr (!STEEP) {
            scale *= from_offset(m);
            c = m * LOG2_E;
        }
    }
    __device__ __forceinline__ Vec<T, VW> operator()(const Vec<T, VW> &x) const {
        A v[VW];
        widen_all<T, VW>(x, v);
        if constexpr (STEEP) {
#pragma unroll
            for (int k = 0; k < VW; ++k) v[k] = slope(exponential(v[k] - m), scale);
        } else {
#pragma unroll
            for (int k = 0; k < VW; k += 2) {
                const float2 e = __ffma2_rn(make_float2(v[k], v[k + 1]), make_float2(LOG2_E, LOG2_E), make_float2(-c, -c));
                const float2 d = __fmul2_rn(make_float2(power_of_two(e.x), power_of_two(e.y)), make_float2(scale, scale));
                v[k] = d.x;
                v[k + 1] = d.y;
            }
        }
        return narrow_all<T, VW>(v);
    }
    __device__ __forceinline__ T at_label(A x, A share) const {
        if constexpr (STEEP) return narrow<T>(slope_at_label(exponential(x - m), scale, share));
        else return narrow<T>(slope_at_label(power_of_two(fmaf(x, LOG2_E, -c)), scale, share));
    }
};
template <typename T, typename F>
__device__ __forceinline__ void with_slope(Acc<T> m, Acc<T> inv, Acc<T> share, F &&f) {
    if constexpr (sizeof(T) == 8) {
        f(VectorSlope<T, true>(m, inv, share));
    } else {
        if (is_steep(m)) f(VectorSlope<T, true>(m, inv, share));
        else f(VectorSlope<T, false>(m, inv, share));
    }
}

// A vector of the gradient to where it belongs, element by element where it is not whole.
template <typename T>
__device__ __forceinline__ void store_vector(T *out, int first, int classes, bool aligned, const Vec<T, 16 / sizeof(T)> &y) {
    constexpr int VW = 16 / sizeof(T);
    if (aligned && first >= 0 && first + VW <= classes) {
        vec_store<T, VW>(out + first, y);
    } else {
#pragma unroll
        for (int k = 0; k < VW; ++k)
            if ((unsigned)(first + k) < (unsigned)classes) out[first + k] = y.v[k];
    }
}

// Rows of more classes: a block holds one row in shared memory.  A thread copies, reads and writes the same vectors
// throughout, so that only the sums over the block need a barrier, and it fetches the next row's vector as soon as it is
// done with this row's: one row is read while the other is written.  8192 x 50001 in bf16, 0.9 of the rows labelled: 327 us
// (1.56 GB, 238 us at the copy rate); the special function unit is 55 % busy, issue slots 53 %, DRAM 46 %.
template <typename T, int THREADS, bool FORWARD>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) loss_row_kernel(const LossArgs<T> a) {
    using A = Acc<T>;
    constexpr int VW = 16 / sizeof(T);
    extern __shared__ uint4 row_vectors[];
    if constexpr (!FORWARD) {
        if (a.skip_one && *a.upstream == A(1)) return;
    }
    if constexpr (FORWARD) asm volatile("griddepcontrol.wait;" ::: "memory");
    int turn = 0;
    int64_t labelled = 0;
    if (FORWARD && a.reduction != CGNN_NONE) labelled = labelled_rows<T, THREADS>(a);
    if (!FORWARD && a.reduction == CGNN_MEAN) labelled = *a.labelled;
    A share = A(0);
    if (a.grad && (FORWARD || a.reduction != CGNN_NONE)) share = share_of(a, FORWARD ? 1.0 : (double)*a.upstream, labelled);
    double total = 0.0;
    const int classes = (int)a.classes;
    const auto vector = [&](int q) { return vec_load<T, VW>(reinterpret_cast<const T *>(row_vectors + q)); };
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
        A m = A(0), inv = A(0);
        if (t >= 0) {
            copies_done();
            if constexpr (FORWARD) {
                // what the first and the last vector hold beside the row counts for nothing
                if (threadIdx.x == 0) row.clear(row_vectors, 0);
                if ((row.vectors - 1) % THREADS == (int)threadIdx.x) row.clear(row_vectors, row.vectors - 1);
                A s;
                row_statistics<T, THREADS, 2>(vector, row.vectors, turn, m, s);
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
        const int leaving = a.grad ? row.vectors : 0, entering = t_next >= 0 ? row_next.vectors : 0;
        with_slope<T>(m, inv, share, [&](auto slopes) {
            const auto pass = [&](int q) {  // any vector
                if (q < leaving) store_vector<T>(out, row.first(q), classes, aligned, t >= 0 ? slopes(vector(q)) : vec_zero<T, VW>());
                if (q < entering) row_next.copy(row_vectors, q);
            };
            // The label's element is written again below by the thread that has its vector.
            const bool mine = t >= 0 && a.grad && (row.shift + t) / VW % THREADS == (int)threadIdx.x;
            T label_slope = narrow<T>(A(0));
            if (mine) label_slope = slopes.at_label(widen(reinterpret_cast<const T *>(row_vectors)[row.shift + t]), share);
            int q = threadIdx.x;
            if (t >= 0 && aligned && leaving && entering) {  // whole vectors on both sides, the usual case
                if (q == 0) {
                    pass(0);
                    q = THREADS;
                }
                const int inner = min(leaving, entering) - 1;
                T *to = out + row.first(0);
                const char *from = row_next.base;
#pragma unroll 2
                for (; q < inner; q += THREADS) {
                    vec_store<T, VW>(to + q * VW, slopes(vector(q)));
                    copy16(row_vectors + q, from + q * 16, 16);
                }
            }
            for (; q < max(leaving, entering); q += THREADS) pass(q);
            if (mine) out[t] = label_slope;
        });
        r = next;
        t = t_next;
        at_label = at_next;
    }
    if constexpr (FORWARD) {
        if (a.reduction != CGNN_NONE) finish<T, THREADS>(a, total, labelled);
    }
}

// Rows that shared memory does not hold: read a second time for the gradient, out of L2.  (8192 x 50001 in bf16, which
// it holds: 441 us this way, 333 with the row kept, timed in turn.)
template <typename T, bool FORWARD>
__global__ void __launch_bounds__(LONG_THREADS, sizeof(T) == 8 ? 1 : 2) loss_long_kernel(const LossArgs<T> a) {
    using A = Acc<T>;
    constexpr int VW = 16 / sizeof(T), BATCH = 4;
    if constexpr (!FORWARD) {
        if (a.skip_one && *a.upstream == A(1)) return;
    }
    if constexpr (FORWARD) asm volatile("griddepcontrol.wait;" ::: "memory");
    int turn = 0;
    int64_t labelled = 0;
    if (FORWARD && a.reduction != CGNN_NONE) labelled = labelled_rows<T, LONG_THREADS>(a);
    if (!FORWARD && a.reduction == CGNN_MEAN) labelled = *a.labelled;
    A share = A(0);
    if (a.grad && (FORWARD || a.reduction != CGNN_NONE)) share = share_of(a, FORWARD ? 1.0 : (double)*a.upstream, labelled);
    double total = 0.0;
    const int classes = (int)a.classes;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int t = (int)class_of(a.target[r], a.classes, a.ignore_index, FORWARD && threadIdx.x == 0);
        const T *scores = a.logits + r * a.stride;
        const Cover<T> row(scores, a.classes);
        const auto vector = [&](int q) {
            const int e = row.first(q);
            if (e >= 0 && e + VW <= classes) return vec_load<T, VW>(reinterpret_cast<const T *>(row.base + (int64_t)q * 16));
            Vec<T, VW> x;
#pragma unroll
            for (int k = 0; k < VW; ++k)
                x.v[k] = (unsigned)(e + k) < (unsigned)classes ? scores[e + k] : narrow<T>(-(A)INFINITY);
            return x;
        };
        A m = A(0), inv = A(0);
        if (t >= 0) {
            if constexpr (FORWARD) {
                A s;
                row_statistics<T, LONG_THREADS, BATCH>(vector, row.vectors, turn, m, s);
                inv = A(1) / s;
                if (threadIdx.x == 0) {
                    const A loss = logarithm(s) + (m - widen(scores[t]));
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
        const bool aligned = ((uintptr_t)out & 15) == (uintptr_t)(row.shift * sizeof(T));
        if (t < 0) {
            for (int q = threadIdx.x; q < row.vectors; q += LONG_THREADS)
                store_vector<T>(out, row.first(q), classes, aligned, vec_zero<T, VW>());
            continue;
        }
        with_slope<T>(m, inv, share, [&](auto slopes) {
            for (int q = threadIdx.x; q < row.vectors; q += BATCH * LONG_THREADS) {
                Vec<T, VW> x[BATCH];
#pragma unroll
                for (int b = 0; b < BATCH; ++b) x[b] = vector(q + b * LONG_THREADS < row.vectors ? q + b * LONG_THREADS : q);
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
                    if (q + b * LONG_THREADS < row.vectors)
                        store_vector<T>(out, row.first(q + b * LONG_THREADS), classes, aligned, slopes(x[b]));
            }
            // (by the thread that has written the vector it lies in)
            if ((row.shift + t) / VW % LONG_THREADS == (int)threadIdx.x) out[t] = slopes.at_label(widen(scores[t]), share);
        });
    }
    if constexpr (FORWARD) {
        if (a.reduction != CGNN_NONE) finish<T, LONG_THREADS>(a, total, labelled);
    }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
static std::atomic<int> wait_limit{WAIT_LIMIT};

// Units of work of a call (tiles or rows) that one cluster does alone, saving the launch that counts: as many rounds of its
// blocks take no longer than that launch.
constexpr int64_t CLUSTER_TILES = 4 * CLUSTER, CLUSTER_LONG_ROWS = CLUSTER;

// units: of work; blocks: to a multiprocessor, by their registers.  follows: a reduced forward pass, which one cluster does
// where that is enough for the units, and which otherwise stands behind the launch that counts and may overlap it until it
// waits.
template <typename T>
static int launch(void (*kernel)(LossArgs<T>), LossArgs<T> a, int64_t units, int64_t cluster_units, int threads, int blocks,
                  size_t shared, bool follows, cudaStream_t stream) {
    // (With the kernels' own variables no more than 48 KB need no leave.  The leave belongs to the kernel, and another thread may
    // be between its own and its launch: it is always the same.)
    if (shared > 44 * 1024)
        CGNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DYNAMIC_MOST));
    a.clustered = follows && units <= cluster_units;
    if (follows && !a.clustered) {
        a.count_blocks = a.reduction == CGNN_MEAN ? (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(a.rows, COUNT_THREADS), SMS)) : 1;
        loss_count_kernel<<<(unsigned)a.count_blocks, COUNT_THREADS, 0, stream>>>(
            a.target, a.reduction == CGNN_MEAN ? a.rows : 0, a.classes, a.ignore_index, a.scratch);
        CGNN_LAUNCH_CHECK();
    }
    // (no more than run at once: blocks that began when others end would double the time)
    const int64_t resident = SMS * std::max<int64_t>(1, std::min<int64_t>(blocks, (int64_t)(SHARED_MOST / (shared + 2048))));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(a.clustered ? (unsigned)CLUSTER : (unsigned)std::max<int64_t>(1, std::min<int64_t>(units, resident)));
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    if (a.clustered) {
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = (unsigned)CLUSTER;
        attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    } else {
        attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attribute.val.programmaticStreamSerializationAllowed = 1;
    }
    config.attrs = &attribute;
    config.numAttrs = follows ? 1 : 0;
    CGNN_CUDA(cudaLaunchKernelEx(&config, kernel, a));
    return CGNN_OK;
}

// Whether rows of that many classes begin in too few banks for their lanes: words from row to row a multiple of two.
static bool meet_in_banks(size_t item, int64_t classes) { return classes * item % 8 == 0; }

template <typename T, int LANES, int ROWS, bool FORWARD, int COLUMNS = HELD>
static int launch_tiles(const LossArgs<T> &a, bool follows, cudaStream_t stream) {
    const size_t shared = 2 * ((ROWS * a.classes * sizeof(T) + 15) / 16 * 16);
    auto kernel = meet_in_banks(sizeof(T), a.classes) && LANES < 32 ? loss_tile_kernel<T, LANES, ROWS, COLUMNS, (LANES < 32), FORWARD>
                                                                    : loss_tile_kernel<T, LANES, ROWS, COLUMNS, false, FORWARD>;
    return launch<T>(kernel, a, ceil_div(a.rows, ROWS), CLUSTER_TILES, LANES * ROWS, TILE_BLOCKS<T, LANES * ROWS, COLUMNS>, shared, follows, stream);
}

template <typename T, int THREADS, bool FORWARD>
static int launch_long_rows(const LossArgs<T> &a, size_t shared, bool follows, cudaStream_t stream) {
    return launch<T>(loss_row_kernel<T, THREADS, FORWARD>, a, a.rows, CLUSTER_LONG_ROWS, THREADS, 1024 / THREADS, shared, follows, stream);
}

// follows: a reduced forward pass.
template <typename T, bool FORWARD>
static int launch_rows(const LossArgs<T> &a, bool follows, cudaStream_t stream) {
    // (Forward by twice the columns a lane, where a row has that many: less work around a row for each of its columns, but
    // fewer threads.  60 M scores with their gradient, 24 and 48 columns a lane, us: 50 classes 150 and 128, 64 121 and 106, 192
    // 98 and 92; in bf16 47 classes 85 and 69, 349 84 and 71, but 768 72 and 85.  Backward by twice the columns: 47 classes
    // 95 and 108.)
    if (a.classes <= HELD) return launch_tiles<T, 1, 128, FORWARD>(a, follows, stream);
    if constexpr (FORWARD) {
        if (a.classes <= 2 * HELD) return launch_tiles<T, 1, 128, FORWARD, 2 * HELD>(a, follows, stream);
        if (a.classes <= 4 * HELD) return launch_tiles<T, 2, 64, FORWARD, 2 * HELD>(a, follows, stream);
        if (a.classes <= 8 * HELD) return launch_tiles<T, 4, 32, FORWARD, 2 * HELD>(a, follows, stream);
        if (a.classes <= 16 * HELD) return launch_tiles<T, 8, 16, FORWARD, 2 * HELD>(a, follows, stream);
    } else {
        if (a.classes <= 2 * HELD) return launch_tiles<T, 2, 64, FORWARD>(a, follows, stream);
        if (a.classes <= 4 * HELD) return launch_tiles<T, 4, 32, FORWARD>(a, follows, stream);
        if (a.classes <= 8 * HELD) return launch_tiles<T, 8, 16, FORWARD>(a, follows, stream);
        if (a.classes <= 16 * HELD) return launch_tiles<T, 16, 8, FORWARD>(a, follows, stream);
    }
    if (a.classes <= 32 * HELD) return launch_tiles<T, 32, 8, FORWARD>(a, follows, stream);
    // (60 M scores of 1000 classes with their gradient: 271 us by blocks of 256 threads, 119 by blocks of 64)
    const size_t shared = (a.classes * sizeof(T) + 15) / 16 * 16 + 16;
    if (shared <= 8 * 1024) return launch_long_rows<T, 64, FORWARD>(a, shared, follows, stream);
    if (shared <= 20 * 1024) return launch_long_rows<T, 128, FORWARD>(a, shared, follows, stream);
    if (shared <= 48 * 1024) return launch_long_rows<T, 256, FORWARD>(a, shared, follows, stream);
    if (shared <= SHARED_MOST / 2 - 2048) return launch_long_rows<T, 512, FORWARD>(a, shared, follows, stream);
    if (shared <= DYNAMIC_MOST) return launch_long_rows<T, 1024, FORWARD>(a, shared, follows, stream);
    return launch<T>(loss_long_kernel<T, FORWARD>, a, a.rows, CLUSTER_LONG_ROWS, LONG_THREADS, sizeof(T) == 8 ? 1 : 2, 0, follows, stream);
}

template <typename T>
static int forward(const LossArgs<T> &a, cudaStream_t stream) {
    if (a.reduction == CGNN_NONE) return a.rows ? launch_rows<T, true>(a, false, stream) : CGNN_OK;
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
    a.polls = wait_limit.load(std::memory_order_relaxed);
    a.dense = (stride == classes || rows == 1) && (((uintptr_t)logits | (uintptr_t)grad) & 15) == 0;
    // (a row of 96 bytes shares half of the 64-byte pieces it lies in, and small copies cost ten cycles each: 8.6 M x 7 with a
    // copy for every row 298 us)
    a.whole_tiles = a.dense && classes * (int64_t)sizeof(T) <= 96;
    return a;
}

static int check_call(const char *what, int dtype, int64_t rows, int64_t classes, int64_t stride, int reduction, const void *stats) {
    CGNN_REQUIRE(dtype >= CGNN_F32 && dtype <= CGNN_F16, "%s: unknown dtype %d", what, dtype);
    CGNN_REQUIRE(reduction >= CGNN_NONE && reduction <= CGNN_MEAN, "%s: unknown reduction %d", what, reduction);
    CGNN_REQUIRE(rows >= 0 && stride >= 0, "%s: negative size", what);
    CGNN_REQUIRE(classes >= 1 && classes <= INT32_MAX / 2, "%s: %lld classes are not supported", what, (long long)classes);
    CGNN_REQUIRE(((uintptr_t)stats & (dtype == CGNN_F64 ? 15 : 7)) == 0, "%s: the statistics are pairs on their own boundaries", what);
    return CGNN_OK;
}

}  // namespace cgnn

using namespace cgnn;

extern "C" {

size_t cgnn_cross_entropy_scratch_bytes(void) { return sizeof(LossScratch); }

int cgnn_cross_entropy_wait_limit(int polls) { return wait_limit.exchange(polls < 0 ? WAIT_LIMIT : polls); }

int cgnn_cross_entropy(int dtype, int64_t rows, int64_t classes, int64_t stride, const void *logits, const int64_t *target,
                       int64_t ignore_index, int reduction, void *loss, void *stats, void *grad, int64_t *labelled, void *scratch,
                       size_t scratch_bytes, cgnn_stream_t stream_) {
    if (int rc = check_call("cross_entropy", dtype, rows, classes, stride, reduction, stats)) return rc;
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
    if (int rc = check_call("cross_entropy_backward", dtype, rows, classes, stride, reduction, stats)) return rc;
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
