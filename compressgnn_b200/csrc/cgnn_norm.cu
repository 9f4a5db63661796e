// Layer normalisation of the rows of a matrix, with the ReLU and the dropout that may follow it, both ways.
//
// Forward, per row x of `width` elements:  mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) * rstd,
// z = h * weight + bias, out = dropout(relu(z)).
// Backward: g = the incoming gradient where out depends on z (times the dropout's factor), u = g * weight,
// dx = rstd * (u - mean(u) - h * mean(u * h)), dweight = sum over the rows of g * h, dbias = sum of g.  h and z are
// recomputed from x and the row's two statistics, the mask of the dropout from its key.
//
// Memory bounds both: a row is read once into the registers of its team and everything is computed from there, in
// two passes over the registers (mean, then squared deviations: no cancellation).
#include <algorithm>

#include "cgnn_dropout.cuh"
#include "cgnn_rows.cuh"

namespace cgnn {

constexpr int SMS = 148;
constexpr int LONG_THREADS = 512;     // a block of the kernels that re-read their rows
constexpr int COLUMN_ROWS = 512;      // least rows of a block of norm_columns_kernel

template <typename T>
struct NormArgs {
    using A = Acc<T>;
    const T *x;
    int64_t rows, width, stride;  // x: elements from row to row
    const void *weight, *bias;    // optional [width]
    bool wide_params;             // they are fp32 beside a 16-bit x
    bool whole_params;            // they begin on 32-byte boundaries
    int relu;
    A eps;
    Drop drop;
    T *out;         // forward
    A *mean, *rstd; // [rows]; forward: written unless null
    const T *grad;  // backward: [rows, width]
    T *dx;          // optional
    A *partial;     // optional: [blocks, 2, width], sums of g * h and of g over a block's rows
};

template <typename T, int VW>
__device__ __forceinline__ void params_at(const NormArgs<T> &a, int64_t col, Acc<T> (&w)[VW], Acc<T> (&b)[VW]) {
#pragma unroll
    for (int k = 0; k < VW; ++k) {
        w[k] = Acc<T>(1);
        b[k] = Acc<T>(0);
    }
    if (a.weight) load_params<T, VW>(a.weight, a.wide_params, a.whole_params, col, w);
    if (a.bias) load_params<T, VW>(a.bias, a.wide_params, a.whole_params, col, b);
}

// The dropout of a vector of a row: by a verdict made before (of a row whose lanes have single elements), by the words of
// whole blocks from the row's first one on, or by its own words.
template <int VW, typename A>
__device__ __forceinline__ void drop(const Drop &d, int64_t row_begin, int col, Philox &words, PhiloxRun &run, bool decided, bool gone,
                                     A (&v)[VW]) {
    if (decided) v[0] = gone ? A(0) : v[0] * (A)d.scale;
    else if constexpr (VW % 4 == 0) drop_blocks<A, VW>(v, (uint32_t)col / 4, d.threshold, (A)d.scale, run);
    else drop_values<A, VW>(v, row_begin + col, d.threshold, (A)d.scale, words);
}

// max(z, 0); NaN stays NaN.
__device__ __forceinline__ float positive(float z) {
    float y;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(z));
    return y;
}
__device__ __forceinline__ double positive(double z) { return z < 0.0 ? 0.0 : z; }

template <int TEAM>
constexpr int FORWARD_THREADS = TEAM > 32 ? TEAM : 256;
template <int TEAM>
constexpr int BACKWARD_THREADS = TEAM > 32 ? TEAM : 128;
// Blocks of the backward kernel to a multiprocessor, by the registers that a lane's elements of so many words take.
template <int TEAM, int WORDS>
constexpr int BACKWARD_BLOCKS = std::max(1, (WORDS <= 4 ? 768 : WORDS <= 8 ? 512 : WORDS <= 16 ? 384 : 256) / BACKWARD_THREADS<TEAM>);

// First column of a lane's vector p.  The warps of a large team that holds single elements have runs of columns, so that
// each can draw the random words of its own.
template <int VW, int TEAM, int VPL>
__device__ __forceinline__ int column_of(int lane, int p) {
    if constexpr (VW == 1 && TEAM > 32) return ((lane / 32) * VPL + p) * 32 + lane % 32;
    else return (p * TEAM + lane) * VW;
}

// The team's row, vector by vector; elements beyond the row are zero.
template <typename T, int VW, int TEAM, int VPL>
__device__ __forceinline__ void load_row(const T *row, int width, int lane, Vec<T, VW> (&raw)[VPL]) {
#pragma unroll
    for (int p = 0; p < VPL; ++p) {
        const int col = column_of<VW, TEAM, VPL>(lane, p);
        raw[p] = vec_zero<T, VW>();
        if (col < width) raw[p] = vec_load<T, VW>(row + col);
    }
}

// Forward.  600,000 x 128 in fp32 with dropout: 96 us for 614 MB, the copy rate.  16384 x 4096 in bf16 with ReLU and dropout:
// 76 us, and 45.5 without the dropout (268 MB, 41 us): the random words double the instructions, and 16 warps a multiprocessor
// (112 registers) do not hide their latency between a row's two barriers; issue slots 56 % busy, DRAM 35 %.
template <typename T, int VW, int TEAM, int VPL, bool DROP>
__global__ void __launch_bounds__(FORWARD_THREADS<TEAM>, 512 / FORWARD_THREADS<TEAM>) norm_kernel(const NormArgs<T> a) {
    using A = Acc<T>;
    constexpr int TEAMS = FORWARD_THREADS<TEAM> / TEAM;
    constexpr bool KEEP = VPL * VW <= 16;          // the parameters of a lane's columns stay in registers
    constexpr bool VOTES = TEAM >= 32 && VW == 1;  // a warp draws the words of its columns together
    constexpr int SUMS = VW % 2 == 0 ? 2 : 1;
    __shared__ A shared[2 * (TEAM > 32 ? TEAM / 32 : 1)];
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM, width = (int)a.width;
    Philox words(DROP ? a.drop.key() : 0);
    int turn = 0;
    const A inv = A(1) / (A)a.width;
    A w[KEEP ? VPL : 1][VW], b[KEEP ? VPL : 1][VW];
    if constexpr (KEEP)
#pragma unroll
        for (int p = 0; p < VPL; ++p)
            if (column_of<VW, TEAM, VPL>(lane, p) < width) params_at<T, VW>(a, column_of<VW, TEAM, VPL>(lane, p), w[p], b[p]);
    // While a row is worked on the next one is on its way.
    Vec<T, VW> raw[VPL];
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    int64_t r = (int64_t)blockIdx.x * TEAMS + team;
    if (r < a.rows) load_row<T, VW, TEAM, VPL>(a.x + r * a.stride, width, lane, raw);
    for (; r < a.rows; r += step) {
        A v[VPL][VW], two[SUMS] = {}, s[1];
#pragma unroll
        for (int p = 0; p < VPL; ++p) widen_all<T, VW>(raw[p], v[p]);
        if (r + step < a.rows) load_row<T, VW, TEAM, VPL>(a.x + (r + step) * a.stride, width, lane, raw);
        uint32_t gone = 0;
        PhiloxRun run(words, (uint64_t)(r * a.width) >> 2, (uint32_t)width >> 2);
        if constexpr (VOTES)
            if (DROP) gone = dropped_of_row<VPL>(r * a.width + lane / 32 * (32 * VPL), a.drop.threshold, words);
#pragma unroll
        for (int p = 0; p < VPL; ++p) add(v[p], two);
        s[0] = SUMS == 2 ? two[0] + two[SUMS - 1] : two[0];
        team_sum<A, TEAM, 1>(s, shared, turn);
        const A mean = s[0] * inv;
        two[0] = two[SUMS - 1] = A(0);
#pragma unroll
        for (int p = 0; p < VPL; ++p) {
            add_to_all(v[p], -mean);
            if (column_of<VW, TEAM, VPL>(lane, p) < width) multiply_add(v[p], v[p], two);
        }
        s[0] = SUMS == 2 ? two[0] + two[SUMS - 1] : two[0];
        team_sum<A, TEAM, 1>(s, shared, turn);
        const A rstd = inverse_root(fused(s[0], inv, a.eps));
        if (a.mean && lane == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        T *const out = a.out + r * a.width;
#pragma unroll
        for (int p = 0; p < VPL; ++p) {
            const int col = column_of<VW, TEAM, VPL>(lane, p);
            if (col >= width) continue;
            A z[VW];
            multiply_all(v[p], rstd);
            if constexpr (KEEP) {
                multiply_add_to(v[p], w[p], b[p], z);
            } else {
                params_at<T, VW>(a, col, w[0], b[0]);
                multiply_add_to(v[p], w[0], b[0], z);
            }
            if (a.relu)
#pragma unroll
                for (int k = 0; k < VW; ++k) z[k] = positive(z[k]);
            if (DROP) drop(a.drop, r * a.width, col, words, run, VOTES, gone >> p & 1u, z);
            vec_store<T, VW>(out + col, narrow_all<T, VW>(z));
        }
    }
}

// dx and a block's share of the parameters' gradients.  A lane keeps the same columns for all its rows, so their sums
// stay in registers; teams of a warp, then the warps of the block, are added up in a fixed order at the end.
// 600,000 x 128 in fp32 with dropout: 140 us for 922 MB, the copy rate; the launch that adds up the shares takes 3.
template <typename T, int VW, int TEAM, int VPL, bool DROP>
__global__ void __launch_bounds__(BACKWARD_THREADS<TEAM>, BACKWARD_BLOCKS<TEAM, VPL * VW * (int)sizeof(Acc<T>) / 4>) norm_backward_kernel(const NormArgs<T> a) {
    using A = Acc<T>;
    constexpr int THREADS = BACKWARD_THREADS<TEAM>, TEAMS = THREADS / TEAM, WARPS = THREADS / 32;
    constexpr int COLUMNS = TEAM * VPL * VW;
    constexpr bool VOTES = TEAM >= 32 && VW == 1;
    constexpr int SUMS = VW % 2 == 0 ? 2 : 1;
    __shared__ A shared[TEAM > 32 ? 4 * TEAM / 32 : 2 * COLUMNS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the launch that adds up the shares)
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM, width = (int)a.width;
    Philox words(DROP ? a.drop.key() : 0);
    int turn = 0;
    const A inv = A(1) / (A)a.width;
    A w[VPL][VW], dw[VPL][VW], db[VPL][VW];
#pragma unroll
    for (int p = 0; p < VPL; ++p) {
        const int col = column_of<VW, TEAM, VPL>(lane, p);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
            w[p][k] = A(0);
            dw[p][k] = db[p][k] = A(0);
        }
        if (col < width) {
            A b[VW];
            params_at<T, VW>(a, col, w[p], b);
        }
    }
    // The next row of both matrices is on its way while one is worked on (without: 148 us for 139 of the 600,000 x 128 case).
    Vec<T, VW> raw_x[VPL], raw_g[VPL];
    A mean_next = A(0), rstd_next = A(0);
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    const auto load = [&](int64_t r) {
        mean_next = a.mean[r];
        rstd_next = a.rstd[r];
        load_row<T, VW, TEAM, VPL>(a.x + r * a.stride, width, lane, raw_x);
        load_row<T, VW, TEAM, VPL>(a.grad + r * a.width, width, lane, raw_g);
    };
    int64_t r = (int64_t)blockIdx.x * TEAMS + team;
    if (r < a.rows) load(r);
    for (; r < a.rows; r += step) {
        A h[VPL][VW], g[VPL][VW], s0[SUMS] = {}, s1[SUMS] = {}, s[2];
        const A mean = mean_next, rstd = rstd_next;
#pragma unroll
        for (int p = 0; p < VPL; ++p) {
            widen_all<T, VW>(raw_x[p], h[p]);
            widen_all<T, VW>(raw_g[p], g[p]);
        }
        if (r + step < a.rows) load(r + step);
        uint32_t gone = 0;
        PhiloxRun run(words, (uint64_t)(r * a.width) >> 2, (uint32_t)width >> 2);
        if constexpr (VOTES)
            if (DROP) gone = dropped_of_row<VPL>(r * a.width + lane / 32 * (32 * VPL), a.drop.threshold, words);
#pragma unroll
        for (int p = 0; p < VPL; ++p) {
            const int col = column_of<VW, TEAM, VPL>(lane, p);
            if (col >= width) continue;
            add_to_all(h[p], -mean);
            multiply_all(h[p], rstd);
            if (DROP) drop(a.drop, r * a.width, col, words, run, VOTES, gone >> p & 1u, g[p]);
            if (a.relu) {
                A again[VW], b[VW], z[VW];
                params_at<T, VW>(a, col, again, b);
                multiply_add_to(h[p], w[p], b, z);
#pragma unroll
                for (int k = 0; k < VW; ++k) g[p][k] = z[k] <= A(0) ? A(0) : g[p][k];
            }
            multiply_add(g[p], h[p], dw[p]);
            add(g[p], db[p]);
            multiply_pairwise(g[p], w[p]);
            add(g[p], s0);
            multiply_add(g[p], h[p], s1);
        }
        if (!a.dx) continue;
        s[0] = SUMS == 2 ? s0[0] + s0[SUMS - 1] : s0[0];
        s[1] = SUMS == 2 ? s1[0] + s1[SUMS - 1] : s1[0];
        team_sum<A, TEAM, 2>(s, shared, turn);
        const A c0 = s[0] * inv, c1 = s[1] * inv;
        T *const dx = a.dx + r * a.width;
#pragma unroll
        for (int p = 0; p < VPL; ++p) {
            const int col = column_of<VW, TEAM, VPL>(lane, p);
            if (col >= width) continue;
            // rstd * (u - (h * c1 + c0))
            A minus_c1[VW];
#pragma unroll
            for (int k = 0; k < VW; ++k) minus_c1[k] = -c1;
            add_to_all(g[p], -c0);
            multiply_add(h[p], minus_c1, g[p]);
            multiply_all(g[p], rstd);
            vec_store<T, VW>(dx + col, narrow_all<T, VW>(g[p]));
        }
    }
    if (!a.partial) return;
    A *mine = a.partial + (int64_t)blockIdx.x * 2 * a.width;
    if constexpr (TEAM <= 32) {
#pragma unroll
        for (int p = 0; p < VPL; ++p)
#pragma unroll
            for (int k = 0; k < VW; ++k)
#pragma unroll
                for (int off = TEAM; off < 32; off <<= 1) {
                    dw[p][k] += __shfl_xor_sync(0xffffffffu, dw[p][k], off);
                    db[p][k] += __shfl_xor_sync(0xffffffffu, db[p][k], off);
                }
        for (int warp = 0; warp < WARPS; ++warp) {
            if ((int)(threadIdx.x >> 5) == warp && (threadIdx.x & 31) < TEAM)
#pragma unroll
                for (int p = 0; p < VPL; ++p)
#pragma unroll
                    for (int k = 0; k < VW; ++k) {
                        A *at = shared + (p * TEAM + lane) * VW + k;
                        at[0] = warp ? at[0] + dw[p][k] : dw[p][k];
                        at[COLUMNS] = warp ? at[COLUMNS] + db[p][k] : db[p][k];
                    }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < width; c += THREADS) {
            mine[c] = shared[c];
            mine[a.width + c] = shared[COLUMNS + c];
        }
    } else {
#pragma unroll
        for (int p = 0; p < VPL; ++p)
#pragma unroll
            for (int k = 0; k < VW; ++k) {
                const int col = column_of<VW, TEAM, VPL>(lane, p) + k;
                if (col < width) {
                    mine[col] = dw[p][k];
                    mine[a.width + col] = db[p][k];
                }
            }
    }
}

// Rows too long for a team's registers: a block passes over its row again instead (it lies in L2 by then).
template <typename T>
__global__ void __launch_bounds__(LONG_THREADS) norm_long_kernel(const NormArgs<T> a) {
    using A = Acc<T>;
    __shared__ A shared[2 * LONG_THREADS / 32];
    Philox words(a.drop.threshold ? a.drop.key() : 0);
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *row = a.x + r * a.stride;
        A s[1] = {A(0)};
        for (int64_t c = threadIdx.x; c < a.width; c += LONG_THREADS) s[0] += widen(row[c]);
        team_sum<A, LONG_THREADS, 1>(s, shared, turn);
        const A mean = s[0] / (A)a.width;
        s[0] = A(0);
        for (int64_t c = threadIdx.x; c < a.width; c += LONG_THREADS) {
            const A d = widen(row[c]) - mean;
            s[0] = fused(d, d, s[0]);
        }
        team_sum<A, LONG_THREADS, 1>(s, shared, turn);
        const A rstd = inverse_root(s[0] / (A)a.width + a.eps);
        if (a.mean && threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int64_t c = threadIdx.x; c < a.width; c += LONG_THREADS) {
            A h[1] = {(widen(row[c]) - mean) * rstd}, w[1], b[1], z[1];
            params_at<T, 1>(a, c, w, b);
            multiply_add_to(h, w, b, z);
            if (a.relu && z[0] < A(0)) z[0] = A(0);
            if (a.drop.threshold) drop_values(z, r * a.width + c, a.drop.threshold, (A)a.drop.scale, words);
            a.out[r * a.width + c] = narrow<T>(z[0]);
        }
    }
}

// One element of a long row on the way back: h and the gradient of z.
template <typename T>
__device__ __forceinline__ void long_element(const NormArgs<T> &a, int64_t r, int64_t c, Acc<T> mean, Acc<T> rstd, Philox &words,
                                             Acc<T> &h, Acc<T> &g, Acc<T> &weight) {
    Acc<T> hat[1] = {(widen(a.x[r * a.stride + c]) - mean) * rstd}, grad[1] = {widen(a.grad[r * a.width + c])}, w[1], b[1], z[1];
    params_at<T, 1>(a, c, w, b);
    multiply_add_to(hat, w, b, z);
    if (a.drop.threshold) drop_values(grad, r * a.width + c, a.drop.threshold, (Acc<T>)a.drop.scale, words);
    if (a.relu && z[0] <= Acc<T>(0)) grad[0] = Acc<T>(0);
    h = hat[0];
    g = grad[0];
    weight = w[0];
}

template <typename T>
__global__ void __launch_bounds__(LONG_THREADS) norm_long_backward_kernel(const NormArgs<T> a) {
    using A = Acc<T>;
    __shared__ A shared[4 * LONG_THREADS / 32];
    Philox words(a.drop.threshold ? a.drop.key() : 0);
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const A mean = a.mean[r], rstd = a.rstd[r];
        A s[2] = {A(0), A(0)}, h, g, w;
        for (int64_t c = threadIdx.x; c < a.width; c += LONG_THREADS) {
            long_element(a, r, c, mean, rstd, words, h, g, w);
            s[0] = fused(g, w, s[0]);
            s[1] = fused(g * w, h, s[1]);
        }
        team_sum<A, LONG_THREADS, 2>(s, shared, turn);
        const A c0 = s[0] / (A)a.width, c1 = s[1] / (A)a.width;
        for (int64_t c = threadIdx.x; c < a.width; c += LONG_THREADS) {
            long_element(a, r, c, mean, rstd, words, h, g, w);
            a.dx[r * a.width + c] = narrow<T>(rstd * (g * w - fused(h, c1, c0)));
        }
    }
}

// Sums over rows_per_block rows of g * h and g, a thread per column.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_kernel(const NormArgs<T> a, int64_t rows_per_block) {
    using A = Acc<T>;
    Philox words(a.drop.threshold ? a.drop.key() : 0);
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) return;
    const int64_t r0 = (int64_t)blockIdx.y * rows_per_block, r1 = min(a.rows, r0 + rows_per_block);
    A dw = A(0), db = A(0), h, g, w;
    for (int64_t r = r0; r < r1; ++r) {
        long_element(a, r, c, a.mean[r], a.rstd[r], words, h, g, w);
        dw = fused(g, h, dw);
        db += g;
    }
    a.partial[(int64_t)blockIdx.y * 2 * a.width + c] = dw;
    a.partial[((int64_t)blockIdx.y * 2 + 1) * a.width + c] = db;
}

// The blocks' shares added up in block order: column c of [dweight, dbias] by the lane c of a block of 32 warps, warp w
// adding shares w, w + 32, ...
template <typename T>
__global__ void __launch_bounds__(1024) norm_sums_kernel(const Acc<T> *partial, int64_t blocks, int64_t width, void *dweight,
                                                         void *dbias, bool wide_params) {
    using A = Acc<T>;
    __shared__ A sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    A s = A(0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (c < 2 * width)
#pragma unroll 4
        for (int64_t b = warp; b < blocks; b += 32) s += partial[b * 2 * width + c];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp || c >= 2 * width) return;
#pragma unroll
    for (int w = 1; w < 32; ++w) s += sums[w][lane];
    void *to = c < width ? dweight : dbias;
    if (!to) return;
    const int64_t at = c < width ? c : c - width;
    if (sizeof(T) == 2 && wide_params) static_cast<float *>(to)[at] = (float)s;
    else static_cast<T *>(to)[at] = narrow<T>(s);
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
// Rows of `vectors` vectors of VW elements: the least team that holds them with at most 16 elements a lane, whose
// parameters then stay in registers.  (600,000 x 128 in fp32 and 100,000 x 768 in bf16, forward / backward with dropout: 96 / 139 and
// 104 / 142 us, for 94 / 141 and 47 / 70 us at the copy rate; 8 elements: 111 / 227 and 110 / 162.)  Single elements are held by a
// warp, whose lanes draw random words together.  Its steps are closer than powers of two because idle columns cost as much as
// others.  60 M elements, us forward / backward, with dropout forward / backward, by these steps and by powers of two:
//   fp32  187: 85 149 146 174, 95 149 197 228    319: 81 138 133 174, 97 145 203 283    603: 119 134 190 233, 140 238 278 608
//         383: 89 130 139 180, 92 133 173 246    761: 117 126 191 221, 136 205 235 534
//   bf16  187: 60 118 150 184, 75 125 206 244    319: 59 113 140 186, 75 143 212 294    603: 172 143 240 248, 199 250 313 571
//         383: 68 110 149 199, 69 127 183 255    761: 164 138 223 238, 179 215 270 479
// f(team, vectors a lane) with both as constants.
template <int N>
struct Num {
    static constexpr int value = N;
};
template <typename A>
constexpr int ELEMENTS = 64 / sizeof(A);  // (8 of fp64)
template <typename A, int VW>
constexpr int64_t TEAM_VECTORS = VW > 1 || sizeof(A) == 4 ? 512 * ELEMENTS<A> / VW : 512;
template <typename A, int VW, typename F>
static int with_team(int64_t vectors, F &&f) {
    if (vectors <= 2) return f(Num<2>(), Num<1>());
    if (vectors <= 4) return f(Num<4>(), Num<1>());
    if (vectors <= 8) return f(Num<8>(), Num<1>());
    if constexpr (VW == 1) {
        if (vectors <= 16) return f(Num<8>(), Num<2>());
        if (vectors <= 32) return f(Num<32>(), Num<1>());
        if (vectors <= 64) return f(Num<32>(), Num<2>());
        if (vectors <= 96) return f(Num<32>(), Num<3>());
        if (vectors <= 128) return f(Num<32>(), Num<4>());
        if (vectors <= 192) return f(Num<32>(), Num<6>());
        if (vectors <= 256) return f(Num<32>(), Num<8>());
        if (vectors <= 320) return f(Num<32>(), Num<10>());
        if (vectors <= 384) return f(Num<32>(), Num<12>());
        if (vectors <= 512) return f(Num<32>(), Num<16>());
        if constexpr (sizeof(A) == 4) {
            if (vectors <= 640) return f(Num<32>(), Num<20>());
            if (vectors <= 768) return f(Num<32>(), Num<24>());
            if (vectors <= 1024) return f(Num<32>(), Num<32>());
            if (vectors <= 2048) return f(Num<128>(), Num<16>());
            if (vectors <= 4096) return f(Num<256>(), Num<16>());
            return f(Num<512>(), Num<16>());
        }
        return CGNN_ERR_INVALID;  // (more are no team's: TEAM_VECTORS)
    } else {
        constexpr int VPL = ELEMENTS<A> / VW;
        if constexpr (VPL > 2)
            if (vectors <= 16) return f(Num<8>(), Num<2>());
        if (vectors <= 8 * VPL) return f(Num<8>(), Num<VPL>());
        if (vectors <= 16 * VPL) return f(Num<16>(), Num<VPL>());
        if (vectors <= 32 * VPL) return f(Num<32>(), Num<VPL>());
        if (vectors <= 64 * VPL) return f(Num<64>(), Num<VPL>());
        if (vectors <= 128 * VPL) return f(Num<128>(), Num<VPL>());
        if (vectors <= 256 * VPL) return f(Num<256>(), Num<VPL>());
        return f(Num<512>(), Num<VPL>());
    }
}

// Elements a vector holds: 16 bytes where rows and pointers allow, 8 where only those fit (not of fp64), else one.
// (600,000 x 100 in bf16: 84 us by single elements forward.)
template <typename T>
constexpr int WIDEST = 16 / (int)sizeof(T);

// Whether rows are whole vectors of n elements, in their places too.
static bool vectors_fit(size_t item, int64_t n, int64_t width, int64_t stride, std::initializer_list<const void *> pointers) {
    uintptr_t bits = 0;
    for (const void *p : pointers) bits |= (uintptr_t)p;
    return width % n == 0 && stride % n == 0 && bits % (n * item) == 0;
}

template <typename T, int VW>
static int forward_typed(const NormArgs<T> &a, cudaStream_t stream) {
    return with_team<Acc<T>, VW>(a.width / VW, [&](auto team, auto vpl) -> int {
        constexpr int TEAM = decltype(team)::value, VPL = decltype(vpl)::value, THREADS = FORWARD_THREADS<TEAM>;
        // (no more than run at once: blocks that began when others end would double the time)
        static const int resident[2] = {resident_blocks(norm_kernel<T, VW, TEAM, VPL, false>, THREADS),
                                        resident_blocks(norm_kernel<T, VW, TEAM, VPL, true>, THREADS)};
        const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(a.rows, THREADS / TEAM), SMS * resident[a.drop.threshold != 0]);
        if (a.drop.threshold) norm_kernel<T, VW, TEAM, VPL, true><<<blocks, THREADS, 0, stream>>>(a);
        else norm_kernel<T, VW, TEAM, VPL, false><<<blocks, THREADS, 0, stream>>>(a);
        CGNN_LAUNCH_CHECK();
        return CGNN_OK;
    });
}

template <typename T>
static int forward(const NormArgs<T> &a, cudaStream_t stream) {
    constexpr int VW = WIDEST<T>;
    const auto fit = [&](int64_t n) { return vectors_fit(sizeof(T), n, a.width, a.stride, {a.x, a.out}); };
    if (fit(VW) && a.width / VW <= TEAM_VECTORS<Acc<T>, VW>) return forward_typed<T, VW>(a, stream);
    if constexpr (VW > 2)
        if (fit(VW / 2) && a.width / (VW / 2) <= TEAM_VECTORS<Acc<T>, VW / 2>) return forward_typed<T, VW / 2>(a, stream);
    if (a.width <= TEAM_VECTORS<Acc<T>, 1>) return forward_typed<T, 1>(a, stream);
    norm_long_kernel<T><<<(unsigned)std::min<int64_t>(a.rows, SMS * 4), LONG_THREADS, 0, stream>>>(a);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

// Blocks of a backward launch, each of which leaves a partial row: those that run at once.
template <int TEAM, int WORDS>
static int64_t backward_blocks(int64_t rows) {
    return std::min<int64_t>(ceil_div(rows, BACKWARD_THREADS<TEAM> / TEAM), SMS * BACKWARD_BLOCKS<TEAM, WORDS>);
}

static int64_t column_blocks(int64_t rows, int64_t width) {
    return std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, COLUMN_ROWS), SMS * 8 / std::max<int64_t>(1, width / 256)));
}

// Partial rows of a backward pass by vectors of VW elements, or the most of the ways it may go.
template <typename A, int VW>
static int64_t partial_rows(int64_t rows, int64_t width) {
    if (width / VW > TEAM_VECTORS<A, VW>) return column_blocks(rows, width);
    int64_t blocks = 0;
    with_team<A, VW>(width / VW, [&](auto team, auto vpl) -> int {
        blocks = backward_blocks<decltype(team)::value, decltype(vpl)::value * VW * (int)sizeof(A) / 4>(rows);
        return 0;
    });
    return blocks;
}
static int64_t partial_rows(size_t item, int64_t rows, int64_t width) {
    if (item == 8) return std::max(partial_rows<double, 1>(rows, width), partial_rows<double, 2>(rows, width));
    const int64_t most = std::max({partial_rows<float, 1>(rows, width), partial_rows<float, 2>(rows, width), partial_rows<float, 4>(rows, width)});
    return item == 4 ? most : std::max(most, partial_rows<float, 8>(rows, width));
}

template <typename T, int VW>
static int backward_typed(const NormArgs<T> &a, int64_t *blocks, cudaStream_t stream) {
    return with_team<Acc<T>, VW>(a.width / VW, [&](auto team, auto vpl) -> int {
        constexpr int TEAM = decltype(team)::value, VPL = decltype(vpl)::value;
        *blocks = backward_blocks<TEAM, VPL * VW * (int)sizeof(Acc<T>) / 4>(a.rows);
        if (a.drop.threshold) norm_backward_kernel<T, VW, TEAM, VPL, true><<<(unsigned)*blocks, BACKWARD_THREADS<TEAM>, 0, stream>>>(a);
        else norm_backward_kernel<T, VW, TEAM, VPL, false><<<(unsigned)*blocks, BACKWARD_THREADS<TEAM>, 0, stream>>>(a);
        CGNN_LAUNCH_CHECK();
        return CGNN_OK;
    });
}

template <typename T>
static int backward(const NormArgs<T> &a, void *dweight, void *dbias, cudaStream_t stream) {
    constexpr int VW = WIDEST<T>;
    int64_t blocks = 0;
    int rc = CGNN_OK;
    const auto fit = [&](int64_t n) { return vectors_fit(sizeof(T), n, a.width, a.stride, {a.x, a.grad, a.dx}); };
    if (fit(VW) && a.width / VW <= TEAM_VECTORS<Acc<T>, VW>) {
        rc = backward_typed<T, VW>(a, &blocks, stream);
    } else if (VW > 2 && fit(VW / 2) && a.width / (VW / 2) <= TEAM_VECTORS<Acc<T>, VW / 2>) {
        rc = backward_typed<T, VW / 2>(a, &blocks, stream);
    } else if (a.width <= TEAM_VECTORS<Acc<T>, 1>) {
        rc = backward_typed<T, 1>(a, &blocks, stream);
    } else {
        if (a.dx) {
            norm_long_backward_kernel<T><<<(unsigned)std::min<int64_t>(a.rows, SMS * 4), LONG_THREADS, 0, stream>>>(a);
            CGNN_LAUNCH_CHECK();
        }
        if (a.partial) {
            blocks = column_blocks(a.rows, a.width);
            const int64_t each = ceil_div(a.rows, blocks);
            blocks = ceil_div(a.rows, each);
            norm_columns_kernel<T><<<dim3((unsigned)ceil_div(a.width, 256), (unsigned)blocks), 256, 0, stream>>>(a, each);
            CGNN_LAUNCH_CHECK();
        }
    }
    if (rc != CGNN_OK || !a.partial) return rc;
    // Its blocks are there when the last of the launch before it end, and wait for them.
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)ceil_div(2 * a.width, 32));
    config.blockDim = dim3(1024);
    config.stream = stream;
    cudaLaunchAttribute follows = {};
    follows.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    follows.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &follows;
    config.numAttrs = 1;
    CGNN_CUDA(cudaLaunchKernelEx(&config, norm_sums_kernel<T>, (const Acc<T> *)a.partial, blocks, a.width, dweight, dbias, a.wide_params));
    return CGNN_OK;
}

// What both directions are given, checked.
struct NormCall {
    int dtype, param_dtype;
    int64_t rows, width, stride;
    const void *x, *weight, *bias;
    double p;
    bool with_params;  // something of param_dtype is read or written
};

static int check_call(const char *what, const NormCall &c) {
    CGNN_REQUIRE(c.dtype >= CGNN_F32 && c.dtype <= CGNN_F16, "%s: unknown dtype %d", what, c.dtype);
    CGNN_REQUIRE(!c.with_params || c.param_dtype == c.dtype ||
                     ((c.dtype == CGNN_BF16 || c.dtype == CGNN_F16) && c.param_dtype == CGNN_F32),
                 "%s: weight, bias and their gradients are of the matrix' type, or fp32 beside a 16-bit one", what);
    CGNN_REQUIRE(c.rows >= 0 && c.width >= 0 && c.stride >= 0, "%s: negative size", what);
    CGNN_REQUIRE(c.p >= 0.0 && c.p < 1.0, "%s: the drop probability must lie in [0, 1)", what);
    CGNN_REQUIRE(c.width <= INT32_MAX / 2, "%s: rows of %lld elements are not supported", what, (long long)c.width);
    return CGNN_OK;
}

template <typename T>
static NormArgs<T> args_of(const NormCall &c, int relu, uint64_t seed, const int64_t *device_seed) {
    NormArgs<T> a{};
    a.x = (const T *)c.x;
    a.rows = c.rows;
    a.width = c.width;
    a.stride = c.stride;
    a.weight = c.weight;
    a.bias = c.bias;
    a.wide_params = c.param_dtype == CGNN_F32 && c.dtype != CGNN_F32;
    a.whole_params = (((uintptr_t)c.weight | (uintptr_t)c.bias) & 31) == 0;
    a.relu = relu;
    a.drop = Drop::of(c.p, seed, device_seed);
    return a;
}

static size_t item_of(int dtype) { return dtype == CGNN_F64 ? 8 : dtype == CGNN_F32 ? 4 : 2; }
static size_t acc_of(int dtype) { return dtype == CGNN_F64 ? 8 : 4; }

}  // namespace cgnn

using namespace cgnn;

extern "C" {

int cgnn_layer_norm(int dtype, int param_dtype, int64_t rows, int64_t width, int64_t stride, const void *x, const void *weight,
                    const void *bias, double eps, int relu, double p, uint64_t seed, const int64_t *device_seed, void *out,
                    void *mean, void *rstd, cgnn_stream_t stream) {
    const NormCall c{dtype, param_dtype, rows, width, stride, x, weight, bias, p, weight || bias};
    if (int rc = check_call("layer_norm", c)) return rc;
    CGNN_REQUIRE((mean == nullptr) == (rstd == nullptr), "layer_norm: both statistics are written, or none");
    if (rows == 0 || width == 0) return CGNN_OK;
    CGNN_REQUIRE(x != nullptr && out != nullptr, "layer_norm: null pointer");
    const auto run = [&](auto zero) -> int {
        using T = decltype(zero);
        NormArgs<T> a = args_of<T>(c, relu, seed, device_seed);
        a.eps = (Acc<T>)eps;
        a.out = (T *)out;
        a.mean = (Acc<T> *)mean;
        a.rstd = (Acc<T> *)rstd;
        return forward<T>(a, (cudaStream_t)stream);
    };
    switch (dtype) {
        case CGNN_F32: return run(0.0f);
        case CGNN_F64: return run(0.0);
        case CGNN_BF16: return run(__nv_bfloat16());
        default: return run(__half());
    }
}

size_t cgnn_layer_norm_scratch_bytes(int dtype, int64_t rows, int64_t width) {
    if (dtype < CGNN_F32 || dtype > CGNN_F16 || rows <= 0 || width <= 0) return 0;
    return (size_t)partial_rows(item_of(dtype), rows, width) * 2 * width * acc_of(dtype);
}

int cgnn_layer_norm_backward(int dtype, int param_dtype, int64_t rows, int64_t width, int64_t stride, const void *x,
                             const void *weight, const void *bias, const void *mean, const void *rstd, const void *grad,
                             int relu, double p, uint64_t seed, const int64_t *device_seed, void *dx, void *dweight,
                             void *dbias, void *scratch, size_t scratch_bytes, cgnn_stream_t stream) {
    const NormCall c{dtype, param_dtype, rows, width, stride, x, weight, bias, p, weight || bias || dweight || dbias};
    if (int rc = check_call("layer_norm_backward", c)) return rc;
    const size_t param = param_dtype == dtype ? item_of(dtype) : 4;
    if (rows == 0 && width > 0) {  // sums of nothing
        if (dweight) CGNN_CUDA(cudaMemsetAsync(dweight, 0, width * param, (cudaStream_t)stream));
        if (dbias) CGNN_CUDA(cudaMemsetAsync(dbias, 0, width * param, (cudaStream_t)stream));
    }
    if (rows == 0 || width == 0 || (!dx && !dweight && !dbias)) return CGNN_OK;
    CGNN_REQUIRE(x != nullptr && mean != nullptr && rstd != nullptr && grad != nullptr, "layer_norm_backward: null pointer");
    CGNN_REQUIRE((!dweight && !dbias) || scratch != nullptr, "layer_norm_backward: null scratch");
    if (dweight || dbias)
        CGNN_REQUIRE(scratch_bytes >= cgnn_layer_norm_scratch_bytes(dtype, rows, width) && ((uintptr_t)scratch & 15) == 0,
                     "layer_norm_backward: the scratch is too small or not 16-byte aligned");
    const auto run = [&](auto zero) -> int {
        using T = decltype(zero);
        NormArgs<T> a = args_of<T>(c, relu, seed, device_seed);
        a.mean = (Acc<T> *)mean;
        a.rstd = (Acc<T> *)rstd;
        a.grad = (const T *)grad;
        a.dx = (T *)dx;
        a.partial = dweight || dbias ? (Acc<T> *)scratch : nullptr;
        return backward<T>(a, dweight, dbias, (cudaStream_t)stream);
    };
    switch (dtype) {
        case CGNN_F32: return run(0.0f);
        case CGNN_F64: return run(0.0);
        case CGNN_BF16: return run(__nv_bfloat16());
        default: return run(__half());
    }
}

}  // extern "C"
