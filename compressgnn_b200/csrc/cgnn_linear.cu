// A dense layer as one product, and its gradients.
//
//   forward    y = residual + dropout(act(x W^T + b)), and a mask of the elements that act and dropout let through
//   backward   z = grad where the mask has a bit, 0 elsewhere, s = 1 / (1 - p):
//              dx = s z W,  dW = s z^T x,  db = s (column sums of z)
#include <algorithm>
#include <atomic>

#include "cgnn_dropout.cuh"
#include "cgnn_linear.cuh"
#include "cgnn_rows.cuh"

namespace cgnn {

namespace {

// ---------------------------------------------------------------------------------------------
// products by single elements: fp64, and calls too small to fill tiles of 128 x 128
// ---------------------------------------------------------------------------------------------
constexpr int TM = 32, TN = 64, TK = 16, TILE_THREADS = 128;
constexpr int TILE_WAVE = 148 * 4;

// Groups of TILE_THREADS that share a block's terms where blocks are few: one group is one warp to each of an SM's four
// schedulers, and its own instructions bound it.  4 groups of fp32 (2 of fp64: what they stage is what static shared memory holds).
template <typename A>
constexpr int GROUPS = 16 / (int)sizeof(A);

// C[m, n] = sum over k of A(m, k) B(n, k).  A: x, or z (masked); B: the weight, its transpose, or x.
template <typename T>
struct Small {
    const T *a, *b;
    int64_t a_m, a_k, b_n, b_k;   // strides
    int64_t M, N, K;
    const uint8_t *mask;          // of A's elements; null: all of them
    int64_t mask_pitch;
    int64_t k_per_split;
    void *out;                    // FORWARD, INPUT: [M, N] of T; WEIGHT: [splits, M, N] sums, or, of one split, T
    double scale;
    Epilogue<T> epilogue;         // FORWARD
};

template <typename T, int FORM, int GROUPS>
__global__ void __launch_bounds__(GROUPS *TILE_THREADS) small_kernel(const Small<T> s) {
    using A = Acc<T>;
    __shared__ A as_of[GROUPS][TK][TM + 1];
    __shared__ A bs_of[GROUPS][TK][TN + 1];
    const int group = GROUPS > 1 ? threadIdx.x / TILE_THREADS : 0, thread = GROUPS > 1 ? threadIdx.x % TILE_THREADS : threadIdx.x;
    auto &as = as_of[group];
    auto &bs = bs_of[group];
    const int64_t tiles_n = (s.N + TN - 1) / TN > 0 ? (s.N + TN - 1) / TN : 1;
    const int64_t m0 = (blockIdx.x / tiles_n) * TM, n0 = (blockIdx.x % tiles_n) * TN;
    const int64_t k_begin = (int64_t)blockIdx.y * s.k_per_split, k_end = min(s.K, k_begin + s.k_per_split);
    const int tx = thread % 16, ty = thread / 16;  // columns tx + 16 j, rows ty * 4 + i
    A acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = A(0);
    constexpr bool A_ALONG_K = FORM != WEIGHT, B_ALONG_K = FORM == FORWARD;
    for (int64_t stage = k_begin; stage < k_end; stage += GROUPS * TK) {
        const int64_t k0 = stage + group * TK;  // (may lie behind the end: zeros)
#pragma unroll
        for (int i = thread; i < TM * TK; i += TILE_THREADS) {
            const int m = A_ALONG_K ? i / TK : i % TM, k = A_ALONG_K ? i % TK : i / TM;
            A v = A(0);
            if (m0 + m < s.M && k0 + k < k_end) {
                v = widen(s.a[(m0 + m) * s.a_m + (k0 + k) * s.a_k]);
                if (FORM != FORWARD && s.mask != nullptr) {
                    const int64_t row = A_ALONG_K ? m0 + m : k0 + k, column = A_ALONG_K ? k0 + k : m0 + m;
                    if (!(s.mask[row * s.mask_pitch + column / 8] >> (column % 8) & 1)) v = A(0);
                }
            }
            as[k][m] = v;
        }
#pragma unroll
        for (int i = thread; i < TN * TK; i += TILE_THREADS) {
            const int n = B_ALONG_K ? i / TK : i % TN, k = B_ALONG_K ? i % TK : i / TN;
            bs[k][n] = n0 + n < s.N && k0 + k < k_end ? A(widen(s.b[(n0 + n) * s.b_n + (k0 + k) * s.b_k])) : A(0);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TK; ++k) {
            A av[4], bv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) av[i] = as[k][ty * 4 + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) bv[j] = bs[k][tx + 16 * j];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fused(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
    if constexpr (GROUPS > 1) {  // (the last stage's barrier is behind every thread: its place is free)
        static_assert(16 * TILE_THREADS <= GROUPS * TK * (TN + 1), "a group's sums are wider than the stages");
        A *const sums = &bs_of[0][0][0];
        for (int g = 1; g < GROUPS; ++g) {
            if (group == g)
#pragma unroll
                for (int i = 0; i < 16; ++i) sums[i * TILE_THREADS + thread] = acc[i / 4][i % 4];
            __syncthreads();
            if (group == 0)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[i / 4][i % 4] += sums[i * TILE_THREADS + thread];
            __syncthreads();
        }
        if (group > 0) return;
    }
    const bool whole = gridDim.y == 1;
    if constexpr (FORM == FORWARD) {
        Philox words(s.epilogue.drop.key());
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + ty * 4 + i;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t n = n0 + tx + 16 * j;
                const bool inside = m < s.M && n < s.N;
                bool passed = false;
                if (inside) {
                    A y = acc[i][j];
                    passed = s.epilogue.element(y, m, n, words);
                    static_cast<T *>(s.out)[m * s.N + n] = narrow<T>(y);
                }
                // 16 neighbouring lanes hold 16 neighbouring columns of a row, from a multiple of 16 on
                const uint32_t bits = __ballot_sync(0xffffffffu, passed) >> (threadIdx.x & 16);
                if (s.epilogue.mask != nullptr && tx == 0 && m < s.M && n0 + 16 * j < (int64_t)s.epilogue.mask_pitch * 8)
                    *reinterpret_cast<uint16_t *>(s.epilogue.mask + m * s.epilogue.mask_pitch + (n0 + 16 * j) / 8) = (uint16_t)bits;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + ty * 4 + i;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t n = n0 + tx + 16 * j;
                if (m >= s.M || n >= s.N) continue;
                if (FORM == INPUT || whole) static_cast<T *>(s.out)[m * s.N + n] = narrow<T>(acc[i][j] * (A)s.scale);
                else static_cast<A *>(s.out)[((int64_t)blockIdx.y * s.M + m) * s.N + n] = acc[i][j];
            }
        }
    }
}

int64_t small_tiles(int64_t M, int64_t N) { return ceil_div(M, TM) * std::max<int64_t>(1, ceil_div(N, TN)); }

// Splits of the rows for a weight gradient: one wave of blocks, and none of fewer than 8 stages.
int64_t small_splits(int64_t rows, int64_t in, int64_t out) {
    return std::max<int64_t>(1, std::min<int64_t>(TILE_WAVE / std::max<int64_t>(1, small_tiles(out, in)), rows / (8 * TK)));
}

// Whether groups share a block's terms: while no SM has a second block, and where there are stages to share.  Us by groups / by
// one: fp32 1 x 560 -> 544 forward 22.6 / 28.7, input gradient 19.4 / 38.9, bf16 24.6 / 39.0 and 21.1 / 43.0;
// 1000 x 301 -> 47 (32 tiles) 14.4 / 18.5, its input gradient (160 tiles) 10.3 / 8.2; 10,000 x 64 -> 47 (313) 12.3 / 10.3;
// 2708 x 16 -> 7 (one stage) 6.2 / 5.4.
bool shared_terms(int64_t tiles, int64_t terms) { return tiles <= 148 && terms > 2 * TK; }

template <typename T, int FORM>
int small_product(Small<T> &s, int64_t splits, cudaStream_t stream) {
    const int64_t tiles = small_tiles(s.M, s.N);
    CGNN_REQUIRE(tiles < (1ll << 31), "linear: grid too large");
    s.k_per_split = ceil_div(ceil_div(std::max<int64_t>(s.K, 1), splits), TK) * TK;
    const dim3 grid((unsigned)tiles, (unsigned)splits);
    constexpr int groups = FORM == WEIGHT ? 1 : GROUPS<Acc<T>>;
    if (groups > 1 && shared_terms(tiles, s.K))
        small_kernel<T, FORM, groups><<<grid, groups * TILE_THREADS, 0, stream>>>(s);
    else
        small_kernel<T, FORM, 1><<<grid, TILE_THREADS, 0, stream>>>(s);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

// ---------------------------------------------------------------------------------------------
// the bias' gradient by itself: column sums of z, for which neither x nor the weight is looked at
// ---------------------------------------------------------------------------------------------
// Splits of the rows: some blocks for every multiprocessor, and none of fewer rows than a block has on their way.
int64_t column_splits(int64_t rows, int64_t out) {
    return std::max<int64_t>(1, std::min<int64_t>(148 * 4 / ceil_div(out, 256), rows / (COLUMN_UNROLL * 8)));
}

size_t column_bytes(int64_t rows, int64_t out) {
    const int64_t splits = column_splits(rows, out);
    return splits == 1 ? 0 : (size_t)splits * (size_t)out * sizeof(double);
}

template <typename T, int VW>
int column_sums_by(const Call &c, const T *grad, const uint8_t *mask, double scale, T *dbias, void *scratch, cudaStream_t stream) {
    const int64_t splits = column_splits(c.rows, c.out), vectors = ceil_div(c.out, VW);
    const int across = columns_across(vectors);
    double *const parts = static_cast<double *>(scratch);
    columns_kernel<T, T, VW><<<dim3((unsigned)ceil_div(vectors, 1 << across), (unsigned)splits), COLUMN_THREADS, 0, stream>>>(
        grad, mask, mask_pitch(c.out), c.rows, ceil_div(c.rows, splits), c.out, across, scale, parts, dbias);
    CGNN_LAUNCH_CHECK();
    return splits == 1 ? CGNN_OK : join_columns(parts, splits, c.out, scale, dbias, stream);
}

template <typename T>
int column_sums(const Call &c, const T *grad, const uint8_t *mask, double scale, T *dbias, void *scratch, cudaStream_t stream) {
    constexpr int VW = 16 / sizeof(T);
    return c.out % VW == 0 && (uintptr_t)grad % 16 == 0 ? column_sums_by<T, VW>(c, grad, mask, scale, dbias, scratch, stream)
                                                        : column_sums_by<T, 1>(c, grad, mask, scale, dbias, scratch, stream);
}

size_t small_backward_bytes(int64_t acc_bytes, int64_t rows, int64_t in, int64_t out) {
    const int64_t splits = small_splits(rows, in, out);
    return splits == 1 ? 0 : (size_t)splits * (size_t)out * (size_t)in * (size_t)acc_bytes;
}

template <typename T>
int small_forward(const Call &c, const T *weight, const Epilogue<T> &epilogue, T *y, cudaStream_t stream) {
    Small<T> s{};
    s.a = static_cast<const T *>(c.x);
    s.a_m = c.stride;
    s.a_k = 1;
    s.b = weight;
    s.b_n = c.in;
    s.b_k = 1;
    s.M = c.rows;
    s.N = c.out;
    s.K = c.in;
    s.out = y;
    s.epilogue = epilogue;
    return small_product<T, FORWARD>(s, 1, stream);
}

template <typename T>
int small_backward(const Call &c, const T *weight, const T *grad, const uint8_t *mask, double scale, T *dx, T *dweight, void *scratch,
                   cudaStream_t stream) {
    using A = Acc<T>;
    Small<T> s{};
    s.a = grad;
    s.mask = mask;
    s.mask_pitch = mask_pitch(c.out);
    s.scale = scale;
    if (dx != nullptr) {
        s.a_m = c.out;
        s.a_k = 1;
        s.b = weight;
        s.b_n = 1;
        s.b_k = c.in;
        s.M = c.rows;
        s.N = c.in;
        s.K = c.out;
        s.out = dx;
        const int rc = small_product<T, INPUT>(s, 1, stream);
        if (rc != CGNN_OK) return rc;
    }
    if (dweight == nullptr) return CGNN_OK;
    s.a_m = 1;
    s.a_k = c.out;
    s.b = static_cast<const T *>(c.x);
    s.b_n = 1;
    s.b_k = c.stride;
    s.M = c.out;
    s.N = c.in;
    s.K = c.rows;
    const int64_t splits = small_splits(c.rows, c.in, c.out);
    A *const parts = static_cast<A *>(scratch);
    s.out = splits == 1 ? static_cast<void *>(dweight) : parts;
    const int rc = small_product<T, WEIGHT>(s, splits, stream);
    return rc == CGNN_OK && splits > 1 ? join(parts, splits, c.out * c.in, scale, dweight, stream) : rc;
}

template <typename T>
constexpr bool HAS_TILES = sizeof(T) < 8;

// Whether a call goes to the tensor cores: by its number of multiplications, earlier where rows are whole vectors and where one
// contraction is long (a tile of single elements takes it alone).  Us by tiles / by single elements, forward + input gradient +
// weight gradient: fp32 10,000 x 64 -> 64 (4e7) 47 / 48, 20,000 x 64 -> 64 54 / 64, 2708 x 64 -> 64 46 / 38;
// 40,000 x 64 -> 47 (1e8) 72 / 92, 20,000 x 64 -> 47 60 / 61; 32 x 4096 -> 64 107 / 140;
// bf16 2708 x 64 -> 64 (1e7) 38 / 40, 1024 x 64 -> 64 38 / 40, 256 x 64 -> 64 30 / 37; 20,000 x 64 -> 47 (6e7) 70 / 66.
bool by_tiles(int dtype, int64_t rows, int64_t in, int64_t out) {
    if (dtype == CGNN_F64 || in <= 0) return false;
    const double products = (double)rows * (double)in * (double)out;
    const bool whole = in % 8 == 0 && out % 8 == 0;
    if (std::max(in, out) >= 1024 && products >= 4e6) return true;
    return products >= (dtype == CGNN_F32 ? (whole ? 4e7 : 1e8) : whole ? 4e6 : 6e7);
}

std::atomic<int> wait_limit{WAIT_LIMIT};

template <typename F>
size_t bytes_of_type(int dtype, F &&call) {
    switch (dtype) {
        case CGNN_F32: return call(float());
        case CGNN_BF16: return call(__nv_bfloat16());
        default: return call(__half());
    }
}

template <typename T>
int forward(const Call &c, const void *weight, const void *bias, const void *residual, int relu, double p, const Drop &drop, void *y,
            void *mask, void *scratch, bool tiles, cudaStream_t stream) {
    Epilogue<T> e{};
    e.bias = static_cast<const T *>(bias);
    e.residual = static_cast<const T *>(residual);
    e.mask = relu || p > 0.0 ? static_cast<uint8_t *>(mask) : nullptr;  // (of a p below 2^-32, which drops nothing, too)
    e.mask_pitch = mask_pitch(c.out);
    e.width = c.out;
    e.relu = relu;
    e.drop = drop;
    if constexpr (HAS_TILES<T>)
        if (tiles) return tiles_forward<T>(c, static_cast<const T *>(weight), e, static_cast<T *>(y), scratch, wait_limit.load(), stream);
    return small_forward<T>(c, static_cast<const T *>(weight), e, static_cast<T *>(y), stream);
}

template <typename T>
int backward(const Call &c, const void *weight, const void *mask, const void *grad, double scale, void *dx, void *dweight, void *dbias,
             void *scratch, bool tiles, cudaStream_t stream) {
    // The tensor core path sums the columns on their way to the weight's gradient.  By single elements that is a kernel of its own (sums
    // beside the products: 200,000 x 16 -> 7 weight gradient with the bias' 103 us, without 95; apart 92 and 86; 2708 x 16 -> 7
    // 38 and 34, apart 35 and 28).  Behind it on the stream the other gradients take the scratch anew.
    if (dbias != nullptr && (dweight == nullptr || !tiles)) {
        const int rc = column_sums<T>(c, static_cast<const T *>(grad), static_cast<const uint8_t *>(mask), scale, static_cast<T *>(dbias),
                                      scratch, stream);
        if (rc != CGNN_OK) return rc;
        dbias = nullptr;
    }
    if constexpr (HAS_TILES<T>)
        if (tiles)
            return tiles_backward<T>(c, static_cast<const T *>(weight), static_cast<const T *>(grad), static_cast<const uint8_t *>(mask),
                                     scale, static_cast<T *>(dx), static_cast<T *>(dweight), static_cast<T *>(dbias), scratch,
                                     wait_limit.load(), stream);
    return small_backward<T>(c, static_cast<const T *>(weight), static_cast<const T *>(grad), static_cast<const uint8_t *>(mask),
                             scale, static_cast<T *>(dx), static_cast<T *>(dweight), scratch, stream);
}

int check_call(int dtype, const Call &c, double p) {
    CGNN_REQUIRE(dtype >= CGNN_F32 && dtype <= CGNN_F16, "linear: unknown dtype");
    CGNN_REQUIRE(c.rows >= 0 && c.in >= 0 && c.out >= 0 && c.stride >= 0, "linear: negative size");
    CGNN_REQUIRE(c.in < WIDEST && c.out < WIDEST, "linear: %lld x %lld is not supported", (long long)c.in, (long long)c.out);
    CGNN_REQUIRE(p >= 0.0 && p < 1.0, "linear: dropout probability must lie in [0, 1)");
    return CGNN_OK;
}

}  // namespace
}  // namespace cgnn

using namespace cgnn;

extern "C" {

size_t cgnn_linear_mask_bytes(int64_t rows, int64_t out) { return rows <= 0 || out <= 0 ? 0 : (size_t)rows * mask_pitch(out); }

size_t cgnn_linear_scratch_bytes(int dtype, int64_t rows, int64_t in, int64_t out) {
    if (dtype < CGNN_F32 || dtype > CGNN_F16 || rows <= 0 || in <= 0 || out <= 0 || in >= WIDEST || out >= WIDEST) return 0;
    if (!by_tiles(dtype, rows, in, out)) return 0;
    return bytes_of_type(dtype, [&](auto zero) { return tiles_forward_bytes<decltype(zero)>(rows, in, out); });
}

int cgnn_linear(int dtype, int64_t rows, int64_t in, int64_t out, int64_t stride, const void *x, const void *weight, const void *bias,
                const void *residual, int relu, double p, uint64_t seed, const int64_t *device_seed, void *y, void *mask,
                void *scratch, size_t scratch_bytes, cgnn_stream_t stream_) {
    cudaStream_t stream = (cudaStream_t)stream_;
    const Call c{rows, in, out, stride, x};
    const int rc = check_call(dtype, c, p);
    if (rc != CGNN_OK) return rc;
    if (rows == 0 || out == 0) return CGNN_OK;
    CGNN_REQUIRE(y != nullptr && (in == 0 || (x != nullptr && weight != nullptr)), "linear: null pointer");
    CGNN_REQUIRE(((uintptr_t)mask & 7) == 0, "linear: the mask lies on an 8-byte boundary");
    const size_t need = cgnn_linear_scratch_bytes(dtype, rows, in, out);
    CGNN_REQUIRE(need == 0 || (scratch != nullptr && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0),
                 "linear: scratch too small or not on a 16-byte boundary");
    const Drop drop = Drop::of(p, seed, device_seed);
    const bool tiles = by_tiles(dtype, rows, in, out);
    switch (dtype) {
        case CGNN_F32: return forward<float>(c, weight, bias, residual, relu, p, drop, y, mask, scratch, tiles, stream);
        case CGNN_F64: return forward<double>(c, weight, bias, residual, relu, p, drop, y, mask, scratch, tiles, stream);
        case CGNN_BF16: return forward<__nv_bfloat16>(c, weight, bias, residual, relu, p, drop, y, mask, scratch, tiles, stream);
        default: return forward<__half>(c, weight, bias, residual, relu, p, drop, y, mask, scratch, tiles, stream);
    }
}

size_t cgnn_linear_backward_scratch_bytes(int dtype, int64_t rows, int64_t in, int64_t out) {
    if (dtype < CGNN_F32 || dtype > CGNN_F16 || rows <= 0 || in < 0 || out <= 0 || in >= WIDEST || out >= WIDEST) return 0;
    const size_t columns = column_bytes(rows, out);
    if (by_tiles(dtype, rows, in, out))
        return std::max(columns, bytes_of_type(dtype, [&](auto zero) { return tiles_backward_bytes<decltype(zero)>(rows, in, out); }));
    return std::max(columns, small_backward_bytes(dtype == CGNN_F64 ? 8 : 4, rows, in, out));
}

int cgnn_linear_backward(int dtype, int64_t rows, int64_t in, int64_t out, int64_t stride, const void *x, const void *weight,
                         const void *mask, const void *grad, double p, void *dx, void *dweight, void *dbias, void *scratch,
                         size_t scratch_bytes, cgnn_stream_t stream_) {
    cudaStream_t stream = (cudaStream_t)stream_;
    const Call c{rows, in, out, stride, x};
    const int rc = check_call(dtype, c, p);
    if (rc != CGNN_OK) return rc;
    const size_t item = dtype == CGNN_F64 ? 8 : dtype == CGNN_F32 ? 4 : 2;
    if (rows == 0 || out == 0) {  // sums of nothing
        if (dx != nullptr && rows > 0 && in > 0) CGNN_CUDA(cudaMemsetAsync(dx, 0, (size_t)rows * in * item, stream));
        if (dweight != nullptr && out > 0 && in > 0) CGNN_CUDA(cudaMemsetAsync(dweight, 0, (size_t)out * in * item, stream));
        if (dbias != nullptr && out > 0) CGNN_CUDA(cudaMemsetAsync(dbias, 0, (size_t)out * item, stream));
        return CGNN_OK;
    }
    if (in == 0) dx = dweight = nullptr;
    CGNN_REQUIRE(grad != nullptr, "linear backward: null pointer");
    CGNN_REQUIRE(dx == nullptr || weight != nullptr, "linear backward: the input's gradient needs the weight");
    CGNN_REQUIRE(dweight == nullptr || x != nullptr, "linear backward: the weight's gradient needs the input");
    CGNN_REQUIRE(((uintptr_t)mask & 7) == 0, "linear backward: the mask lies on an 8-byte boundary");
    const size_t need = dx != nullptr || dweight != nullptr || dbias != nullptr ? cgnn_linear_backward_scratch_bytes(dtype, rows, in, out) : 0;
    CGNN_REQUIRE(need == 0 || (scratch != nullptr && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0),
                 "linear backward: scratch too small or not on a 16-byte boundary");
    const double scale = Drop::of(p, 0, nullptr).scale;
    const bool tiles = by_tiles(dtype, rows, in, out);
    switch (dtype) {
        case CGNN_F32: return backward<float>(c, weight, mask, grad, scale, dx, dweight, dbias, scratch, tiles, stream);
        case CGNN_F64: return backward<double>(c, weight, mask, grad, scale, dx, dweight, dbias, scratch, tiles, stream);
        case CGNN_BF16: return backward<__nv_bfloat16>(c, weight, mask, grad, scale, dx, dweight, dbias, scratch, tiles, stream);
        default: return backward<__half>(c, weight, mask, grad, scale, dx, dweight, dbias, scratch, tiles, stream);
    }
}

int cgnn_linear_wait_limit(int polls) { return wait_limit.exchange(polls < 0 ? WAIT_LIMIT : polls); }

}  // extern "C"
