// The products of a dense layer on the tensor cores.
//
// C[m, n] = sum over k of A(m, k) B(n, k) in tiles of 128 x BN by a block for each multiprocessor that walks over them.
//
//   FORWARD  A = x,            B = W        contraction along the rows of both
//   INPUT    A = z (masked),   B = W^T
//   WEIGHT   A = z^T,          B = x^T      contraction over the nodes, which is split over the blocks and joined afterwards
//
// fp32 operands become three bf16 numbers each, high + middle + low (8 bits of the fraction apiece, 24 together), and a
// product six: hh, hm, mh, hl, lh, mm; what is left out is below 2^-23 of a term.  A tensor core adds to its fp32
// accumulator with truncation, so that the error grows with the number of additions: hh has an accumulator of its own, the five
// small ones share another, and after 256 terms both are added to fp32 registers and begin anew.  Six products at
// the bf16 rate are 275 TFLOP/s of fp32, where the fp32 pipes have 72.
//
// The streamed operand goes through registers (loads of 32 bytes a lane, a chunk ahead), because it has to be masked and split; it is
// written to shared memory in the swizzled layout that the tensor core reads.  The weight is laid out and split once a
// call by a kernel of its own, as the images of shared memory that bulk copies fetch.
#include <algorithm>

#include "cgnn_linear.cuh"

namespace cgnn {
namespace {

constexpr int BM = 128, BK = 64;  // BK 16-bit elements are a row of 128 bytes, the width of the swizzle
constexpr int EPILOGUE_WARPS = 8, PRODUCER_WARPS = 8;
constexpr int PRODUCERS = PRODUCER_WARPS * 32;
constexpr int MMA_WARP = EPILOGUE_WARPS + PRODUCER_WARPS, COPY_WARP = MMA_WARP + 1;
constexpr int THREADS = (COPY_WARP + 1) * 32;
constexpr int SMS = 148;
constexpr int TMEM_COLUMNS = 512;  // two buffers of 256

template <typename T>
struct Shape {
    static constexpr bool SPLIT = sizeof(T) == 4;
    static constexpr int PLANES = SPLIT ? 3 : 1;
    static constexpr int BN = SPLIT ? 128 : 256;
    static constexpr int STAGES = SPLIT ? 2 : 4;
    static constexpr int A_PLANE = BM * BK * 2, B_PLANE = BN * BK * 2;
    static constexpr int STAGE = PLANES * (A_PLANE + B_PLANE);
    static constexpr int SEGMENT = SPLIT ? 4 : 1 << 30;  // chunks of BK that an accumulator takes
    static constexpr int SUMS = 16 * BM * 4;             // shared memory of the column sums
    static constexpr int SHARED = STAGES * STAGE + SUMS + 1024;
};

template <typename T>
struct Tiles {
    const T *a, *b;               // b: the weight (FORWARD, INPUT) or x (WEIGHT)
    int64_t a_stride, b_stride;   // of their rows
    const uint8_t *packed;        // FORWARD, INPUT: the weight's images
    const uint8_t *mask;          // of A's elements; null: all of them
    int64_t mask_pitch;
    int64_t M, N, K;
    int64_t k_per_item;
    int tiles_m, tiles_n, items;
    int a_whole, b_whole;         // rows lie on vectors of 8 elements
    void *out;                    // [M, N] of T, or (WEIGHT of several splits) [splits, M, N] of fp32
    int64_t out_whole;            // its rows lie on vectors of 8 elements
    int partial;
    float *column_sums;           // WEIGHT: [splits, M]
    float scale;
    Epilogue<T> epilogue;         // FORWARD
    int polls;
    int *status;
};

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(uint64_t *barrier, int arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(barrier)), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t *barrier) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(barrier)) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t *barrier, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(barrier)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_poll(uint64_t *barrier, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done)
                 : "r"(shared_address(barrier)), "r"(parity)
                 : "memory");
    return done != 0;
}
// Waits for the phase of that parity; gives up after `polls`, or when another thread of the block has.
__device__ __forceinline__ bool barrier_wait(uint64_t *barrier, uint32_t parity, int polls, volatile int *given_up) {
    for (int i = 0; i < polls; ++i) {
        if (barrier_poll(barrier, parity)) return true;
        if (*given_up) return false;
    }
    *given_up = 1;
    return false;
}
__device__ __forceinline__ void bulk_copy(uint32_t to, const void *from, uint32_t bytes, uint64_t *barrier) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from),
                 "r"(bytes), "r"(shared_address(barrier))
                 : "memory");
}

// ---------------------------------------------------------------------------------------------
// tensor core instructions
// ---------------------------------------------------------------------------------------------
// A matrix in shared memory, rows of 128 bytes swizzled in groups of eight.  `leading`: bytes between panels of 64 elements along
// m or n where those are contiguous; `stride`: bytes between groups of eight rows.
__device__ __forceinline__ uint64_t matrix_descriptor(uint32_t address, uint32_t leading, uint32_t stride) {
    return (uint64_t)((address >> 4) & 0x3fff) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// fp32 accumulators; operands bf16 or fp16, contiguous along k or (along_mn) along m and n.
__host__ __device__ constexpr uint32_t product_descriptor(bool bf16, bool along_mn) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (along_mn ? 1u << 15 | 1u << 16 : 0u) | (uint32_t)(BM / 16) << 24;
}
__device__ __forceinline__ void multiply(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t descriptor, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(accumulator),
                 "l"(a), "l"(b), "r"(descriptor), "r"((uint32_t)add)
                 : "memory");
}
// The barrier is told when the products issued by this thread up to here are done.
__device__ __forceinline__ void commit(uint64_t *barrier) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(barrier)) : "memory");
}
// Sixteen columns of the warp's 32 rows (a row a lane), with the sixteen of the small products' accumulator added.  Load and wait in
// one statement: a register is not looked at before its value has arrived.
#define CGNN_SIXTEEN(r) "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]), "=&r"(r[8]), \
    "=&r"(r[9]), "=&r"(r[10]), "=&r"(r[11]), "=&r"(r[12]), "=&r"(r[13]), "=&r"(r[14]), "=&r"(r[15])
template <bool TWO>
__device__ __forceinline__ void tmem_load16(uint32_t address, float (&v)[16]) {
    uint32_t r[16];
    if constexpr (TWO) {
        uint32_t q[16];
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n"
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
            "[%33];\n"
            "tcgen05.wait::ld.sync.aligned;"
            : CGNN_SIXTEEN(r), CGNN_SIXTEEN(q)
            : "r"(address), "r"(address + 128)
            : "memory");
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]) + __uint_as_float(q[i]);
    } else {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
            "tcgen05.wait::ld.sync.aligned;"
            : CGNN_SIXTEEN(r)
            : "r"(address)
            : "memory");
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
    }
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void store_shared(uint32_t address, const uint4 &v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// ---------------------------------------------------------------------------------------------
// units: 8 elements of a row
// ---------------------------------------------------------------------------------------------
template <typename T>
struct Unit;
template <>
struct Unit<float> {
    float v[8];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.f;
    }
    __device__ __forceinline__ void load(const float *p, int64_t left, bool whole) {
        if (whole && left >= 8) {
            asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                         : "l"(p));
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < left ? p[k] : 0.f;
        }
    }
    __device__ __forceinline__ void keep(uint32_t bits) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (!(bits >> k & 1)) v[k] = 0.f;
    }
    __device__ __forceinline__ float value(int k) const { return v[k]; }
    // The three bf16 planes.
    __device__ __forceinline__ void planes(uint4 (&out)[3]) const {
        uint32_t *const h = &out[0].x, *const m = &out[1].x, *const l = &out[2].x;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            float2 rest = make_float2(v[k], v[k + 1]);
            uint32_t *const part[3] = {h, m, l};
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(rest.x, rest.y);
                const uint32_t bits = *reinterpret_cast<const uint32_t *>(&two);
                part[q][k / 2] = bits;
                if (q < 2) {
                    rest.x -= __uint_as_float(bits << 16);
                    rest.y -= __uint_as_float(bits & 0xffff0000u);
                }
            }
        }
    }
};
template <typename T>
struct Unit16 {
    uint4 v;
    __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const T *p, int64_t left, bool whole) {
        if (whole && left >= 8) {
            v = *reinterpret_cast<const uint4 *>(p);
        } else {
            const uint16_t *const q = reinterpret_cast<const uint16_t *>(p);
            uint32_t *const w = &v.x;
#pragma unroll
            for (int k = 0; k < 8; k += 2)
                w[k / 2] = (k < left ? (uint32_t)q[k] : 0u) | (k + 1 < left ? (uint32_t)q[k + 1] : 0u) << 16;
        }
    }
    __device__ __forceinline__ void keep(uint32_t bits) {
        uint32_t *const w = &v.x;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] &= (bits >> (2 * k) & 1 ? 0xffffu : 0u) | (bits >> (2 * k + 1) & 1 ? 0xffff0000u : 0u);
    }
    __device__ __forceinline__ float value(int k) const {
        const uint32_t w = (&v.x)[k / 2];
        const uint16_t bits = (uint16_t)(k % 2 ? w >> 16 : w);
        return widen(*reinterpret_cast<const T *>(&bits));
    }
    __device__ __forceinline__ void planes(uint4 (&out)[1]) const { out[0] = v; }
};
template <>
struct Unit<__nv_bfloat16> : Unit16<__nv_bfloat16> {};
template <>
struct Unit<__half> : Unit16<__half> {};

// Where a unit lies in a plane of shared memory: row r, unit c of its 128 bytes.
__device__ __forceinline__ uint32_t place(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// ---------------------------------------------------------------------------------------------
// the weight as images of shared memory: [tile of BN][chunk of BK][plane][BN rows of 128 bytes]
// ---------------------------------------------------------------------------------------------
template <typename T, int FORM>
__global__ void __launch_bounds__(256) pack_kernel(const T *weight, int64_t in, int64_t N, int64_t K, int64_t chunks, uint8_t *packed,
                                                   int whole) {
    using S = Shape<T>;
    const int64_t n_rows = (N + S::BN - 1) / S::BN * S::BN;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n_rows * chunks * 8) return;
    // neighbouring threads take neighbouring places in memory: units of a row, or (transposed) columns
    const int64_t n = FORM == FORWARD ? i / (chunks * 8) : i % n_rows, unit = FORM == FORWARD ? i % (chunks * 8) : i / n_rows;
    const int64_t k = unit * 8;
    Unit<T> u;
    u.clear();
    if (n < N && k < K) {
        if (FORM == FORWARD) {
            u.load(weight + n * in + k, K - k, whole);
        } else {
            T v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k + j < K ? weight[(k + j) * in + n] : narrow<T>(0.f);
            u.load(v, 8, false);
        }
    }
    uint4 planes[S::PLANES];
    u.planes(planes);
    uint8_t *const image = packed + ((n / S::BN) * chunks + unit / 8) * S::PLANES * S::B_PLANE;
#pragma unroll
    for (int q = 0; q < S::PLANES; ++q)
        *reinterpret_cast<uint4 *>(image + q * S::B_PLANE + place((int)(n % S::BN), (int)(unit % 8))) = planes[q];
}

// ---------------------------------------------------------------------------------------------
// the walk of a block
// ---------------------------------------------------------------------------------------------
struct Item {
    int64_t m0, n0, k0, k1;
    int split, chunks;
};
template <typename T, int FORM>
__device__ __forceinline__ Item item_of(const Tiles<T> &t, int item) {
    Item i;
    const int tiles = t.tiles_m * t.tiles_n;
    i.split = FORM == WEIGHT ? item / tiles : 0;
    const int tile = FORM == WEIGHT ? item % tiles : item;
    i.m0 = (int64_t)(tile / t.tiles_n) * BM;
    i.n0 = (int64_t)(tile % t.tiles_n) * Shape<T>::BN;
    i.k0 = i.split * t.k_per_item;
    i.k1 = min(t.K, i.k0 + t.k_per_item);
    i.chunks = (int)((i.k1 - i.k0 + BK - 1) / BK);
    return i;
}

// One element by fp32 arithmetic: where an operand is infinite, no number or beyond bf16's range, its parts say nothing.
template <typename T, int FORM>
__device__ __noinline__ float single_element(const Tiles<T> &t, int64_t m, int64_t n, int64_t k0, int64_t k1) {
    float sum = 0.f;
    for (int64_t k = k0; k < k1; ++k) {
        const int64_t row = FORM == WEIGHT ? k : m, column = FORM == WEIGHT ? m : k;
        float a = widen(t.a[row * t.a_stride + column]);
        if (FORM != FORWARD && t.mask != nullptr && !(t.mask[row * t.mask_pitch + column / 8] >> (column % 8) & 1)) a = 0.f;
        sum = fmaf(a, widen(FORM == FORWARD ? t.b[n * t.b_stride + k] : t.b[k * t.b_stride + n]), sum);
        if (sum != sum) break;
    }
    return sum;
}

// Eight neighbouring outputs.
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&y)[8], int64_t left, bool whole) {
    if (whole && left >= 8) {
        if constexpr (sizeof(T) == 4)
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]),
                         "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7])
                         : "memory");
        else
            vec_store<T, 8>(p, narrow_all<T, 8>(y));
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < left) p[k] = narrow<T>(y[k]);
    }
}

// What follows the product of eight neighbouring elements of a row; the bits of those that ReLU and dropout let through.
template <typename T>
__device__ __forceinline__ uint32_t follow(const Epilogue<T> &e, float (&y)[8], int64_t m, int64_t n, int64_t left, bool whole,
                                           const float *bias, Philox &words) {
    uint32_t passed = 0xff;
    if (e.bias != nullptr) {
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] += bias[k];
    }
    if (e.relu) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (y[k] <= 0.f) {  // (a NaN stays one)
                y[k] = 0.f;
                passed &= ~(1u << k);
            }
    }
    const int64_t at = m * e.width + n;
    if (e.drop.threshold) {
        const uint64_t block = (uint64_t)at >> 2;
        const int ahead = (int)(at & 3);
        const uint4 q0 = words(block), q1 = words(block + 1);
        uint32_t w[12] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w, 0, 0, 0, 0};
        if (ahead) {  // the row does not begin with a block
            const uint4 q2 = words(block + 2);
            w[8] = q2.x, w[9] = q2.y, w[10] = q2.z, w[11] = q2.w;
#pragma unroll
            for (int k = 0; k < 11; ++k) w[k] = ahead & 1 ? w[k + 1] : w[k];
#pragma unroll
            for (int k = 0; k < 9; ++k) w[k] = ahead & 2 ? w[k + 2] : w[k];
        }
        const float scale = (float)e.drop.scale;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool kept = w[k] >= e.drop.threshold;
            y[k] = kept ? y[k] * scale : 0.f;
            if (!kept) passed &= ~(1u << k);
        }
    }
    if (e.residual != nullptr) {
        Unit<T> r;
        r.load(e.residual + at, left, whole);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] += r.value(k);
    }
    return passed;
}

template <typename T, int FORM>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ Tiles<T> t) {
    using S = Shape<T>;
    constexpr int BN = S::BN, STAGES = S::STAGES, PLANES = S::PLANES;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t a_full[STAGES], b_full[STAGES], empty[STAGES], sums_full[2], sums_empty[2], drained;
    __shared__ uint32_t tmem_base;
    __shared__ int given_up;
    __shared__ float bias_of_tile[2][BN];
    uint8_t *const stages = raw + (1024 - shared_address(raw) % 1024) % 1024;  // groups of eight swizzled rows lie on 1024 bytes
    float *const column_parts = reinterpret_cast<float *>(stages + STAGES * S::STAGE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            barrier_init(&a_full[s], PRODUCER_WARPS);
            barrier_init(&b_full[s], 1);
            barrier_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            barrier_init(&sums_full[b], 1);
            barrier_init(&sums_empty[b], EPILOGUE_WARPS);
        }
        barrier_init(&drained, 1);
        given_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&tmem_base)),
                     "r"(TMEM_COLUMNS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        fence_before();
    }
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base;
    const int polls = t.polls;

    if (warp < EPILOGUE_WARPS) {
        // ------------------------------------------------------------------ accumulators to results
        constexpr int COLUMNS = 64, PASSES = BN / (2 * COLUMNS);  // of a warp's half of the tile
        const int quarter = warp & 3, half = warp >> 2;
        Philox words(FORM == FORWARD ? t.epilogue.drop.key() : 0);
        uint32_t segment = 0;
        for (int item = blockIdx.x; item < t.items; item += gridDim.x) {
            const Item i = item_of<T, FORM>(t, item);
            const int64_t m = i.m0 + quarter * 32 + lane;
            const bool inside = m < t.M;
            float *const bias = bias_of_tile[half];
            if (FORM == FORWARD && t.epilogue.bias != nullptr) {
                // the half's columns, by the four warps of the half
                asm volatile("bar.sync %0, %1;" ::"r"(1 + half), "n"(EPILOGUE_WARPS / 2 * 32) : "memory");
                for (int c = quarter * 32 + lane; c < BN / 2; c += EPILOGUE_WARPS / 2 * 32) {
                    const int64_t n = i.n0 + half * (BN / 2) + c;
                    bias[c] = n < t.N ? widen(t.epilogue.bias[n]) : 0.f;
                }
                asm volatile("bar.sync %0, %1;" ::"r"(1 + half), "n"(EPILOGUE_WARPS / 2 * 32) : "memory");
            }
            if (FORM == FORWARD && t.epilogue.residual != nullptr && inside) {  // on its way while the products are formed
                const int64_t first = i.n0 + half * (BN / 2), last = min(first + BN / 2, t.N);
                for (int64_t n = first; n < last; n += 128 / (int)sizeof(T))
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(t.epilogue.residual + m * t.N + n));
            }
            float sum[COLUMNS];
            const int segments = S::SPLIT ? (i.chunks + S::SEGMENT - 1) / S::SEGMENT : 1;
            for (int s = 0; s < segments; ++s, ++segment) {
                const uint32_t buffer = segment & 1, parity = segment >> 1 & 1;
                const bool good = barrier_wait(&sums_full[buffer], parity, polls, &given_up);
                const bool alive = __all_sync(0xffffffffu, good);
                const float lost = __uint_as_float(0x7fffffffu);
                fence_after();
#pragma unroll
                for (int pass = 0; pass < PASSES; ++pass) {
                    const int64_t first = i.n0 + half * (BN / 2) + pass * COLUMNS;
                    const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16) + buffer * 256 + half * (BN / 2) + pass * COLUMNS;
#pragma unroll
                    for (int c = 0; c < COLUMNS; c += 16) {
                        float part[16];
                        if (alive) tmem_load16<S::SPLIT>(at + c, part);
#pragma unroll
                        for (int k = 0; k < 16; ++k) sum[c + k] = !alive ? lost : s == 0 ? part[k] : sum[c + k] + part[k];
                    }
                    if (pass == PASSES - 1) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) barrier_arrive(&sums_empty[buffer]);
                    }
                    if (s + 1 < segments || !inside || first >= t.N) continue;
                    uint32_t bits[2] = {0, 0};
#pragma unroll
                    for (int c = 0; c < COLUMNS; c += 8) {
                        const int64_t n = first + c, left = t.N - n;
                        if (left <= 0) continue;
                        float y[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) y[k] = sum[c + k];
                        if constexpr (S::SPLIT) {
                            bool finite = true;
#pragma unroll
                            for (int k = 0; k < 8; ++k) finite = finite && fabsf(y[k]) <= 3.402823466e38f;
                            if (!finite && alive) {
#pragma unroll 1
                                for (int k = 0; k < 8 && k < left; ++k) {
                                    const float exact = single_element<T, FORM>(t, m, n + k, i.k0, i.k1);
#pragma unroll
                                    for (int j = 0; j < 8; ++j)
                                        if (j == k) y[j] = exact;
                                }
                            }
                        }
                        if constexpr (FORM == FORWARD) {
                            const uint32_t passed = follow<T>(t.epilogue, y, m, n, left, t.out_whole, bias + pass * COLUMNS + c, words);
                            bits[c / 32] |= (left >= 8 ? passed : passed & ((1u << left) - 1u)) << (c % 32);
                            store8<T>(static_cast<T *>(t.out) + m * t.N + n, y, left, t.out_whole);
                        } else if (FORM == WEIGHT && t.partial) {
                            store8<float>(static_cast<float *>(t.out) + (i.split * t.M + m) * t.N + n, y, left, t.out_whole);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) y[k] *= t.scale;
                            store8<T>(static_cast<T *>(t.out) + m * t.N + n, y, left, t.out_whole);
                        }
                    }
                    if (FORM == FORWARD && t.epilogue.mask != nullptr)
                        *reinterpret_cast<uint2 *>(t.epilogue.mask + m * t.epilogue.mask_pitch + first / 8) = make_uint2(bits[0], bits[1]);
                }
            }
        }
    } else if (warp < MMA_WARP) {
        // ------------------------------------------------------------------ operands to shared memory
        const int p = threadIdx.x - EPILOGUE_WARPS * 32;
        constexpr int A_UNITS = BM * BK / 8 / PRODUCERS, B_UNITS = FORM == WEIGHT ? BN * BK / 8 / PRODUCERS : 1;
        Unit<T> a[A_UNITS], b[B_UNITS];
        uint32_t keep[A_UNITS];
        const bool masked = FORM != FORWARD && t.mask != nullptr;
        float columns[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) columns[k] = 0.f;

        const auto load = [&](const Item &i, int chunk) {
            const int64_t k0 = i.k0 + (int64_t)chunk * BK;
#pragma unroll
            for (int u = 0; u < A_UNITS; ++u) {
                const int64_t row = FORM == WEIGHT ? k0 + p / 16 + u * 16 : i.m0 + p / 8 + u * 32;
                const int64_t column = FORM == WEIGHT ? i.m0 + p % 16 * 8 : k0 + p % 8 * 8;
                const int64_t rows = FORM == WEIGHT ? i.k1 : t.M, width = FORM == WEIGHT ? t.M : t.K;
                keep[u] = 0xff;
                if (row < rows && column < width) {
                    a[u].load(t.a + row * t.a_stride + column, width - column, t.a_whole);
                    if (masked) keep[u] = t.mask[row * t.mask_pitch + column / 8];
                } else {
                    a[u].clear();
                }
            }
            if constexpr (FORM == WEIGHT) {
                constexpr int ACROSS = BN / 8;
#pragma unroll
                for (int u = 0; u < B_UNITS; ++u) {
                    const int64_t row = k0 + p / ACROSS + u * (PRODUCERS / ACROSS), column = i.n0 + p % ACROSS * 8;
                    if (row < i.k1 && column < t.N) b[u].load(t.b + row * t.b_stride + column, t.N - column, t.b_whole);
                    else b[u].clear();
                }
            }
        };
        const auto store = [&](uint32_t stage, bool summed) {
            float four[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) four[k] = 0.f;
#pragma unroll
            for (int u = 0; u < A_UNITS; ++u) {
                if (masked) a[u].keep(keep[u]);
                if (FORM == WEIGHT && summed)
#pragma unroll
                    for (int k = 0; k < 8; ++k) four[k] += a[u].value(k);
                uint4 planes[PLANES];
                a[u].planes(planes);
                const uint32_t at = FORM == WEIGHT ? (p % 16 / 8) * (BK * 128) + place(p / 16 + u * 16, p % 8)
                                                   : place(p / 8 + u * 32, p % 8);
#pragma unroll
                for (int q = 0; q < PLANES; ++q) store_shared(stage + q * S::A_PLANE + at, planes[q]);
            }
            if constexpr (FORM == WEIGHT) {
#pragma unroll
                for (int k = 0; k < 8; ++k) columns[k] += four[k];
                constexpr int ACROSS = BN / 8;
#pragma unroll
                for (int u = 0; u < B_UNITS; ++u) {
                    uint4 planes[PLANES];
                    b[u].planes(planes);
                    const uint32_t at = (p % ACROSS / 8) * (BK * 128) + place(p / ACROSS + u * (PRODUCERS / ACROSS), p % 8);
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) store_shared(stage + PLANES * S::A_PLANE + q * S::B_PLANE + at, planes[q]);
                }
            }
        };

        uint32_t round = 0;
        bool alive = true;
        int item = blockIdx.x;
        if (item < t.items) load(item_of<T, FORM>(t, item), 0);
        for (; item < t.items; item += gridDim.x) {  // (to the end whatever happens: the barriers below want every thread)
            const Item i = item_of<T, FORM>(t, item);
            const bool summed = FORM == WEIGHT && t.column_sums != nullptr && i.n0 == 0;
            for (int chunk = 0; alive && chunk < i.chunks; ++chunk, ++round) {
                const uint32_t s = round % STAGES, parity = (round / STAGES & 1) ^ 1;
                alive = __all_sync(0xffffffffu, barrier_wait(&empty[s], parity, polls, &given_up));
                if (!alive) break;
                store(shared_address(stages) + s * S::STAGE, summed);
                fence_to_async();
                __syncwarp();
                if (lane == 0) barrier_arrive(&a_full[s]);
                if (chunk + 1 < i.chunks) load(i, chunk + 1);
                else if (item + gridDim.x < t.items) load(item_of<T, FORM>(t, item + gridDim.x), 0);
            }
            if (FORM == WEIGHT && summed) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    column_parts[(p / 16) * BM + p % 16 * 8 + k] = columns[k];
                    columns[k] = 0.f;
                }
                asm volatile("bar.sync 3, %0;" ::"n"(PRODUCERS) : "memory");
                if (p < BM && i.m0 + p < t.M) {
                    float sum = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += column_parts[r * BM + p];
                    if (*(volatile int *)&given_up) sum = __uint_as_float(0x7fffffffu);
                    t.column_sums[i.split * t.M + i.m0 + p] = sum;
                }
                asm volatile("bar.sync 3, %0;" ::"n"(PRODUCERS) : "memory");
            }
        }
    } else if (warp == MMA_WARP) {
        // ------------------------------------------------------------------ products
        if (lane == 0) {
            constexpr bool ALONG_MN = FORM == WEIGHT;
            constexpr uint32_t base = product_descriptor(sizeof(T) == 4 || __is_same(T, __nv_bfloat16), ALONG_MN);
            constexpr uint32_t LEADING = ALONG_MN ? BK * 128 : 16, STEP = ALONG_MN ? 16 * 128 : 32;  // STEP: 16 along k
            uint32_t round = 0, segment = 0;
            bool alive = true;
            for (int item = blockIdx.x; alive && item < t.items; item += gridDim.x) {
                const Item i = item_of<T, FORM>(t, item);
                const int columns = (int)min((int64_t)BN, (t.N - i.n0 + 15) / 16 * 16);
                const uint32_t descriptor = base | (uint32_t)(columns / 8) << 17;
                for (int chunk = 0; alive && chunk < i.chunks; ++chunk, ++round) {
                    const uint32_t buffer = segment & 1, accumulator = tmem + buffer * 256;
                    const bool fresh = chunk % S::SEGMENT == 0;
                    if (fresh) alive = barrier_wait(&sums_empty[buffer], (segment >> 1 & 1) ^ 1, polls, &given_up);
                    const uint32_t s = round % STAGES, parity = round / STAGES & 1;
                    alive = alive && barrier_wait(&a_full[s], parity, polls, &given_up);
                    if (FORM != WEIGHT) alive = alive && barrier_wait(&b_full[s], parity, polls, &given_up);
                    if (!alive) break;
                    fence_after();
                    const uint32_t stage = shared_address(stages) + s * S::STAGE;
                    uint64_t a[PLANES], b[PLANES];
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
                        a[q] = matrix_descriptor(stage + q * S::A_PLANE, LEADING, 1024);
                        b[q] = matrix_descriptor(stage + PLANES * S::A_PLANE + q * S::B_PLANE, LEADING, 1024);
                    }
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k) {
                        const uint64_t step = (uint64_t)(k * STEP >> 4);
                        const bool add = !fresh || k > 0;
                        multiply(accumulator, a[0] + step, b[0] + step, descriptor, add);
                        if constexpr (S::SPLIT) {
                            const uint32_t small = accumulator + 128;
                            multiply(small, a[0] + step, b[1] + step, descriptor, add);
                            multiply(small, a[1] + step, b[0] + step, descriptor, true);
                            multiply(small, a[0] + step, b[2] + step, descriptor, true);
                            multiply(small, a[2] + step, b[0] + step, descriptor, true);
                            multiply(small, a[1] + step, b[1] + step, descriptor, true);
                        }
                    }
                    commit(&empty[s]);
                    if (chunk + 1 == i.chunks || (chunk + 1) % S::SEGMENT == 0) {
                        commit(&sums_full[buffer]);
                        ++segment;
                    }
                }
            }
            for (uint32_t r = round > STAGES ? round - STAGES : 0; alive && r < round; ++r)  // the last reports have come in
                alive = barrier_wait(&empty[r % STAGES], r / STAGES & 1, polls, &given_up);
            if (!alive) {  // products that are still under way read shared memory and write the accumulators
                atomicOr(t.status, STATUS_WAIT_EXPIRED);
                commit(&drained);
                for (int k = 0; k < WAIT_LIMIT && !barrier_poll(&drained, 0); ++k) {}
            }
        }
    } else if (FORM != WEIGHT) {
        // ------------------------------------------------------------------ the weight's images
        if (lane == 0) {
            uint32_t round = 0;
            bool alive = true;
            const int64_t chunks = (t.K + BK - 1) / BK;
            for (int item = blockIdx.x; alive && item < t.items; item += gridDim.x) {
                const Item i = item_of<T, FORM>(t, item);
                const uint32_t rows = (uint32_t)min((int64_t)BN, (t.N - i.n0 + 15) / 16 * 16);
                const uint8_t *image = t.packed + (i.n0 / BN) * chunks * PLANES * S::B_PLANE;
                for (int chunk = 0; alive && chunk < i.chunks; ++chunk, ++round, image += PLANES * S::B_PLANE) {
                    const uint32_t s = round % STAGES;
                    alive = barrier_wait(&empty[s], (round / STAGES & 1) ^ 1, polls, &given_up);
                    if (!alive) break;
                    const uint32_t to = shared_address(stages) + s * S::STAGE + PLANES * S::A_PLANE;
                    barrier_expect(&b_full[s], rows * 128 * PLANES);
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) bulk_copy(to + q * S::B_PLANE, image + q * S::B_PLANE, rows * 128, &b_full[s]);
                }
            }
            if (!alive)  // copies that are still under way write shared memory
                for (uint32_t r = round > STAGES ? round - STAGES : 0; r < round; ++r)
                    for (int k = 0; k < WAIT_LIMIT && !barrier_poll(&b_full[r % STAGES], r / STAGES & 1); ++k) {}
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && given_up) atomicOr(t.status, STATUS_WAIT_EXPIRED);
    if (warp == MMA_WARP) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLUMNS) : "memory");
    }
}

bool whole_rows(const void *p, int64_t stride, size_t item) {
    return stride % 8 == 0 && (uintptr_t)p % (8 * item) == 0;
}

template <typename T>
size_t packed_bytes(int64_t N, int64_t K) {
    using S = Shape<T>;
    return (size_t)ceil_div(N, S::BN) * (size_t)ceil_div(K, BK) * S::PLANES * S::B_PLANE;
}

template <typename T, int FORM>
int launch(Tiles<T> &t, int64_t splits, cudaStream_t stream) {
    using S = Shape<T>;
    const int64_t tiles_m = ceil_div(t.M, BM), tiles_n = ceil_div(t.N, S::BN);
    CGNN_REQUIRE(tiles_m * tiles_n * splits < (1ll << 30), "linear: too many tiles");
    t.tiles_m = (int)tiles_m;
    t.tiles_n = (int)tiles_n;
    t.items = (int)(tiles_m * tiles_n * splits);
    CGNN_CUDA(cudaFuncSetAttribute(tile_kernel<T, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SHARED));
    tile_kernel<T, FORM><<<(unsigned)std::min(t.items, SMS), THREADS, S::SHARED, stream>>>(t);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

template <typename T, int FORM>
int pack(const T *weight, int64_t in, int64_t N, int64_t K, uint8_t *packed, cudaStream_t stream) {
    using S = Shape<T>;
    const int64_t chunks = ceil_div(K, BK), units = ceil_div(N, S::BN) * S::BN * chunks * 8;
    pack_kernel<T, FORM><<<(unsigned)ceil_div(units, 256), 256, 0, stream>>>(weight, in, N, K, chunks, packed,
                                                                              whole_rows(weight, in, sizeof(T)));
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

}  // namespace

template <typename T>
size_t tiles_forward_bytes(int64_t in, int64_t out) {
    return packed_bytes<T>(out, in);
}

template <typename T>
int tiles_forward(const Call &c, const T *weight, const Epilogue<T> &epilogue, T *y, void *scratch, int polls, int *status,
                  cudaStream_t stream) {
    uint8_t *const packed = static_cast<uint8_t *>(scratch);
    int rc = pack<T, FORWARD>(weight, c.in, c.out, c.in, packed, stream);
    if (rc != CGNN_OK) return rc;
    Tiles<T> t{};
    t.a = static_cast<const T *>(c.x);
    t.a_stride = c.stride;
    t.a_whole = whole_rows(c.x, c.stride, sizeof(T));
    t.b = weight;
    t.b_stride = c.in;
    t.packed = packed;
    t.M = c.rows;
    t.N = c.out;
    t.K = t.k_per_item = c.in;
    t.out = y;
    t.out_whole = whole_rows(y, c.out, sizeof(T)) && (epilogue.residual == nullptr || whole_rows(epilogue.residual, c.out, sizeof(T)));
    t.epilogue = epilogue;
    t.polls = polls;
    t.status = status;
    return launch<T, FORWARD>(t, 1, stream);
}

// Splits of the rows of a weight gradient: what gives every multiprocessor one item, and none of fewer than four chunks.
template <typename T>
static int64_t weight_splits(int64_t rows, int64_t in, int64_t out, int64_t *rows_per_split) {
    const int64_t tiles = ceil_div(out, BM) * ceil_div(in, Shape<T>::BN);
    const int64_t wanted = std::max<int64_t>(1, std::min<int64_t>(SMS / tiles, rows / (4 * BK)));
    *rows_per_split = ceil_div(ceil_div(rows, wanted), BK) * BK;
    return ceil_div(rows, *rows_per_split);
}

template <typename T>
size_t tiles_backward_bytes(int64_t rows, int64_t in, int64_t out) {
    int64_t per_split;
    const int64_t splits = weight_splits<T>(rows, in, out, &per_split);
    return packed_bytes<T>(in, out) + (size_t)splits * out * (in + 1) * sizeof(float) + 64;
}

template <typename T>
int tiles_backward(const Call &c, const T *weight, const T *grad, const uint8_t *mask, double scale, T *dx, T *dweight, T *dbias,
                   void *scratch, int polls, int *status, cudaStream_t stream) {
    uint8_t *const packed = static_cast<uint8_t *>(scratch);
    Tiles<T> t{};
    t.a = grad;
    t.a_stride = c.out;
    t.a_whole = whole_rows(grad, c.out, sizeof(T));
    t.mask = mask;
    t.mask_pitch = mask_pitch(c.out);
    t.scale = (float)scale;
    t.polls = polls;
    t.status = status;
    if (dx != nullptr) {
        int rc = pack<T, INPUT>(weight, c.in, c.in, c.out, packed, stream);
        if (rc != CGNN_OK) return rc;
        t.b = weight;
        t.b_stride = c.in;
        t.packed = packed;
        t.M = c.rows;
        t.N = c.in;
        t.K = t.k_per_item = c.out;
        t.out = dx;
        t.out_whole = whole_rows(dx, c.in, sizeof(T));
        rc = launch<T, INPUT>(t, 1, stream);
        if (rc != CGNN_OK) return rc;
    }
    if (dweight == nullptr && dbias == nullptr) return CGNN_OK;
    int64_t per_split;
    const int64_t splits = weight_splits<T>(c.rows, c.in, c.out, &per_split);
    float *const parts = reinterpret_cast<float *>(align_up((size_t)packed + packed_bytes<T>(c.in, c.out), 32));
    float *const sums = parts + splits * c.out * c.in;
    t.b = static_cast<const T *>(c.x);
    t.b_stride = c.stride;
    t.b_whole = whole_rows(c.x, c.stride, sizeof(T));
    t.packed = nullptr;
    t.M = c.out;
    t.N = c.in;
    t.K = c.rows;
    t.k_per_item = per_split;
    t.partial = splits > 1 || dweight == nullptr;
    t.out = t.partial ? static_cast<void *>(parts) : dweight;
    t.out_whole = t.partial ? c.in % 8 == 0 : whole_rows(dweight, c.in, sizeof(T));
    t.column_sums = dbias != nullptr ? sums : nullptr;
    int rc = launch<T, WEIGHT>(t, splits, stream);
    if (rc == CGNN_OK && t.partial && dweight != nullptr) rc = join<T>(parts, splits, c.out * c.in, scale, dweight, stream);
    if (rc == CGNN_OK && dbias != nullptr) rc = join<T>(sums, splits, c.out, scale, dbias, stream);
    return rc;
}

#define CGNN_TILES_OF(T)                                                                                                        \
    template size_t tiles_forward_bytes<T>(int64_t, int64_t);                                                                   \
    template int tiles_forward<T>(const Call &, const T *, const Epilogue<T> &, T *, void *, int, int *, cudaStream_t);         \
    template size_t tiles_backward_bytes<T>(int64_t, int64_t, int64_t);                                                         \
    template int tiles_backward<T>(const Call &, const T *, const T *, const uint8_t *, double, T *, T *, T *, void *, int, int *, \
                                   cudaStream_t);
CGNN_TILES_OF(float)
CGNN_TILES_OF(__nv_bfloat16)
CGNN_TILES_OF(__half)

}  // namespace cgnn
