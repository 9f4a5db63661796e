// The products of a dense layer on the tensor cores.
//
// C[m, n] = sum over k of A(m, k) B(n, k) in tiles of 128 x BN by a block for each multiprocessor that walks over them.
//
//   FORWARD  A = x,            B = W        contraction along the rows of both
//   INPUT    A = z (masked),   B = W^T
//   WEIGHT   A = z^T,          B = x^T      contraction over the nodes, which is split over the blocks and joined afterwards
//
// fp32 operands become three bf16 numbers each, high + middle + low (8 bits of the fraction apiece, 24 together), and a
// product six: hh, hm, mh, hl, lh, mm; what is left out is below 2^-23 of a term, or, of an operand below 2^-110, the rest beyond a
// multiple of 2^-133, bf16's least number.  A tensor core adds to its fp32
// accumulator with truncation, so that the error grows with the number of additions: hh has an accumulator of its own, the
// five small ones share another, and after 256 terms both are added to fp32 registers and begin
// anew (325,557 x 256 -> 128: outputs 1.5e-7 of their size from 64 bits, the fp32 pipes' 1.8e-7).  Six products at the bf16
// rate are 275 TFLOP/s of fp32, where the fp32 pipes have 72.
//
// What it takes, us (a few per cent more or less from one card to the next): 325,557 x 256 -> 128 fp32 forward 159 (floor 78, by
// products and by bytes alike; the library's product and bias on the fp32 pipes 585), input gradient 177 (467), weight gradient with the
// bias' 185 (641 and 203); 100,000 x 1024 -> 1024 forward 1232 (floor 763; 3858).  In bf16: 2.45 M x 128 -> 256, which bytes bound,
// forward 407 (floor 287; 283), input gradient 312 (300), weight gradient with the bias' 398 (312 and 492); 16,384 x 4096 -> 4096 forward
// 409 (floor 333; 343), input gradient 441 (331), weight gradient 517, with the bias' 900 (349 and 51).
//
// Operands lie in shared memory in the swizzled layout that the tensor core reads.  The streamed ones are masked and split on
// their way there.  The weight is laid out and split once a call by a kernel of its own, as the images of shared memory
// that bulk copies fetch.
#include <algorithm>

#include "cgnn_linear.cuh"

namespace cgnn {

static __device__ int g_linear_status = 0;

int linear_status(int *out) {
    const int zero = 0;
    CGNN_CUDA(cudaMemcpyFromSymbol(out, g_linear_status, sizeof(int)));
    CGNN_CUDA(cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int)));
    return CGNN_OK;
}

namespace {

constexpr int BM = 128;
constexpr int EPILOGUE_WARPS = 8, PRODUCER_WARPS = 8;
constexpr int PRODUCERS = PRODUCER_WARPS * 32;
constexpr int MMA_WARP = EPILOGUE_WARPS + PRODUCER_WARPS, COPY_WARP = MMA_WARP + 1;
constexpr int THREADS = (MMA_WARP + 4) * 32;
// Registers of a thread by warpgroup; a launch brings 96 a thread, and the five groups share that: 2 x 112 + 2 x 112 + 32 = 5 x 96.
constexpr int EPILOGUE_REGISTERS = 112, PRODUCER_REGISTERS = 112, OTHER_REGISTERS = 32;
constexpr int SMS = 148;
constexpr int TMEM_COLUMNS = 512;  // two buffers of 256
constexpr int PIECE = 16;          // columns that a warp of the epilogue takes at once

// Terms of 16-bit operands that an accumulator takes: its truncations lose 1e-7 of a sum of one sign for every sixteen, so 5e-5 of so
// many (half a step of fp16 is 4.9e-4; 300,000 terms in one accumulator were 2e-3 off).  Longer contractions add up in fp32
// in memory, a segment after the other (weight gradients without the bias' in bf16: 2.45 M x 128 -> 256 310 us, in one accumulator
// 292; 16,384 x 4096 -> 4096 496 and 470).
constexpr int LONGEST = 8192;

// A stage holds BK of the contraction: rows of BK 16-bit elements (FORWARD, INPUT), or BK rows of panels of 64 (WEIGHT).
//
// HBM wants 35 KB on their way to each multiprocessor.  16-bit operands are copied asynchronously to where the tensor core
// reads them, as many stages early as there are, or AHEAD where somebody looks at them on their way.  fp32 ones go through
// registers, by two groups of producers that take every other chunk: a warp's wait for one load is a wait for its latest, so that
// loads further ahead by the same warps did not help (325,557 x 256 -> 128 forward: 4 chunks ahead 180 us, 1 chunk 178,
// two groups 157; weight gradient: one group of four units a thread 197, two groups of eight 213).
template <typename T, int FORM, bool WHOLE>
struct Shape {
    static constexpr bool SPLIT = sizeof(T) == 4;
    static constexpr bool ASYNC = WHOLE && !SPLIT;
    static constexpr int PLANES = SPLIT ? 3 : 1;
    static constexpr int BN = SPLIT ? 128 : 256;
    static constexpr int BK = SPLIT || (FORM == WEIGHT && !WHOLE) ? 32 : 64;
    static constexpr int A_PLANE = BM * BK * 2, B_PLANE = BN * BK * 2;
    static constexpr int STAGE = PLANES * (A_PLANE + B_PLANE);
    static constexpr int STAGES = SPLIT || FORM != WEIGHT || WHOLE ? 4 : 7;
    static constexpr int AHEAD = 1;  // of a group's own chunks
    static constexpr int SEGMENT = (SPLIT ? 256 : LONGEST) / BK;  // chunks of BK that an accumulator takes
    static constexpr int GROUPS = SPLIT && FORM == WEIGHT ? 1 : 2, MEMBERS = PRODUCERS / GROUPS;  // producers that fill a stage
    static constexpr int A_UNITS = BM * BK / 8 / MEMBERS, B_UNITS = FORM == WEIGHT ? BN * BK / 8 / MEMBERS : 0;
    static constexpr int MASK_SLOT = ASYNC && FORM != FORWARD ? A_UNITS * MEMBERS : 0;  // a word of the mask for four units of a row
    static constexpr int STAGING = EPILOGUE_WARPS * 32 * (PIECE + 1) * 4;
    static constexpr int SUMS = FORM == WEIGHT ? PRODUCER_WARPS * BM * 8 : 0;  // of the columns
    static constexpr int SHARED = STAGES * (STAGE + MASK_SLOT) + STAGING + SUMS + 1024;
    static_assert(SHARED + (FORM == FORWARD ? 2048 : 512) <= 232448 && (SPLIT || 2 * (AHEAD + 1) <= STAGES), "a block has 227 KB");
};
// What does not depend on the way of the operands.
template <typename T, int FORM>
using Tile = Shape<T, FORM, true>;

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
    int out_whole, out_wide;      // rows of the output and the residual lie on vectors of 8 elements, of 32 bytes
    void *out;                    // [M, N] of T, or (WEIGHT of several splits) [splits, M, N] of fp32
    int partial;
    float *running;               // contractions of more than LONGEST, 16 bits: [M, N] (WEIGHT: of each split) of fp32
    int running_whole;            // its rows lie on vectors of 8
    double *column_sums;          // WEIGHT: [splits, M]
    float scale;
    Epilogue<T> epilogue;         // FORWARD
    int polls;
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
// What the warps of a block know of each other's waits.
struct Waits {
    int given_up;
    int computed;  // what `compute_again` has come through
    uint32_t again[EPILOGUE_WARPS][4];  // of a warp's item: rows with an element in that piece of columns that is to be computed again
};
// Waits for the phase of that parity; gives up after `polls`, or when another thread of the block has.  PATIENT: not while a warp is
// computing elements again, which the others may have to wait for.
template <bool PATIENT>
__device__ __forceinline__ bool barrier_wait(uint64_t *barrier, uint32_t parity, int polls, volatile Waits *waits) {
    [[maybe_unused]] int seen = 0;
    do {
        for (int i = 0; i < polls; ++i) {
            if (barrier_poll(barrier, parity)) return true;
            if (waits->given_up) return false;
        }
        if constexpr (PATIENT) {
            const int now = waits->computed;
            if (now == seen) break;
            seen = now;
        }
    } while (PATIENT);
    waits->given_up = 1;
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
// A matrix in shared memory, rows of ROW bytes (128 or 64) swizzled in groups of eight.  The lower word of its descriptor: its
// address, and the bytes between panels of 64 elements along m or n where those are contiguous.  The upper word is the same for all.
__device__ __forceinline__ uint32_t matrix_descriptor(uint32_t address, uint32_t leading) {
    return (address >> 4 & 0x3fff) | leading >> 4 << 16;
}
template <int ROW>
constexpr uint32_t MATRIX_UPPER = 8 * ROW >> 4 | 1u << 14 | (ROW == 128 ? 2u : 4u) << 29;
// fp32 accumulators; operands bf16 or fp16, contiguous along k or (along_mn) along m and n.
__host__ __device__ constexpr uint32_t product_descriptor(bool bf16, bool along_mn) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (along_mn ? 1u << 15 | 1u << 16 : 0u) | (uint32_t)(BM / 16) << 24;
}
template <uint32_t UPPER>
__device__ __forceinline__ void multiply(uint32_t accumulator, uint32_t a, uint32_t b, uint32_t descriptor, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}" ::"r"(accumulator),
        "r"(a), "r"(b), "r"(descriptor), "r"((uint32_t)add), "n"(UPPER)
        : "memory");
}
// True for one lane of the warp, the same every time.
__device__ __forceinline__ bool leader_of_warp() {
    uint32_t leads;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(leads));
    return leads != 0;
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
// Thirty-two columns of one accumulator.
__device__ __forceinline__ void tmem_load32(uint32_t address, float (&v)[2][16]) {
    uint32_t r[16], q[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : CGNN_SIXTEEN(r), CGNN_SIXTEEN(q)
        : "r"(address), "r"(address + 16)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[0][i] = __uint_as_float(r[i]), v[1][i] = __uint_as_float(q[i]);
}
// Eight columns, with the small products'.
__device__ __forceinline__ void tmem_load8(uint32_t address, float (&v)[8]) {
    uint32_t r[8], q[8];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%16];\n"
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%17];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]), "=&r"(q[0]), "=&r"(q[1]),
          "=&r"(q[2]), "=&r"(q[3]), "=&r"(q[4]), "=&r"(q[5]), "=&r"(q[6]), "=&r"(q[7])
        : "r"(address), "r"(address + 128)
        : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]) + __uint_as_float(q[i]);
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 16 bytes, of which the first `there` are copied and the others zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void *from, int there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}
// The barrier is told when this thread's copies up to here have arrived.
__device__ __forceinline__ void copies_report(uint64_t *barrier) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(shared_address(barrier)) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}
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
    // The first `left` elements, zeros behind them.
    __device__ __forceinline__ void load(const float *p, int left) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < left ? p[k] : 0.f;
    }
    __device__ __forceinline__ void load_whole(const float *p) {
        const float4 x = *reinterpret_cast<const float4 *>(p), y = *reinterpret_cast<const float4 *>(p + 4);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    }
    // All of them (on a boundary of 32 bytes), or zeros; without a branch.
    __device__ __forceinline__ void load_or_clear(const float *p, bool there) {
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.u32 p, %9, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n mov.b32 %2, 0;\n mov.b32 %3, 0;\n"
            " mov.b32 %4, 0;\n mov.b32 %5, 0;\n mov.b32 %6, 0;\n mov.b32 %7, 0;\n"
            " @p ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n}"
            : "=&f"(v[0]), "=&f"(v[1]), "=&f"(v[2]), "=&f"(v[3]), "=&f"(v[4]), "=&f"(v[5]), "=&f"(v[6]), "=&f"(v[7])
            : "l"(p), "r"((uint32_t)there));
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
                if (q < 2)  // (exact: what is left has the lower bits only)
                    rest = __ffma2_rn(make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u)), make_float2(-1.f, -1.f),
                                      rest);
            }
        }
    }
};
template <typename T>
struct Unit16 {
    uint4 v;
    __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const T *p, int left) {
        const uint16_t *const q = reinterpret_cast<const uint16_t *>(p);
        uint32_t *const w = &v.x;
#pragma unroll
        for (int k = 0; k < 8; k += 2)
            w[k / 2] = (k < left ? (uint32_t)q[k] : 0u) | (k + 1 < left ? (uint32_t)q[k + 1] : 0u) << 16;
    }
    __device__ __forceinline__ void load_whole(const T *p) { v = *reinterpret_cast<const uint4 *>(p); }
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

// Where a unit lies in a plane of shared memory: row r of ROW bytes, unit c of them.
template <int ROW>
__device__ __forceinline__ uint32_t place(int r, int c) {
    return (uint32_t)(r * ROW + ((ROW == 128 ? c ^ (r & 7) : c ^ (r >> 1 & 3)) << 4));
}

// ---------------------------------------------------------------------------------------------
// the weight as images of shared memory: [tile of BN][chunk of BK][plane][BN rows of BK]
// ---------------------------------------------------------------------------------------------
template <typename T, int FORM>
__global__ void __launch_bounds__(256) pack_kernel(const T *weight, int64_t in, int64_t N, int64_t K, int64_t chunks, uint8_t *packed,
                                                   int whole) {
    using S = Tile<T, FORM>;
    constexpr int UNITS = S::BK / 8;  // of a row
    const int64_t n_rows = (N + S::BN - 1) / S::BN * S::BN;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n_rows * chunks * UNITS) return;
    // neighbouring threads take neighbouring places in memory: units of a row, or (transposed) columns
    const int64_t n = FORM == FORWARD ? i / (chunks * UNITS) : i % n_rows, unit = FORM == FORWARD ? i % (chunks * UNITS) : i / n_rows;
    const int64_t k = unit * 8;
    Unit<T> u;
    u.clear();
    if (n < N && k < K) {
        if (FORM == FORWARD) {
            if (whole && k + 8 <= K) u.load_whole(weight + n * in + k);
            else u.load(weight + n * in + k, (int)min(K - k, (int64_t)8));
        } else {
            T v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k + j < K ? weight[(k + j) * in + n] : narrow<T>(0.f);
            u.load(v, 8);
        }
    }
    uint4 planes[S::PLANES];
    u.planes(planes);
    uint8_t *const image = packed + ((n / S::BN) * chunks + unit / UNITS) * S::PLANES * S::B_PLANE;
#pragma unroll
    for (int q = 0; q < S::PLANES; ++q)
        *reinterpret_cast<uint4 *>(image + q * S::B_PLANE + place<S::BK * 2>((int)(n % S::BN), (int)(unit % UNITS))) = planes[q];
}

// ---------------------------------------------------------------------------------------------
// the walk of a block
// ---------------------------------------------------------------------------------------------
struct Item {
    int64_t m0, n0, k0, k1;
    int split;
};
template <typename T, int FORM>
__device__ __forceinline__ Item item_of(const Tiles<T> &t, int item) {
    Item i;
    const int tiles = t.tiles_m * t.tiles_n;
    i.split = FORM == WEIGHT ? item / tiles : 0;
    const int tile = FORM == WEIGHT ? item % tiles : item;
    i.m0 = (int64_t)(tile / t.tiles_n) * BM;
    i.n0 = (int64_t)(tile % t.tiles_n) * Tile<T, FORM>::BN;
    i.k0 = i.split * t.k_per_item;
    i.k1 = min(t.K, i.k0 + t.k_per_item);
    return i;
}
template <typename T, int FORM, bool WHOLE>
__device__ __forceinline__ int chunks_of(const Tiles<T> &t, int item) {
    using S = Shape<T, FORM, WHOLE>;
    int64_t k = t.K;
    if (FORM == WEIGHT) {
        const int64_t k0 = item / (t.tiles_m * t.tiles_n) * t.k_per_item;
        k = min(k, k0 + t.k_per_item) - k0;
    }
    return (int)((k + S::BK - 1) / S::BK);
}

// Sixteen neighbouring elements of a row, on a boundary of 32 bytes (fp32, wide) or 16.
__device__ __forceinline__ void load16(const float *p, int left, bool, float (&y)[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.u32 p, %9, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n mov.b32 %2, 0;\n mov.b32 %3, 0;\n"
            " mov.b32 %4, 0;\n mov.b32 %5, 0;\n mov.b32 %6, 0;\n mov.b32 %7, 0;\n"
            " @p ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n}"
            : "=&f"(y[8 * h]), "=&f"(y[8 * h + 1]), "=&f"(y[8 * h + 2]), "=&f"(y[8 * h + 3]), "=&f"(y[8 * h + 4]), "=&f"(y[8 * h + 5]),
              "=&f"(y[8 * h + 6]), "=&f"(y[8 * h + 7])
            : "l"(p + 8 * h), "r"((uint32_t)(left > 8 * h)));
}
template <typename T>
__device__ __forceinline__ void load16(const T *p, int left, bool, float (&y)[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        Vec<T, 8> v = vec_zero<T, 8>();
        if (left > 8 * h) v = vec_load<T, 8>(p + 8 * h);
        float part[8];
        widen_all<T, 8>(v, part);
#pragma unroll
        for (int k = 0; k < 8; ++k) y[8 * h + k] = part[k];
    }
}
__device__ __forceinline__ void store16(float *p, int left, bool, const float (&y)[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (left > 8 * h)
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + 8 * h), "f"(y[8 * h]), "f"(y[8 * h + 1]),
                         "f"(y[8 * h + 2]), "f"(y[8 * h + 3]), "f"(y[8 * h + 4]), "f"(y[8 * h + 5]), "f"(y[8 * h + 6]), "f"(y[8 * h + 7])
                         : "memory");
}
template <typename T>
__device__ __forceinline__ void store16(T *p, int left, bool wide, const float (&y)[16]) {
    const Vec<T, 16> v = narrow_all<T, 16>(y);
    const uint32_t *const w = reinterpret_cast<const uint32_t *>(&v);
    if (wide) {  // a whole sector at once
        if (left > 0)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                         "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (left > 8 * h) *reinterpret_cast<uint4 *>(p + 8 * h) = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
    }
}

// What few warps come to stands in functions of its own: what all of them read again and again has to fit the instruction caches
// (2.45 M x 128 -> 256 bf16 forward with these and the dropout inside: 450 us,
// without 386).

// Rows of no whole vectors: what the lanes left in `staging` ([32][PIECE + 1]) by neighbouring lanes for neighbouring columns.
template <typename O>
__device__ __noinline__ void write_rows(const float *staging, O *out, int64_t N, int64_t m0, int64_t M, int64_t n) {
    const int lane = threadIdx.x & 31, k = lane % PIECE;
    O *to = out + (m0 + lane / PIECE) * N + n + k;
    const int rows = (int)min(M - m0 - lane / PIECE, (int64_t)32);
    if (n + k < N)
        for (int j = 0; j < PIECE; ++j, to += 2 * N)
            if (2 * j < rows) *to = narrow<O>(staging[(lane / PIECE + 2 * j) * (PIECE + 1) + k]);
}
template <typename T>
__device__ __noinline__ void read_row(float *staging, const T *row, int left) {
    for (int k = 0; k < PIECE; ++k) staging[k] = k < left ? widen(row[k]) : 0.f;
}
// Elements of a warp's 32 x 64 of an item computed again by fp32 arithmetic and written over: where an operand is infinite, no
// number or beyond bf16's range, its parts say nothing.  PIECE columns at once: of few rows one row after the other, its terms by all
// lanes (one infinity in an incoming gradient makes a row of the weight's gradient infinite, of as many terms as there are
// nodes); of more than 8 every lane its own.  (Not a function of its own: around a call the fp32 forward pass spilled registers, 191 us for 159.)
template <typename T, int FORM>
__device__ __forceinline__ void compute_again(const Tiles<T> &t, int item, Waits *waits) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Item i = item_of<T, FORM>(t, item);
    const int64_t m0 = i.m0 + (warp & 3) * 32, n0 = i.n0 + (warp >> 2) * (Tile<T, FORM>::BN / 2);
    for (int p = 0; p < Tile<T, FORM>::BN / 2 / PIECE; ++p) {
        uint32_t rows = waits->again[warp][p];
        __syncwarp();
        if (lane == 0) waits->again[warp][p] = 0;
        const int64_t n = n0 + p * PIECE;
        const int left = (int)min(t.N - n, (int64_t)PIECE);
        const bool own = __popc(rows) > 8;
        while (rows) {
            const int64_t m = m0 + (own ? lane : __ffs(rows) - 1);
            const bool mine = !own || (rows >> lane & 1);
            float sum[PIECE];
#pragma unroll
            for (int c = 0; c < PIECE; ++c) sum[c] = 0.f;
#pragma unroll 1
            for (int64_t first = i.k0; first < i.k1; first += own ? 1 : 32) {
                const int64_t k = first + (own ? 0 : lane);
                bool lost = false;  // every column's sum is no number any more, and stays none
                if (k < i.k1 && mine) {
                    const int64_t row = FORM == WEIGHT ? k : m, column = FORM == WEIGHT ? m : k;
                    const T *const from = FORM == FORWARD ? t.b + n * t.b_stride + k : t.b + k * t.b_stride + n;
                    float a = widen(t.a[row * t.a_stride + column]), b[PIECE];
#pragma unroll
                    for (int c = 0; c < PIECE; ++c) b[c] = c < left ? widen(from[FORM == FORWARD ? c * t.b_stride : c]) : 0.f;
                    if (FORM != FORWARD && t.mask != nullptr && !(t.mask[row * t.mask_pitch + column / 8] >> (column % 8) & 1)) a = 0.f;
                    lost = true;
#pragma unroll
                    for (int c = 0; c < PIECE; ++c) {
                        sum[c] = fmaf(a, b[c], sum[c]);
                        lost = lost && (sum[c] != sum[c] || c >= left);
                    }
                }
                if (own ? __all_sync(0xffffffffu, lost || !mine) : __any_sync(0xffffffffu, lost)) break;
                if (lane == 0 && first % 1024 < 32) atomicAdd(&waits->computed, 1);
            }
            if (!own) {  // every lane's sums to the first lane's: half of the columns each time, with the other half's lane
#pragma unroll
                for (int half = PIECE / 2; half > 0; half >>= 1)
#pragma unroll
                    for (int c = 0; c < half; ++c) {
                        const bool upper = lane & (2 * half);
                        const float kept = upper ? sum[c + half] : sum[c], given = upper ? sum[c] : sum[c + half];
                        sum[c] = kept + __shfl_xor_sync(0xffffffffu, given, 2 * half);
                    }
                sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 1);
                sum[0] = __shfl_sync(0xffffffffu, sum[0], 2 * lane & 31);  // column n + lane
            }
            uint32_t bits = 0;
            [[maybe_unused]] Philox words(FORM == FORWARD ? t.epilogue.drop.key() : 0);
#pragma unroll
            for (int c = 0; c < PIECE; ++c)
                if (own ? mine && c < left : c == 0 && lane < left) {
                    const int64_t column = n + (own ? c : lane);
                    float y = sum[c];
                    if constexpr (FORM == FORWARD) bits |= (uint32_t)t.epilogue.element(y, m, column, words) << c;
                    else if (!(FORM == WEIGHT && t.partial)) y *= t.scale;
                    if (FORM == WEIGHT && t.partial) static_cast<float *>(t.out)[(i.split * t.M + m) * t.N + column] = y;
                    else static_cast<T *>(t.out)[m * t.N + column] = narrow<T>(y);
                }
            if constexpr (FORM == FORWARD)
                if (t.epilogue.mask != nullptr) {
                    const uint32_t of_row = __ballot_sync(0xffffffffu, bits & 1);
                    if (own ? mine : lane == 0)
                        *reinterpret_cast<uint16_t *>(t.epilogue.mask + m * t.epilogue.mask_pitch + n / 8) = (uint16_t)(own ? bits : of_row);
                }
            rows = own ? 0 : rows & (rows - 1);
        }
    }
    if (lane == 0) atomicAdd(&waits->computed, 1);
}

// The epilogue of one warp: 32 rows, a row a lane as they lie in the accumulators, PIECE columns at a time.  Rows of whole vectors are
// read and written by their lane, a sector or two at once; of others the results go through shared memory, from where
// neighbouring lanes take neighbouring columns.
template <typename T, int FORM, bool DROP>
struct Finish {
    const Tiles<T> &t;
    float *const staging;  // [32][PIECE + 1]
    const float *const bias;
    const int lane;
    Waits *const waits;
    Philox words;
    // of the present item
    int64_t m, n0, first;  // the lane's row, the first column, and the output's element that they are
    int columns;           // from there on, none for a row that is not there
    uint64_t passed;       // a bit for each column, 64 a turn

    __device__ __forceinline__ Finish(const Tiles<T> &t_, float *staging_, const float *bias_, int lane_, Waits *waits_)
        : t(t_), staging(staging_), bias(bias_), lane(lane_), waits(waits_),
          words(DROP ? t_.epilogue.drop.key() : 0) {}

    __device__ __forceinline__ void begin(int64_t m0, int64_t n0_) {
        m = m0 + lane;
        n0 = n0_;
        first = m * t.N + n0;
        columns = m < t.M ? (int)max((int64_t)0, min(t.N - n0, (int64_t)1024)) : 0;
        passed = 0;
    }

    // What the rest of the forward pass adds, on its way while the accumulators are read.
    __device__ __forceinline__ void fetch(int c, float (&added)[PIECE]) {
        if (FORM == FORWARD && t.epilogue.residual != nullptr) {
            const T *const r = t.epilogue.residual + first + c;
            const int left = columns - c;
            if (t.out_whole) {
                load16(r, left, t.out_wide, added);
            } else {
                float *const row = staging + lane * (PIECE + 1);
                read_row(row, r, left);
#pragma unroll
                for (int k = 0; k < PIECE; ++k) added[k] = row[k];
            }
        }
    }

    // Columns c .. c + PIECE of the item.
    __device__ __forceinline__ void piece(float (&y)[PIECE], const float (&added)[PIECE], const Item &i, int c, bool alive) {
        const int left = columns - c;
        if constexpr (Tile<T, FORM>::SPLIT) {
            float none = 0.f;  // zero unless one of them is no finite number
#pragma unroll
            for (int k = 0; k < PIECE; ++k) none = fmaf(y[k], 0.f, none);
            if (none != 0.f && left > 0 && alive) atomicOr(&waits->again[threadIdx.x >> 5][c / PIECE], 1u << lane);
        }
        if (!alive) {
#pragma unroll
            for (int k = 0; k < PIECE; ++k) y[k] = __uint_as_float(0x7fffffffu);
        }
        if constexpr (FORM == FORWARD) {
            uint32_t through = 0xffff;
            if (t.epilogue.bias != nullptr) {
#pragma unroll
                for (int k = 0; k < PIECE; k += 4) {
                    const float4 b = *reinterpret_cast<const float4 *>(bias + c + k);
                    y[k] += b.x, y[k + 1] += b.y, y[k + 2] += b.z, y[k + 3] += b.w;
                }
            }
            if (t.epilogue.relu) {
#pragma unroll
                for (int k = 0; k < PIECE; ++k)
                    if (y[k] <= 0.f) {  // (a NaN stays one)
                        y[k] = 0.f;
                        through &= ~(1u << k);
                    }
            }
            if constexpr (DROP) {
                const uint32_t threshold = t.epilogue.drop.threshold;
                const float scale = (float)t.epilogue.drop.scale;
                const uint64_t block = (uint64_t)(first + c) >> 2;
                const int ahead = (int)((first + c) & 3);  // not zero: the rows do not begin with a block of words
                uint4 q = words(block);
#pragma unroll
                for (int b = 0; b < PIECE / 4; ++b) {
                    uint32_t w[4] = {q.x, q.y, q.z, q.w};
                    if (ahead || b + 1 < PIECE / 4) {
                        const uint4 r = words(block + b + 1);
                        const uint32_t all[8] = {w[0], w[1], w[2], w[3], r.x, r.y, r.z, r.w};
                        if (ahead)
#pragma unroll
                            for (int k = 0; k < 4; ++k) w[k] = ahead == 1 ? all[k + 1] : ahead == 2 ? all[k + 2] : all[k + 3];
                        q = r;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool kept = w[k] >= threshold;
                        y[4 * b + k] = kept ? y[4 * b + k] * scale : 0.f;
                        if (!kept) through &= ~(1u << (4 * b + k));
                    }
                }
            }
            if (t.epilogue.residual != nullptr) {
#pragma unroll
                for (int k = 0; k < PIECE; ++k) y[k] += added[k];
            }
            if (t.epilogue.mask != nullptr) {
                if (left < PIECE) through &= left > 0 ? (1u << left) - 1u : 0u;
                passed |= (uint64_t)through << (c % 64);
                if (c % 64 + PIECE == 64 || c + PIECE >= columns) {  // (words of 64 columns, the last one whatever is left)
                    if (left > 0)
                        *reinterpret_cast<uint64_t *>(t.epilogue.mask + m * t.epilogue.mask_pitch + (n0 + c / 64 * 64) / 8) = passed;
                    passed = 0;
                }
            }
        } else if (!(FORM == WEIGHT && t.partial)) {
            const float scale = t.scale;
#pragma unroll
            for (int k = 0; k < PIECE; ++k) y[k] *= scale;
        }
        if (FORM == WEIGHT && t.partial) write(static_cast<float *>(t.out) + i.split * t.M * t.N, c, left, y);
        else write(static_cast<T *>(t.out), c, left, y);
    }
    // Columns c .. c + PIECE of the item's sum over the segments before, added or left for the next.  (A lane comes back to its own.)
    __device__ __forceinline__ void add_running(const float *sums, int c, float (&x)[PIECE]) {
        const float *const p = sums + first + c;
        const int left = columns - c;
        float before[PIECE];
        if (t.running_whole) {
            load16(p, left, true, before);
        } else {
#pragma unroll
            for (int k = 0; k < PIECE; ++k) before[k] = k < left ? p[k] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < PIECE; ++k) x[k] += before[k];
    }
    __device__ __forceinline__ void leave_running(float *sums, int c, const float (&x)[PIECE]) {
        float *const p = sums + first + c;
        const int left = columns - c;
        if (t.running_whole) {
            store16(p, left, true, x);
        } else {
#pragma unroll
            for (int k = 0; k < PIECE; ++k)
                if (k < left) p[k] = x[k];
        }
    }
    template <typename O>
    __device__ __forceinline__ void write(O *out, int c, int left, const float (&y)[PIECE]) {
        if (t.out_whole) {
            store16(out + first + c, left, t.out_wide, y);
        } else {
#pragma unroll
            for (int k = 0; k < PIECE; ++k) staging[lane * (PIECE + 1) + k] = y[k];
            __syncwarp();
            write_rows(staging, out, t.N, m - lane, t.M, n0 + c);
            __syncwarp();
        }
    }
};

// Eight LongSums, two at a time.
struct LongSums {
    float2 high[4] = {}, low[4] = {};
    __device__ __forceinline__ static float2 difference(float2 a, float2 b) { return __ffma2_rn(b, make_float2(-1.f, -1.f), a); }
    __device__ __forceinline__ void add(const float (&x)[8]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 v = make_float2(x[2 * k], x[2 * k + 1]), s = __fadd2_rn(high[k], v), part = difference(s, high[k]);
            low[k] = __fadd2_rn(low[k], __fadd2_rn(difference(high[k], difference(s, part)), difference(v, part)));
            high[k] = s;
        }
    }
    __device__ __forceinline__ double value(int k) const {
        const float h = k % 2 ? high[k / 2].y : high[k / 2].x;
        return isfinite(h) ? (double)h + (double)(k % 2 ? low[k / 2].y : low[k / 2].x) : (double)h;
    }
};

// The units of a producer: a thread has the same place in every chunk of its group.  WHOLE: rows lie on vectors of 8 elements;
// units of other rows are loaded an element at a time.
template <typename T, int FORM, bool WHOLE>
struct Producer {
    using S = Shape<T, FORM, WHOLE>;
    static constexpr int BK = S::BK, MEMBERS = S::MEMBERS;
    // Units across a row of A and B, and rows of a turn of the group.
    static constexpr int A_ACROSS = FORM == WEIGHT ? BM / 8 : BK / 8, A_DOWN = MEMBERS / A_ACROSS;
    [[maybe_unused]] static constexpr int B_ACROSS = S::BN / 8, B_DOWN = MEMBERS / B_ACROSS;
    const Tiles<T> &t;
    const int p;
    const bool masked;
    const int64_t a_step, b_step, mask_step;  // elements (bytes of the mask) between the rows of two units
    // where the next chunk is read
    int item, chunk, chunks;
    const T *a, *b;
    const uint8_t *mask;
    int rows, b_rows;   // from this thread's first on
    int a_left, b_left; // elements of a row from this thread's first on

    __device__ __forceinline__ Producer(const Tiles<T> &t_, int p_)
        : t(t_), p(p_), masked(FORM != FORWARD && t_.mask != nullptr), a_step(A_DOWN * t_.a_stride), b_step(B_DOWN * t_.b_stride),
          mask_step(A_DOWN * t_.mask_pitch), item(blockIdx.x), chunk(0), b(nullptr), mask(nullptr) {
        begin();
    }
    __device__ __forceinline__ static int clamped(int64_t n) { return (int)max((int64_t)0, min(n, (int64_t)1 << 28)); }
    __device__ __forceinline__ bool more() const { return item < t.items; }
    __device__ __forceinline__ void begin() {
        if (item >= t.items) return;
        const Item i = item_of<T, FORM>(t, item);
        chunk = 0;
        chunks = chunks_of<T, FORM, WHOLE>(t, item);
        if constexpr (FORM == WEIGHT) {
            const int64_t row = i.k0 + p / A_ACROSS, column = i.m0 + p % A_ACROSS * 8;
            const int64_t b_row = i.k0 + p / B_ACROSS, b_column = i.n0 + p % B_ACROSS * 8;
            a = t.a + row * t.a_stride + column;
            b = t.b + b_row * t.b_stride + b_column;
            mask = t.mask + row * t.mask_pitch + column / 32 * 4;
            rows = clamped(i.k1 - row);
            b_rows = clamped(i.k1 - b_row);
            a_left = clamped(t.M - column);
            b_left = clamped(t.N - b_column);
        } else {
            const int64_t row = i.m0 + p / A_ACROSS, column = p % A_ACROSS * 8;
            a = t.a + row * t.a_stride + column;
            mask = t.mask + row * t.mask_pitch + column / 32 * 4;
            rows = clamped(t.M - row);
            a_left = clamped(t.K - column);
        }
    }
    __device__ __forceinline__ void next() {
        if (++chunk == chunks) {
            item += gridDim.x;
            begin();
        } else if constexpr (FORM == WEIGHT) {
            a += (BK / A_DOWN) * a_step;
            b += (BK / B_DOWN) * b_step;
            mask += (BK / A_DOWN) * mask_step;
            rows -= BK;
            b_rows -= BK;
        } else {
            a += BK;
            mask += BK / 8;
            a_left -= BK;
        }
    }
    // The group's next chunk.
    __device__ __forceinline__ void next_own() {
        next();
        if (S::GROUPS == 2 && more()) next();
    }
    // Where a unit of A or B lies in a plane.
    __device__ __forceinline__ uint32_t a_place(int u) const {
        return FORM == WEIGHT ? p % A_ACROSS / 8 * (BK * 128) + place<128>(p / A_ACROSS + u * A_DOWN, p % 8)
                              : place<BK * 2>(p / A_ACROSS + u * A_DOWN, p % A_ACROSS);
    }
    __device__ __forceinline__ uint32_t b_place(int u) const {
        return p % B_ACROSS / 8 * (BK * 128) + place<128>(p / B_ACROSS + u * B_DOWN, p % 8);
    }
    // The bits of a unit of A in its word of the mask (a unit's column is a multiple of 8).
    __device__ __forceinline__ uint32_t bits_of(uint32_t word) const { return word >> (p % 4 * 8); }

    // The next chunk on its way to its stage (16 bits), the mask's words to theirs.
    __device__ __forceinline__ void issue(uint32_t stage, uint32_t masks) {
        // (Instructions bound this: chunks whose rows are all there, nearly all, go without a look at each unit.)
        constexpr int WHOLE_ROWS = FORM == WEIGHT ? BK : BM;
        const int bytes = min(max(0, a_left) * (int)sizeof(T), 16);
        if (rows >= WHOLE_ROWS) {
            const T *from = bytes ? a : t.a;
            const int64_t down = bytes ? a_step : 0;
#pragma unroll
            for (int u = 0; u < S::A_UNITS; ++u, from += down) copy16(stage + a_place(u), from, bytes);
            if constexpr (FORM != FORWARD) {
                const uint8_t *word = bytes ? mask : t.mask;
                const int64_t word_down = bytes ? mask_step : 0;
                if (masked && p % 4 == 0)
#pragma unroll
                    for (int u = 0; u < S::A_UNITS; ++u, word += word_down) copy4(masks + u * MEMBERS + p, word, bytes != 0);
            }
        } else {
#pragma unroll 1
            for (int u = 0; u < S::A_UNITS; ++u) {
                const int there = u * A_DOWN < rows ? bytes : 0;
                copy16(stage + a_place(u), there ? a + u * a_step : t.a, there);
                if constexpr (FORM != FORWARD)
                    if (masked && p % 4 == 0) copy4(masks + u * MEMBERS + p, there ? mask + u * mask_step : t.mask, there != 0);
            }
        }
        if constexpr (FORM == WEIGHT) {
            const int b_bytes = min(max(0, b_left) * (int)sizeof(T), 16);
            if (b_rows >= WHOLE_ROWS) {
                const T *from = b_bytes ? b : t.b;
                const int64_t down = b_bytes ? b_step : 0;
#pragma unroll
                for (int u = 0; u < S::B_UNITS; ++u, from += down) copy16(stage + S::A_PLANE + b_place(u), from, b_bytes);
            } else {
#pragma unroll 1
                for (int u = 0; u < S::B_UNITS; ++u) {
                    const int there = u * B_DOWN < b_rows ? b_bytes : 0;
                    copy16(stage + S::A_PLANE + b_place(u), there ? b + u * b_step : t.b, there);
                }
            }
        }
        next_own();
    }
    // The next chunk of the group by loads.
    __device__ __forceinline__ void load(Unit<T> (&x)[S::A_UNITS + S::B_UNITS], uint32_t (&keep)[S::A_UNITS]) {
        if (!more()) return;
#pragma unroll
        for (int u = 0; u < S::A_UNITS; ++u) {
            const int left = u * A_DOWN < rows ? a_left : 0;
            if constexpr (WHOLE && S::SPLIT) x[u].load_or_clear(a + u * a_step, left > 0);
            else x[u].load(a + u * a_step, left);
        }
        if constexpr (FORM != FORWARD) {
            if (masked)
#pragma unroll
                for (int u = 0; u < S::A_UNITS; ++u)
                    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %2, 0;\n mov.b32 %0, 0;\n @p ld.global.b32 %0, [%1];\n}"
                                 : "=&r"(keep[u])
                                 : "l"(mask + u * mask_step), "r"((uint32_t)(u * A_DOWN < rows && a_left > 0)));
        }
#pragma unroll
        for (int u = 0; u < S::B_UNITS; ++u) {
            const int left = u * B_DOWN < b_rows ? b_left : 0;
            if constexpr (WHOLE && S::SPLIT) x[S::A_UNITS + u].load_or_clear(b + u * b_step, left > 0);
            else x[S::A_UNITS + u].load(b + u * b_step, left);
        }
        next_own();
    }
    // (Of the 16-bit types eight rows in fp32 first, which lose nothing that their result would keep.)
    __device__ __forceinline__ void add_columns(const Unit<T> (&x)[S::A_UNITS + S::B_UNITS], LongSums &columns) const {
        if constexpr (S::SPLIT) {
#pragma unroll
            for (int u = 0; u < S::A_UNITS; ++u) columns.add(x[u].v);
        } else {
            float sum[8];
#pragma unroll
            for (int u = 0; u < S::A_UNITS; ++u)
#pragma unroll
                for (int k = 0; k < 8; ++k) sum[k] = u == 0 ? x[u].value(k) : sum[k] + x[u].value(k);
            columns.add(sum);
        }
    }
    // Units to their planes in a stage.
    __device__ __forceinline__ void store(Unit<T> (&x)[S::A_UNITS + S::B_UNITS], const uint32_t (&keep)[S::A_UNITS], uint32_t stage,
                                          LongSums &columns) const {
        if constexpr (FORM != FORWARD) {
            if (masked)
#pragma unroll
                for (int u = 0; u < S::A_UNITS; ++u) x[u].keep(bits_of(keep[u]));
        }
        if constexpr (FORM == WEIGHT) {
            if (t.column_sums != nullptr) add_columns(x, columns);
        }
#pragma unroll
        for (int u = 0; u < S::A_UNITS; ++u) {
            uint4 planes[S::PLANES];
            x[u].planes(planes);
#pragma unroll
            for (int q = 0; q < S::PLANES; ++q) store_shared(stage + q * S::A_PLANE + a_place(u), planes[q]);
        }
#pragma unroll
        for (int u = 0; u < S::B_UNITS; ++u) {
            uint4 planes[S::PLANES];
            x[S::A_UNITS + u].planes(planes);
#pragma unroll
            for (int q = 0; q < S::PLANES; ++q) store_shared(stage + S::PLANES * S::A_PLANE + q * S::B_PLANE + b_place(u), planes[q]);
        }
    }
    // 16-bit units of A that have arrived in their stage: those of the mask go, and the others are added up.
    __device__ __forceinline__ void mend(uint8_t *stage, const uint8_t *masks, LongSums &columns) const {
        if constexpr (FORM != FORWARD) {
            const bool summed = FORM == WEIGHT && t.column_sums != nullptr;
            if (!masked && !summed) return;
            __syncwarp();  // a word of the mask was copied by one of four
            Unit<T> x[S::A_UNITS + S::B_UNITS];
#pragma unroll
            for (int u = 0; u < S::A_UNITS; ++u) {
                T *const at = reinterpret_cast<T *>(stage + a_place(u));
                x[u].load_whole(at);
                if (masked) {
                    x[u].keep(bits_of(*reinterpret_cast<const uint32_t *>(masks + u * MEMBERS + p / 4 * 4)));
                    uint4 planes[S::PLANES];
                    x[u].planes(planes);
                    store_shared(shared_address(at), planes[0]);
                }
            }
            if (summed) add_columns(x, columns);
        }
    }
};

// MANY: contractions of more than one segment: in fp32 their sums take registers that the others keep.  DROP: a forward pass with
// dropout, whose instructions the others do without (they are read again for every sixteen columns).
template <typename T, int FORM, bool WHOLE, bool MANY, bool DROP>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ Tiles<T> t) {
    using S = Shape<T, FORM, WHOLE>;
    constexpr int BN = S::BN, BK = S::BK, STAGES = S::STAGES, PLANES = S::PLANES;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[STAGES], empty[STAGES], sums_full[2], sums_empty[2], drained;
    __shared__ uint32_t tmem_base;
    __shared__ Waits waits;
    __shared__ __align__(16) float bias_of_tile[2][BN / 2];
    uint8_t *const stages = raw + (1024 - shared_address(raw) % 1024) % 1024;  // groups of eight swizzled rows lie on 1024 bytes
    [[maybe_unused]] uint8_t *const masks = stages + STAGES * S::STAGE;
    float *const staging = reinterpret_cast<float *>(masks + STAGES * S::MASK_SLOT);
    [[maybe_unused]] double *const column_parts = reinterpret_cast<double *>(staging + S::STAGING / 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // 16-bit operands that nobody looks at on their way: their copies report to the barriers themselves, each thread's.
    const bool direct = S::ASYNC && (FORM == FORWARD || t.mask == nullptr) && (FORM != WEIGHT || t.column_sums == nullptr);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            // (the copies of the weight's images report to the same barrier as whatever fills the rest of the stage)
            barrier_init(&full[s], (direct ? S::MEMBERS : S::MEMBERS / 32) + (FORM == WEIGHT ? 0 : 1));
            barrier_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            barrier_init(&sums_full[b], 1);
            barrier_init(&sums_empty[b], EPILOGUE_WARPS);
        }
        barrier_init(&drained, 1);
        waits.given_up = waits.computed = 0;
        for (int k = 0; k < EPILOGUE_WARPS * 4; ++k) waits.again[k / 4][k % 4] = 0;
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(EPILOGUE_REGISTERS));
        constexpr int COLUMNS = BN / 2;  // of a warp's half of the tile
        // Read from the accumulators at once.  (Two pieces make two copies of what follows, which costs more than it gives where that
        // is much: 2.45 M x 128 -> 256 bf16 forward 712 us for 450, input gradient 314 for 330.)
        constexpr int TURN = S::SPLIT || FORM == FORWARD ? PIECE : 2 * PIECE;
        const int quarter = warp & 3, half = warp >> 2;
        Finish<T, FORM, DROP> finish(t, staging + warp * 32 * (PIECE + 1), bias_of_tile[half], lane, &waits);
        uint32_t segment = 0;
        [[maybe_unused]] int64_t bias_n0 = -1;  // whose bias is there
        bool alive = true;  // A warp that gave up a wait has lost count: it takes nothing and releases nothing from then on.
        for (int item = blockIdx.x; item < t.items; item += gridDim.x) {
            const Item i = item_of<T, FORM>(t, item);
            const int64_t m0 = i.m0 + quarter * 32, n0 = i.n0 + half * COLUMNS;
            if (FORM == FORWARD && t.epilogue.bias != nullptr && n0 != bias_n0) {
                // the half's columns, by the four warps of the half
                bias_n0 = n0;
                asm volatile("bar.sync %0, %1;" ::"r"(1 + half), "n"(EPILOGUE_WARPS / 2 * 32) : "memory");
                for (int c = quarter * 32 + lane; c < COLUMNS; c += EPILOGUE_WARPS / 2 * 32)
                    bias_of_tile[half][c] = n0 + c < t.N ? widen(t.epilogue.bias[n0 + c]) : 0.f;
                asm volatile("bar.sync %0, %1;" ::"r"(1 + half), "n"(EPILOGUE_WARPS / 2 * 32) : "memory");
            }
            if (FORM == FORWARD && t.epilogue.residual != nullptr && m0 + lane < t.M) {  // on its way while the products are formed
                const int64_t last = min(n0 + COLUMNS, t.N);
                for (int64_t n = n0; n < last; n += 128 / (int)sizeof(T))
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(t.epilogue.residual + (m0 + lane) * t.N + n));
            }
            const uint32_t rows = tmem + ((uint32_t)(quarter * 32) << 16) + half * COLUMNS;
            const int pieces_end = m0 < t.M ? (int)min((int64_t)COLUMNS, t.N - n0) : 0;  // (the same for the warp)
            finish.begin(m0, n0);
            const auto await = [&] {
                const uint32_t buffer = segment & 1;
                if (alive) alive = __all_sync(0xffffffffu, barrier_wait<S::SPLIT>(&sums_full[buffer], segment >> 1 & 1, polls, &waits));
                fence_after();
                return buffer;
            };
            const auto release = [&](uint32_t buffer) {
                fence_before();
                __syncwarp();
                if (alive && lane == 0) barrier_arrive(&sums_empty[buffer]);
                ++segment;
            };
            int before = 0;  // segments ahead of the last
            if constexpr (MANY) before = (chunks_of<T, FORM, WHOLE>(t, item) - 1) / S::SEGMENT;
            if constexpr (MANY && !S::SPLIT) {
                float *const running = t.running + (FORM == WEIGHT ? i.split * t.M * t.N : 0);
                for (int s = 0; s <= before; ++s) {
                    const uint32_t buffer = await();
#pragma unroll 1
                    for (int c = 0; c < COLUMNS; c += PIECE) {
                        float x[PIECE], added[PIECE];
                        if (s == before && c < pieces_end) finish.fetch(c, added);
                        if (alive) tmem_load16<false>(rows + buffer * 256 + c, x);
                        if (c + PIECE == COLUMNS) release(buffer);
                        if (c >= pieces_end) continue;
                        if (s > 0) finish.add_running(running, c, x);
                        if (s < before) finish.leave_running(running, c, x);
                        else finish.piece(x, added, i, c, alive);
                    }
                }
            } else if (before == 0) {
                const uint32_t buffer = await();
#pragma unroll 1
                for (int c = 0; c < COLUMNS; c += TURN) {
                    float x[TURN / PIECE][PIECE], added[TURN / PIECE][PIECE];
#pragma unroll
                    for (int q = 0; q < TURN / PIECE; ++q)
                        if (c + q * PIECE < pieces_end) finish.fetch(c + q * PIECE, added[q]);
                    if (alive) {
                        if constexpr (TURN == PIECE) tmem_load16<S::SPLIT>(rows + buffer * 256 + c, x[0]);
                        else tmem_load32(rows + buffer * 256 + c, x);
                    }
                    if (c + TURN == COLUMNS) release(buffer);
#pragma unroll
                    for (int q = 0; q < TURN / PIECE; ++q)
                        if (c + q * PIECE < pieces_end) finish.piece(x[q], added[q], i, c + q * PIECE, alive);
                }
            } else if constexpr (MANY) {
                float sum[COLUMNS];
#pragma unroll
                for (int c = 0; c < COLUMNS; ++c) sum[c] = 0.f;
                for (; before >= 0; --before) {
                    const uint32_t buffer = await();
                    if (alive)
#pragma unroll
                        for (int c = 0; c < COLUMNS; c += 8) {
                            float part[8];
                            tmem_load8(rows + buffer * 256 + c, part);
#pragma unroll
                            for (int k = 0; k < 8; ++k) sum[c + k] += part[k];
                        }
                    release(buffer);
                }
#pragma unroll 1
                for (int c = 0; c < COLUMNS; c += PIECE) {  // (the sums move up, so that one copy of what follows is enough)
                    float x[PIECE], added[PIECE];
                    if (c < pieces_end) finish.fetch(c, added);
#pragma unroll
                    for (int k = 0; k < PIECE; ++k) x[k] = sum[k];
#pragma unroll
                    for (int k = 0; k < COLUMNS - PIECE; ++k) sum[k] = sum[k + PIECE];
                    if (c < pieces_end) finish.piece(x, added, i, c, alive);
                }
            }
            if constexpr (S::SPLIT) {  // (the accumulators have gone back already)
                static_assert(COLUMNS / PIECE == 4, "an item's pieces have a word each");
                __syncwarp();
                if (__any_sync(0xffffffffu, waits.again[warp][lane & 3] != 0)) compute_again<T, FORM>(t, item, &waits);
            }
        }
    } else if (warp < MMA_WARP) {
        // ------------------------------------------------------------------ operands to shared memory
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PRODUCER_REGISTERS));
        const int group = (threadIdx.x - EPILOGUE_WARPS * 32) / S::MEMBERS, p = (threadIdx.x - EPILOGUE_WARPS * 32) % S::MEMBERS;
        LongSums columns;
        Producer<T, FORM, WHOLE> ahead(t, p);
        if (group == 1 && ahead.more()) ahead.next();
        uint32_t s = group, parity = 1;  // of the stage that the group fills next
        bool alive = true;
        int item = blockIdx.x, chunk = 0, chunks = chunks_of<T, FORM, WHOLE>(t, item);
        const auto await = [&] {
            if (alive) alive = __all_sync(0xffffffffu, barrier_wait<S::SPLIT>(&empty[s], parity, polls, &waits));
        };
        const auto filled = [&](uint32_t stage) {
            fence_to_async();
            __syncwarp();
            if (lane == 0) barrier_arrive(&full[stage]);
        };
        const auto step = [&] {
            s += S::GROUPS;
            if (s >= STAGES) s -= STAGES, parity ^= 1;
        };
        // A chunk of the present item is done.  (To the end of all items whatever happens: the barriers here want every thread.)
        const auto done = [&] {
            if (++chunk < chunks) return;
            if (FORM == WEIGHT && t.column_sums != nullptr) {
                const Item i = item_of<T, FORM>(t, item);
                if (i.n0 == 0) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {  // (a warp's halves have the same columns)
                        double sum = columns.value(k);
                        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                        if (lane < 16) column_parts[(warp - EPILOGUE_WARPS) * BM + lane * 8 + k] = sum;
                    }
                    asm volatile("bar.sync 3, %0;" ::"n"(PRODUCERS) : "memory");
                    if (group == 0 && p < BM && i.m0 + p < t.M) {
                        double total = 0.0;
#pragma unroll
                        for (int r = 0; r < PRODUCER_WARPS; ++r) total += column_parts[r * BM + p];
                        if (*(volatile int *)&waits.given_up) total = __longlong_as_double(0x7fffffffffffffffll);
                        t.column_sums[i.split * t.M + i.m0 + p] = total;
                    }
                    asm volatile("bar.sync 3, %0;" ::"n"(PRODUCERS) : "memory");
                }
                columns = LongSums();
            }
            chunk = 0;
            item += gridDim.x;
            if (FORM == WEIGHT && item < t.items) chunks = chunks_of<T, FORM, WHOLE>(t, item);
        };
        if constexpr (S::ASYNC) {
            if (direct) {
                while (ahead.more() && alive) {
                    await();
                    if (alive) {
                        ahead.issue(shared_address(stages) + s * S::STAGE, shared_address(masks) + s * S::MASK_SLOT);
                        copies_report(&full[s]);
                    }
                    step();
                }
            } else {
                const auto issue = [&] {
                    if (ahead.more() && alive) {
                        await();
                        if (alive) ahead.issue(shared_address(stages) + s * S::STAGE, shared_address(masks) + s * S::MASK_SLOT);
                        step();
                    }
                    copies_end();
                };
#pragma unroll
                for (int d = 0; d < S::AHEAD; ++d) issue();
                uint32_t arrived = group;  // the stage of the first chunk on its way
                int turn = 0;              // of the group whose chunk it is
                while (item < t.items) {
                    if (turn == group) {
                        issue();
                        copies_wait<S::AHEAD>();
                        if (alive) {
                            ahead.mend(stages + arrived * S::STAGE, masks + arrived * S::MASK_SLOT, columns);
                            filled(arrived);
                        }
                        arrived += S::GROUPS;
                        if (arrived >= STAGES) arrived -= STAGES;
                    }
                    turn ^= 1;
                    done();
                }
            }
            copies_wait<0>();
        } else {
            Unit<T> x[S::A_UNITS + S::B_UNITS];
            uint32_t keep[S::A_UNITS];
            ahead.load(x, keep);
            int turn = 0;
            while (item < t.items) {
                if (turn == group) {
                    await();
                    if (alive) {
                        ahead.store(x, keep, shared_address(stages) + s * S::STAGE, columns);
                        filled(s);
                        ahead.load(x, keep);
                    }
                    step();
                }
                if (S::GROUPS == 2) turn ^= 1;
                done();
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGISTERS));
        if (warp == MMA_WARP) {
            // -------------------------------------------------------------- products
            // (the whole warp walks, so that what an instruction takes lies in the registers that a warp shares; one lane issues)
            constexpr bool ALONG_MN = FORM == WEIGHT;
            constexpr uint32_t base = product_descriptor(sizeof(T) == 4 || __is_same(T, __nv_bfloat16), ALONG_MN);
            constexpr uint32_t UPPER = MATRIX_UPPER<ALONG_MN ? 128 : BK * 2>;
            constexpr uint32_t LEADING = ALONG_MN ? BK * 128 : 16, STEP = (ALONG_MN ? 16 * 128 : 32) >> 4;  // STEP: 16 along k
            constexpr uint32_t AP = S::A_PLANE >> 4, BP = S::B_PLANE >> 4;
            const uint32_t a_first = matrix_descriptor(shared_address(stages), LEADING);
            const uint32_t b_first = matrix_descriptor(shared_address(stages) + PLANES * S::A_PLANE, LEADING);
            const bool leads = leader_of_warp();
            uint32_t s = 0, parity = 0, buffer = 0, buffer_parity = 1, issued = 0;
            bool alive = true;
            int chunks = chunks_of<T, FORM, WHOLE>(t, blockIdx.x);
            for (int item = blockIdx.x; alive && item < t.items; item += gridDim.x) {
                const int64_t n0 = item_of<T, FORM>(t, item).n0;
                if (FORM == WEIGHT) chunks = chunks_of<T, FORM, WHOLE>(t, item);
                const int columns = (int)min((int64_t)BN, (t.N - n0 + 15) / 16 * 16);
                const uint32_t descriptor = base | (uint32_t)(columns / 8) << 17;
                // Of a whole tile the planes h and m of B lie behind each other in shared memory as the two accumulators do in theirs: one
                // product of twice the columns gives hh and hm and reads A once.  (Reading the operands bounds products of 128
                // columns, at some 108 cycles for 64.  The same for mh and mm would put mh into the accumulator of hh: no faster,
                // for twice the error.)
                [[maybe_unused]] const bool both = columns == BN;
                [[maybe_unused]] constexpr uint32_t descriptor_of_both = base | (uint32_t)(2 * BN / 8) << 17;
                int of_segment = 0;
                for (int chunk = 0; alive && chunk < chunks; ++chunk) {
                    const uint32_t accumulator = tmem + buffer * 256, small = accumulator + 128;
                    const bool fresh = of_segment == 0, last = ++of_segment == S::SEGMENT || chunk + 1 == chunks;
                    bool good = !fresh || barrier_wait<S::SPLIT>(&sums_empty[buffer], buffer_parity, polls, &waits);
                    good = good && barrier_wait<S::SPLIT>(&full[s], parity, polls, &waits);
                    alive = __all_sync(0xffffffffu, good);
                    if (!alive) break;
                    fence_after();
                    if (direct) fence_to_async();  // (what was written by others is for the tensor core from here on)
                    const uint32_t a = a_first + s * (S::STAGE >> 4), b = b_first + s * (S::STAGE >> 4);
                    if (leads) {
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) {
                            const uint32_t ak = a + k * STEP, bk = b + k * STEP;
                            const bool add = !fresh || k > 0;
                            if constexpr (!S::SPLIT) {
                                multiply<UPPER>(accumulator, ak, bk, descriptor, add);
                            } else if (both) {
                                multiply<UPPER>(accumulator, ak, bk, descriptor_of_both, add);
                            } else {
                                multiply<UPPER>(accumulator, ak, bk, descriptor, add);
                                multiply<UPPER>(small, ak, bk + BP, descriptor, add);
                            }
                            if constexpr (S::SPLIT) {
                                multiply<UPPER>(small, ak + AP, bk, descriptor, true);
                                multiply<UPPER>(small, ak, bk + 2 * BP, descriptor, true);
                                multiply<UPPER>(small, ak + 2 * AP, bk, descriptor, true);
                                multiply<UPPER>(small, ak + AP, bk + BP, descriptor, true);
                            }
                        }
                        commit(&empty[s]);
                        if (last) commit(&sums_full[buffer]);
                    }
                    __syncwarp();
                    if (last) {
                        of_segment = 0;
                        buffer ^= 1;
                        if (buffer == 0) buffer_parity ^= 1;
                    }
                    if (++s == STAGES) s = 0, parity ^= 1;
                    if (issued < STAGES) ++issued;
                }
            }
            for (; alive && issued > 0; --issued) {  // the last reports have come in
                if (s == 0) s = STAGES, parity ^= 1;
                --s;
                alive = __all_sync(0xffffffffu, barrier_wait<S::SPLIT>(&empty[s], parity, polls, &waits));
            }
            if (!alive && leads) {  // products that are still under way read shared memory and write the accumulators
                commit(&drained);
                for (int k = 0; k < WAIT_LIMIT && !barrier_poll(&drained, 0); ++k) {}
            }
        } else if (FORM != WEIGHT && warp == COPY_WARP && lane == 0) {
            // -------------------------------------------------------------- the weight's images
            uint32_t round = 0;
            bool alive = true;
            const int chunks = chunks_of<T, FORM, WHOLE>(t, 0);
            for (int item = blockIdx.x; alive && item < t.items; item += gridDim.x) {
                const int64_t n0 = item_of<T, FORM>(t, item).n0;
                const uint32_t rows = (uint32_t)min((int64_t)BN, (t.N - n0 + 15) / 16 * 16);
                const uint8_t *image = t.packed + (n0 / BN) * chunks * PLANES * S::B_PLANE;
                for (int chunk = 0; alive && chunk < chunks; ++chunk, ++round, image += PLANES * S::B_PLANE) {
                    const uint32_t s = round % STAGES;
                    alive = barrier_wait<S::SPLIT>(&empty[s], (round / STAGES & 1) ^ 1, polls, &waits);
                    if (!alive) break;
                    const uint32_t to = shared_address(stages) + s * S::STAGE + PLANES * S::A_PLANE;
                    barrier_expect(&full[s], rows * (BK * 2) * PLANES);
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) bulk_copy(to + q * S::B_PLANE, image + q * S::B_PLANE, rows * (BK * 2), &full[s]);
                }
            }
            // Copies that are still under way write shared memory.  (The producers may not come as far as to complete these phases;
            // the copies take microseconds, and this many polls a hundred times as long.)
            if (!alive)
                for (uint32_t r = round > STAGES ? round - STAGES : 0; r < round; ++r)
                    for (int k = 0; k < 1 << 14 && !barrier_poll(&full[r % STAGES], r / STAGES & 1); ++k) {}
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && waits.given_up) atomicOr(&g_linear_status, STATUS_WAIT_EXPIRED);
    if (warp == MMA_WARP) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLUMNS) : "memory");
    }
}

bool whole_rows(const void *p, int64_t stride, size_t item, int vector = 8) {
    return stride % vector == 0 && (uintptr_t)p % (vector * item) == 0;
}

template <typename T>
void set_out(Tiles<T> &t, void *out, int64_t width, size_t item) {
    t.out = out;
    t.out_whole = whole_rows(out, width, item);
    t.out_wide = whole_rows(out, width, item, (int)(32 / item));
}

template <typename T>
size_t packed_bytes(int64_t N, int64_t K) {
    using S = Tile<T, FORWARD>;  // (and INPUT)
    return (size_t)ceil_div(N, S::BN) * (size_t)ceil_div(K, S::BK) * S::PLANES * S::B_PLANE;
}

template <typename T, int FORM, bool WHOLE, bool MANY, bool DROP>
int launch_as(const Tiles<T> &t, cudaStream_t stream) {
    using S = Shape<T, FORM, WHOLE>;
    auto *const kernel = tile_kernel<T, FORM, WHOLE, MANY, DROP>;
    CGNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SHARED));
    kernel<<<(unsigned)std::min(t.items, SMS), THREADS, S::SHARED, stream>>>(t);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}
template <typename T, int FORM, bool WHOLE, bool MANY>
int launch_dropping(const Tiles<T> &t, cudaStream_t stream) {
    if constexpr (FORM == FORWARD)
        if (t.epilogue.drop.threshold) return launch_as<T, FORM, WHOLE, MANY, true>(t, stream);
    return launch_as<T, FORM, WHOLE, MANY, false>(t, stream);
}

template <typename T, int FORM>
int launch(Tiles<T> &t, int64_t splits, cudaStream_t stream) {
    const int64_t tiles_m = ceil_div(t.M, BM), tiles_n = ceil_div(t.N, Tile<T, FORM>::BN);
    CGNN_REQUIRE(tiles_m * tiles_n * splits < (1ll << 30), "linear: too many tiles");
    t.tiles_m = (int)tiles_m;
    t.tiles_n = (int)tiles_n;
    t.items = (int)(tiles_m * tiles_n * splits);
    // (fp32 units are loaded at once, and are there or not)
    const bool whole = whole_rows(t.a, t.a_stride, sizeof(T)) && (FORM != WEIGHT || whole_rows(t.b, t.b_stride, sizeof(T))) &&
                       (!Tile<T, FORM>::SPLIT || ((FORM == WEIGHT ? t.M : t.K) % 8 == 0 && (FORM != WEIGHT || t.N % 8 == 0)));
    if (t.k_per_item > Tile<T, FORM>::SEGMENT * Tile<T, FORM>::BK)
        return whole ? launch_dropping<T, FORM, true, true>(t, stream) : launch_dropping<T, FORM, false, true>(t, stream);
    return whole ? launch_dropping<T, FORM, true, false>(t, stream) : launch_dropping<T, FORM, false, false>(t, stream);
}

template <typename T, int FORM>
int pack(const T *weight, int64_t in, int64_t N, int64_t K, uint8_t *packed, cudaStream_t stream) {
    using S = Tile<T, FORM>;
    const int64_t chunks = ceil_div(K, S::BK), units = ceil_div(N, S::BN) * S::BN * chunks * (S::BK / 8);
    pack_kernel<T, FORM><<<(unsigned)ceil_div(units, 256), 256, 0, stream>>>(weight, in, N, K, chunks, packed,
                                                                              whole_rows(weight, in, sizeof(T)));
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

}  // namespace

// Whether sums over the segments lie in memory, [rows, columns] of them.
template <typename T>
static bool in_segments(int64_t terms) {
    return !Tile<T, FORWARD>::SPLIT && terms > LONGEST;
}
template <typename T>
static size_t running_bytes(int64_t rows, int64_t columns, int64_t terms) {
    return in_segments<T>(terms) ? (size_t)rows * columns * sizeof(float) + 32 : 0;
}
template <typename T>
static void set_running(Tiles<T> &t, void *behind) {
    t.running = reinterpret_cast<float *>(align_up((size_t)behind, 32));
    t.running_whole = t.N % 8 == 0;
}

template <typename T>
size_t tiles_forward_bytes(int64_t rows, int64_t in, int64_t out) {
    return packed_bytes<T>(out, in) + running_bytes<T>(rows, out, in);
}

template <typename T>
int tiles_forward(const Call &c, const T *weight, const Epilogue<T> &epilogue, T *y, void *scratch, int polls, cudaStream_t stream) {
    uint8_t *const packed = static_cast<uint8_t *>(scratch);
    int rc = pack<T, FORWARD>(weight, c.in, c.out, c.in, packed, stream);
    if (rc != CGNN_OK) return rc;
    Tiles<T> t{};
    t.a = static_cast<const T *>(c.x);
    t.a_stride = c.stride;
    t.b = weight;
    t.b_stride = c.in;
    t.packed = packed;
    t.M = c.rows;
    t.N = c.out;
    t.K = t.k_per_item = c.in;
    set_out(t, y, c.out, sizeof(T));
    if (epilogue.residual != nullptr) t.out_whole = t.out_whole && whole_rows(epilogue.residual, c.out, sizeof(T));
    set_running(t, packed + packed_bytes<T>(c.out, c.in));
    t.epilogue = epilogue;
    t.polls = polls;
    return launch<T, FORWARD>(t, 1, stream);
}

// Splits of the rows of a weight gradient: as many as leave each multiprocessor one item at most, and none of fewer rows than 8 chunks of
// whole vectors (256 rows in fp32, 512 in 16 bits).  From 75 tiles up that is one split: up to 147 leave multiprocessors without an
// item, more take turns.
template <typename T>
static int64_t weight_splits(int64_t rows, int64_t in, int64_t out, int64_t *rows_per_split) {
    using S = Tile<T, WEIGHT>;
    const int64_t tiles = ceil_div(out, BM) * ceil_div(in, S::BN);
    const int64_t wanted = std::max<int64_t>(1, std::min<int64_t>(SMS / tiles, rows / (8 * S::BK)));
    *rows_per_split = ceil_div(ceil_div(rows, wanted), S::BK) * S::BK;
    return ceil_div(rows, *rows_per_split);
}

template <typename T>
size_t tiles_backward_bytes(int64_t rows, int64_t in, int64_t out) {
    int64_t per_split;
    const int64_t splits = weight_splits<T>(rows, in, out, &per_split);
    // (the input's gradient and then the weight's take what is behind the weight's image)
    const bool parts = splits > 1 || in_segments<T>(per_split);
    const size_t of_weight = (size_t)splits * out * ((parts ? in : 0) * sizeof(float) + sizeof(double)) + 64;
    return packed_bytes<T>(in, out) + std::max(of_weight, running_bytes<T>(rows, in, out));
}

template <typename T>
int tiles_backward(const Call &c, const T *weight, const T *grad, const uint8_t *mask, double scale, T *dx, T *dweight, T *dbias,
                   void *scratch, int polls, cudaStream_t stream) {
    uint8_t *const packed = static_cast<uint8_t *>(scratch);
    Tiles<T> t{};
    t.a = grad;
    t.a_stride = c.out;
    t.mask = mask;
    t.mask_pitch = mask_pitch(c.out);
    t.scale = (float)scale;
    t.polls = polls;
    if (dx != nullptr) {
        int rc = pack<T, INPUT>(weight, c.in, c.in, c.out, packed, stream);
        if (rc != CGNN_OK) return rc;
        t.b = weight;
        t.b_stride = c.in;
        t.packed = packed;
        t.M = c.rows;
        t.N = c.in;
        t.K = t.k_per_item = c.out;
        set_out(t, dx, c.in, sizeof(T));
        set_running(t, packed + packed_bytes<T>(c.in, c.out));
        rc = launch<T, INPUT>(t, 1, stream);
        if (rc != CGNN_OK) return rc;
    }
    if (dweight == nullptr) return CGNN_OK;
    int64_t per_split;
    const int64_t splits = weight_splits<T>(c.rows, c.in, c.out, &per_split);
    double *const sums = reinterpret_cast<double *>(align_up((size_t)packed + packed_bytes<T>(c.in, c.out), 32));
    float *const parts = reinterpret_cast<float *>(align_up((size_t)(sums + splits * c.out), 32));
    t.b = static_cast<const T *>(c.x);
    t.b_stride = c.stride;
    t.packed = nullptr;
    t.M = c.out;
    t.N = c.in;
    t.K = c.rows;
    t.k_per_item = per_split;
    t.partial = splits > 1;
    set_out(t, t.partial ? static_cast<void *>(parts) : dweight, c.in, t.partial ? sizeof(float) : sizeof(T));
    set_running(t, parts);  // (of several splits the parts themselves)
    t.column_sums = dbias != nullptr ? sums : nullptr;
    int rc = launch<T, WEIGHT>(t, splits, stream);
    if (rc == CGNN_OK && t.partial) rc = join(parts, splits, c.out * c.in, scale, dweight, stream);
    if (rc == CGNN_OK && dbias != nullptr) rc = join_columns(sums, splits, c.out, scale, dbias, stream);
    return rc;
}

#define CGNN_TILES_OF(T)                                                                                                        \
    template size_t tiles_forward_bytes<T>(int64_t, int64_t, int64_t);                                                                   \
    template int tiles_forward<T>(const Call &, const T *, const Epilogue<T> &, T *, void *, int, cudaStream_t);                \
    template size_t tiles_backward_bytes<T>(int64_t, int64_t, int64_t);                                                         \
    template int tiles_backward<T>(const Call &, const T *, const T *, const uint8_t *, double, T *, T *, T *, void *, int, \
                                   cudaStream_t);
CGNN_TILES_OF(float)
CGNN_TILES_OF(__nv_bfloat16)
CGNN_TILES_OF(__half)

}  // namespace cgnn
