// The random words of every dropout of this library: counter based, so that a mask is never stored.
#pragma once

#include "cgnn_common.cuh"

namespace cgnn {

// 32 x 32 -> 64 bits in one instruction (the product of widened operands compiles to more: 45 instructions a block of four
// words against 34).  The multiplications are what bounds a block, at four cycles each.
__device__ __forceinline__ uint64_t wide_product(uint32_t a, uint32_t b) {
    uint64_t p;
    asm("mul.wide.u32 %0, %1, %2;" : "=l"(p) : "r"(a), "r"(b));
    return p;
}

// Philox4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with 7
// rounds: four 32-bit words for the counter (element-vector index, 0) under the key `seed`.  Counter
// based, so the words of an element do not depend on which thread produces them.
__device__ __forceinline__ uint4 philox4x32_7(uint64_t counter, uint64_t seed) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0x243F6A88u, c3 = 0x85A308D3u;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 7; ++round) {
        const uint64_t p0 = wide_product(c0, 0xD2511F53u), p1 = wide_product(c2, 0xCD9E8D57u);
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// The same function with what does not change from counter to counter worked out before: of the first two rounds what
// depends on the key and the upper half of the counter only, which all counters of a launch but a few share.  Two
// multiplications of fourteen are saved.
struct Philox {
    uint32_t k0, k1, upper, second_upper, second_lower;
    __device__ __forceinline__ explicit Philox(uint64_t seed) : k0((uint32_t)seed), k1((uint32_t)(seed >> 32)) { begin(0); }
    __device__ __forceinline__ void begin(uint32_t counter_upper) {
        constexpr uint64_t constant = (uint64_t)0xCD9E8D57u * 0x243F6A88u;
        upper = counter_upper;
        const uint64_t p = wide_product((uint32_t)(constant >> 32) ^ upper ^ k0, 0xD2511F53u);
        second_upper = (uint32_t)(p >> 32) ^ (k1 + 0xBB67AE85u);
        second_lower = (uint32_t)p;
    }
    __device__ __forceinline__ uint4 operator()(uint64_t counter) {
        if ((uint32_t)(counter >> 32) != upper) begin((uint32_t)(counter >> 32));
        return block((uint32_t)counter);
    }
    // The block of a counter whose upper half is `upper`.
    __device__ __forceinline__ uint4 block(uint32_t counter_lower) const {
        constexpr uint32_t constant_lower = 0xCD9E8D57u * 0x243F6A88u;
        const uint64_t p = wide_product(counter_lower, 0xD2511F53u);
        const uint64_t q = wide_product((uint32_t)(p >> 32) ^ 0x85A308D3u ^ k1, 0xCD9E8D57u);
        uint32_t c0 = (uint32_t)(q >> 32) ^ constant_lower ^ (k0 + 0x9E3779B9u), c1 = (uint32_t)q;
        uint32_t c2 = second_upper ^ (uint32_t)p, c3 = second_lower;
#pragma unroll
        for (uint32_t round = 2; round < 7; ++round) {
            const uint64_t p0 = wide_product(c0, 0xD2511F53u), p1 = wide_product(c2, 0xCD9E8D57u);
            c0 = (uint32_t)(p1 >> 32) ^ c1 ^ (k0 + round * 0x9E3779B9u);
            c1 = (uint32_t)p1;
            c2 = (uint32_t)(p0 >> 32) ^ c3 ^ (k1 + round * 0xBB67AE85u);
            c3 = (uint32_t)p0;
        }
        return make_uint4(c0, c1, c2, c3);
    }
};

// Blocks first, first + 1, ... of a run (a row, a tile): their upper half is looked at once where it is the same for all.
struct PhiloxRun {
    Philox &words;
    uint32_t lower, upper;
    bool one_upper;
    __device__ __forceinline__ PhiloxRun(Philox &words_, uint64_t first, uint32_t count)
        : words(words_), lower((uint32_t)first), upper((uint32_t)(first >> 32)), one_upper(lower + count >= lower) {
        if (words.upper != upper) words.begin(upper);
    }
    __device__ __forceinline__ uint4 operator()(uint32_t at) {
        if (!one_upper) {
            const uint32_t here = upper + (lower + at < lower);
            if (words.upper != here) words.begin(here);
        }
        return words.block(lower + at);
    }
};

// Dropout of the VW values of the vector that starts at element `first` of the output (VW is 1, 2, 4 or a multiple of
// 4 and divides `first`).  Element e takes word e % 4 of the Philox block counted e / 4, so the mask is a
// function of (seed, element index) alone: the same whatever the element type or the kernel that writes it.
// `words`: the block of a counter.
template <typename T, int VW, typename Words>
__device__ __forceinline__ void drop_values(T (&y)[VW], int64_t first, uint32_t threshold, T keep_scale, Words &&words) {
    static_assert(VW == 1 || VW == 2 || VW % 4 == 0, "a vector lies inside one block of four random words, or is whole blocks");
    if constexpr (VW % 4 == 0) {
#pragma unroll
        for (int b = 0; b < VW / 4; ++b) {
            const uint4 q = words(((uint64_t)first >> 2) + b);
            const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) y[4 * b + k] = word[k] < threshold ? T(0) : y[4 * b + k] * keep_scale;
        }
    } else if constexpr (VW == 2) {
        const uint4 r = words((uint64_t)first >> 2);
        const bool upper = (first & 2) != 0;
        const uint32_t w0 = upper ? r.z : r.x, w1 = upper ? r.w : r.y;
        y[0] = w0 < threshold ? T(0) : y[0] * keep_scale;
        y[1] = w1 < threshold ? T(0) : y[1] * keep_scale;
    } else {
        const uint4 r = words((uint64_t)first >> 2);
        const int at = (int)(first & 3);
        const uint32_t w = at == 0 ? r.x : at == 1 ? r.y : at == 2 ? r.z : r.w;
        y[0] = w < threshold ? T(0) : y[0] * keep_scale;
    }
}

// The same of a vector of whole blocks, the block `at` of a run and the ones behind it.
template <typename T, int VW>
__device__ __forceinline__ void drop_blocks(T (&y)[VW], uint32_t at, uint32_t threshold, T keep_scale, PhiloxRun &run) {
#pragma unroll
    for (int b = 0; b < VW / 4; ++b) {
        const uint4 q = run(at + b);
        const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) y[4 * b + k] = word[k] < threshold ? T(0) : y[4 * b + k] * keep_scale;
    }
}

// Which of the elements first + lane + 32 p of a row, p < VPL, a lane loses (bit p), for a whole warp together: a lane
// draws the four words of one block, and votes hand each word's verdict to the lane whose element it is.  A lane alone
// would draw a block for every element.
template <int VPL>
__device__ __forceinline__ uint32_t dropped_of_row(int64_t first, uint32_t threshold, Philox &words) {
    constexpr int WINDOWS = (32 * VPL + 3 + 127) / 128;  // of 32 blocks; the row may begin inside a block
    const int lane = threadIdx.x & 31, ahead = (int)(first & 3) + lane, word = ahead & 3;
    uint32_t verdict[WINDOWS], gone = 0;
#pragma unroll
    for (int w = 0; w < WINDOWS; ++w) {
        const uint4 r = words(((uint64_t)first >> 2) + 32 * w + lane);
        const uint32_t v0 = __ballot_sync(0xffffffffu, r.x < threshold), v1 = __ballot_sync(0xffffffffu, r.y < threshold);
        const uint32_t v2 = __ballot_sync(0xffffffffu, r.z < threshold), v3 = __ballot_sync(0xffffffffu, r.w < threshold);
        verdict[w] = word == 0 ? v0 : word == 1 ? v1 : word == 2 ? v2 : v3;
    }
#pragma unroll
    for (int p = 0; p < VPL; ++p) {
        const int at = 32 * (p % 4) + ahead;  // elements from the beginning of window p / 4
        uint32_t bits = verdict[p / 4];
        if (p % 4 == 3 && p / 4 + 1 < WINDOWS && at >= 128) bits = verdict[p / 4 + 1];
        gone |= (bits >> ((at & 127) >> 2) & 1u) << p;
    }
    return gone;
}

// A probability as the bound its random words are compared with: an element is dropped when its word lies below.
static inline uint32_t drop_threshold_of(double p) {
    const double bound = p * 4294967296.0;
    return (uint32_t)(bound < 4294967295.0 ? bound : 4294967295.0);
}

}  // namespace cgnn
