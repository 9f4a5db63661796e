// One AdamW step over many tensors: t = t + 1, g' = clip * g,
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps),
// with clip = min(1, max_norm / (|all g| + 1e-6)) or 1, and decay applied to the parameter itself.
//
// Memory bounds it with moments of 32 bits, 28 bytes an fp32 parameter (157 M of them 723 us, 0.92 of the copy rate; 101 M bf16
// ones 366, clipped 410).  With moments of 8 bits it is 16 bytes and 82 instructions, and the instructions come first (522).
//
// Moments in 8 bits: m and r = sqrt(v) are e4m3 numbers times a scale for each 256 consecutive elements, the least power
// of two that takes the block's largest value in (448 is e4m3's).  A power of two, so that an element's grid stays where
// it is when its block's scale moves.  The root, because e4m3 spans 17 binary orders of r and would span as many of v only.
// Rounding is stochastic: b2 moves v by a thousandth of itself a step and a step of e4m3 is an eighth, so that rounding to
// nearest would leave v where it is; a random rounding moves it with the right mean.  A root above zero is never
// rounded to zero: it divides m.  The random bits are 16 for each value of the word that the library's generator
// (Philox4x32-7) gives element e of the tensor under the key seed + index * TENSOR_KEY + (t - 1) * STEP_KEY.
#include <algorithm>
#include <cmath>
#include <vector>

#include <cuda_fp8.h>

#include "cgnn_philox.cuh"
#include "cgnn_rows.cuh"

namespace cgnn {
namespace {

constexpr int ADAM_THREADS = 256;
constexpr int ADAM_GROUP = 256;                              // elements a warp takes at once: the block of a scale
constexpr int ADAM_CHUNK = ADAM_GROUP * ADAM_THREADS / 32;   // elements a block takes at once
constexpr int SMS = 148;
constexpr uint64_t TENSOR_KEY = 0x9E3779B97F4A7C15ull, STEP_KEY = 0xD1342543DE82EF95ull;

struct Entry {
    void *param;
    const void *grad;
    void *first, *second;
    float *first_scale, *second_scale;
    // The number of steps taken, in the lower 32 bits.  While a launch runs the upper ones count the chunks that are done;
    // whoever brings in the last one writes the new number.
    unsigned long long *step;
    int64_t n;
    double lr, decay;
    const float *device_lr;
    int32_t first_chunk, chunks;
    int32_t index;
    int32_t whole;  // every array lies on the boundary of its vectors
};

// The tensors of a launch travel as its argument.  Few of them in a small one: the argument is copied at every launch.
template <int CAP>
struct Table {
    Entry entry[CAP];
    int32_t count, chunks;
};
constexpr int FEW = 32, MANY = 300;
static_assert(sizeof(Table<FEW>) <= 3600 && sizeof(Table<MANY>) <= 32000, "a launch takes 32764 bytes of arguments");

struct Step {
    double ln_beta1, ln_beta2, beta1, beta2, eps, max_norm;
    const double *partials;  // of the squared norm; null without clipping
    int32_t partial_count;
    float *norm;             // where the first block leaves the norm; may be null
    uint64_t seed;
};

__device__ __forceinline__ float expm1_of(float x) { return expm1f(x); }
__device__ __forceinline__ double expm1_of(double x) { return expm1(x); }
__device__ __forceinline__ float root_of(float x) { return __fsqrt_rn(x); }
__device__ __forceinline__ double root_of(double x) { return sqrt(x); }
// (Products and sums are rounded one by one, so that the moments do not depend on which of them a compiler joins.)
__device__ __forceinline__ float times(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ double times(double a, double b) { return __dmul_rn(a, b); }
__device__ __forceinline__ float plus(float a, float b) { return __fadd_rn(a, b); }
__device__ __forceinline__ double plus(double a, double b) { return __dadd_rn(a, b); }

// The tensor that a chunk belongs to.
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP> &table, int chunk) {
    int low = 0, high = table.count - 1;
    while (low < high) {
        const int middle = (low + high + 1) >> 1;
        if (table.entry[middle].first_chunk <= chunk) low = middle;
        else high = middle - 1;
    }
    return low;
}

__device__ __forceinline__ double block_sum(double s, double *shared) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < ADAM_THREADS / 32; ++w) s += shared[w];
    return s;
}

// partials[b] = the squares of block b's chunks.  In fp64: the norm is the same in every fp32 digit whatever the order.
template <typename T, int CAP>
__global__ void __launch_bounds__(ADAM_THREADS) squares_kernel(const __grid_constant__ Table<CAP> table, double *partials) {
    __shared__ double shared[ADAM_THREADS / 32];
    double s = 0.0;
    for (int chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
        const Entry &e = table.entry[tensor_of(table, chunk)];
        const int64_t base = (int64_t)(chunk - e.first_chunk) * ADAM_CHUNK;
        const T *const g = static_cast<const T *>(e.grad) + base;
        const int64_t left = e.n - base;
        constexpr int VW = 16 / sizeof(T), ROUNDS = ADAM_CHUNK / (ADAM_THREADS * VW);
        if (e.whole && left >= ADAM_CHUNK) {
            Vec<T, VW> v[ROUNDS];
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r) v[r] = vec_load<T, VW>(g + (r * ADAM_THREADS + threadIdx.x) * VW);
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
                for (int k = 0; k < VW; ++k) {
                    const double x = (double)widen(v[r].v[k]);
                    s = fma(x, x, s);
                }
        } else {
            for (int i = threadIdx.x; i < ADAM_CHUNK && i < left; i += ADAM_THREADS) {
                const double x = (double)widen(g[i]);
                s = fma(x, x, s);
            }
        }
    }
    s = block_sum(s, shared);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// Four values or codes of one lane; the elements behind a tensor's end are zeros and are not written.
// WHOLE: all four are there, on the boundary of their vector.
template <bool WHOLE, typename T>
__device__ __forceinline__ void load4(const T *p, int64_t at, int64_t n, Acc<T> (&x)[4]) {
    if constexpr (WHOLE) {
        if constexpr (sizeof(T) == 8) {
            widen_all<T, 2>(vec_load<T, 2>(p + at), reinterpret_cast<Acc<T>(&)[2]>(x[0]));
            widen_all<T, 2>(vec_load<T, 2>(p + at + 2), reinterpret_cast<Acc<T>(&)[2]>(x[2]));
        } else {
            widen_all<T, 4>(vec_load<T, 4>(p + at), x);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = at + k < n ? widen(p[at + k]) : Acc<T>(0);
    }
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store4(T *p, int64_t at, int64_t n, const Acc<T> (&x)[4]) {
    if constexpr (WHOLE) {
        if constexpr (sizeof(T) == 8) {
            vec_store<T, 2>(p + at, Vec<T, 2>{x[0], x[1]});
            vec_store<T, 2>(p + at + 2, Vec<T, 2>{x[2], x[3]});
        } else {
            vec_store<T, 4>(p + at, narrow_all<T, 4>(x));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (at + k < n) p[at + k] = narrow<T>(x[k]);
    }
}

template <bool WHOLE>
__device__ __forceinline__ uint32_t load_codes(const uint8_t *p, int64_t at, int64_t n) {
    if (WHOLE) return *reinterpret_cast<const uint32_t *>(p + at);
    uint32_t codes = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (at + k < n) codes |= (uint32_t)p[at + k] << (8 * k);
    return codes;
}
template <bool WHOLE>
__device__ __forceinline__ void store_codes(uint8_t *p, int64_t at, int64_t n, uint32_t codes) {
    if (WHOLE) {
        *reinterpret_cast<uint32_t *>(p + at) = codes;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (at + k < n) p[at + k] = (uint8_t)(codes >> (8 * k));
    }
}

// The values of four codes under their block's scale.
__device__ __forceinline__ void values_of(uint32_t codes, float scale, float (&x)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const float2 two = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (8 * k)), __NV_E4M3)));
        x[k] = __fmul_rn(two.x, scale);
        x[k + 1] = __fmul_rn(two.y, scale);
    }
}

// The exponent of the least power of two s with `largest` <= 448 s (448 = 0.875 * 2^9).  Not below 2^-117, whose inverse is a
// normal number.
__device__ __forceinline__ int scale_exponent(uint32_t largest_bits) {
    return max((int)(largest_bits >> 23) - 135 + ((largest_bits & 0x7fffffu) > 0x600000u ? 1 : 0), -117);
}
__device__ __forceinline__ float power_of_two(int exponent) { return __uint_as_float((uint32_t)(exponent + 127) << 23); }

// Four values as codes: |x| * inverse, at most 448, rounded to an e4m3 number, up with the probability that 16 random bits
// allow.  A normal number loses the lower 20 bits of its fraction after they were added to, one below 2^-6 is a multiple of
// 2^-9.  ROOT: a value above zero is not rounded to zero.  `plain`: every value of the warp is finite; others become NaN.
template <bool ROOT>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float inverse, const uint32_t (&random16)[4], bool plain) {
    uint32_t codes = 0;
    float rounded[4];
    bool small = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float size = __fmul_rn(fabsf(x[k]), inverse);
        small = small || size < 1.f / 64.f;
        rounded[k] = __uint_as_float((__float_as_uint(size) + (random16[k] << 4)) & 0xfff00000u);
    }
    if (small || !plain) {  // few blocks have such values
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float size = __fmul_rn(fabsf(x[k]), inverse);
            if (size < 1.f / 64.f) {
                const float steps = floorf(__fadd_rn(__fmul_rn(size, 512.f), __fmul_rn((float)random16[k], 1.f / 65536.f)));
                rounded[k] = __fmul_rn(ROOT && size > 0.f ? fmaxf(steps, 1.f) : steps, 1.f / 512.f);
            }
            if (__float_as_uint(size) > 0x43e00000u) rounded[k] = __uint_as_float(0x7fffffffu);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const float2 two = ROOT ? make_float2(rounded[k], rounded[k + 1])
                                : make_float2(copysignf(rounded[k], x[k]), copysignf(rounded[k + 1], x[k + 1]));
        codes |= (uint32_t)__nv_cvt_float2_to_fp8x2(two, __NV_SATFINITE, __NV_E4M3) << (8 * k);
    }
    return codes;
}

__device__ __forceinline__ uint32_t size_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// The largest of a block's eight values a lane, of the finite ones where there are others.
__device__ __forceinline__ uint32_t largest_of(const float (&x)[2][4], bool &plain) {
    uint32_t largest = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) largest = max(largest, size_bits(x[e / 4][e % 4]));
    largest = __reduce_max_sync(0xffffffffu, largest);
    if (largest >= 0x7f800000u) {
        plain = false;
        largest = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t bits = size_bits(x[e / 4][e % 4]);
            largest = max(largest, bits < 0x7f800000u ? bits : 0u);
        }
        largest = __reduce_max_sync(0xffffffffu, largest);
    }
    return largest;
}

// (The quotient goes into the parameter only, whose rounding is far above its two last bits.)
__device__ __forceinline__ float quotient(float a, float b) { return __fdividef(a, b); }
__device__ __forceinline__ double quotient(double a, double b) { return a / b; }

template <typename A>
struct Rates {
    A clip, b1, b2, c1, c2, eps, keep, rate, inverse_root2;
};

// A warp's group of elements.  WHOLE: all of them are there, on the boundaries of their vectors.  With a test at each access instead
// of one for all, 157 M fp32 parameters with 8-bit moments took 716 us for 522 and 101 M bf16 ones 452 for 365; the next
// group's lines on their way to L2 (prefetches, one a lane) cost 8 %.
template <typename T, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void update(const Entry &e, int64_t base, int lane, const Rates<Acc<T>> &r, Philox &words) {
    using A = Acc<T>;
    A p[2][4], g[2][4], m[2][4], v[2][4];
    uint32_t m_codes[2], r_codes[2];
    int64_t at[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        at[u] = base + u * 128 + lane * 4;
        load4<WHOLE>(static_cast<const T *>(e.param), at[u], e.n, p[u]);
        load4<WHOLE>(static_cast<const T *>(e.grad), at[u], e.n, g[u]);
        if constexpr (EIGHT) {
            m_codes[u] = load_codes<WHOLE>(static_cast<const uint8_t *>(e.first), at[u], e.n);
            r_codes[u] = load_codes<WHOLE>(static_cast<const uint8_t *>(e.second), at[u], e.n);
        } else {
            load4<WHOLE>(static_cast<const A *>(e.first), at[u], e.n, m[u]);
            load4<WHOLE>(static_cast<const A *>(e.second), at[u], e.n, v[u]);
        }
    }
    const int64_t group = base / ADAM_GROUP;
    if constexpr (EIGHT) {
        const float m_scale = e.first_scale[group], r_scale = e.second_scale[group];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            values_of(m_codes[u], m_scale, m[u]);
            values_of(r_codes[u], r_scale, v[u]);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[u][k] = times(v[u][k], v[u][k]);
        }
    }
    A root[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const A gk = times(g[u][k], r.clip);
            m[u][k] = plus(times(m[u][k], r.b1), times(gk, r.c1));
            v[u][k] = plus(times(v[u][k], r.b2), times(times(gk, gk), r.c2));
            root[u][k] = root_of(v[u][k]);
            p[u][k] = plus(times(p[u][k], r.keep), times(r.rate, quotient(m[u][k], plus(times(root[u][k], r.inverse_root2), r.eps))));
        }
#pragma unroll
    for (int u = 0; u < 2; ++u) store4<WHOLE>(static_cast<T *>(e.param), at[u], e.n, p[u]);
    if constexpr (EIGHT) {
        bool plain = true;
        const int m_exponent = scale_exponent(largest_of(m, plain)), r_exponent = scale_exponent(largest_of(root, plain));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint4 w = words((uint64_t)at[u] >> 2);
            const uint32_t low[4] = {w.x & 0xffffu, w.y & 0xffffu, w.z & 0xffffu, w.w & 0xffffu};
            const uint32_t high[4] = {w.x >> 16, w.y >> 16, w.z >> 16, w.w >> 16};
            store_codes<WHOLE>(static_cast<uint8_t *>(e.first), at[u], e.n, codes_of<false>(m[u], power_of_two(-m_exponent), low, plain));
            store_codes<WHOLE>(static_cast<uint8_t *>(e.second), at[u], e.n,
                        codes_of<true>(root[u], power_of_two(-r_exponent), high, plain));
        }
        if (lane == 0) {
            e.first_scale[group] = power_of_two(m_exponent);
            e.second_scale[group] = power_of_two(r_exponent);
        }
    } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            store4<WHOLE>(static_cast<A *>(e.first), at[u], e.n, m[u]);
            store4<WHOLE>(static_cast<A *>(e.second), at[u], e.n, v[u]);
        }
    }
}

// (Moments of 8 bits, 157 M fp32 parameters: three blocks of 80 registers a multiprocessor 522 us, four of 64, which spill, 546, two
// of 96 716.)
template <typename T, bool EIGHT, int CAP>
__global__ void __launch_bounds__(ADAM_THREADS, sizeof(T) == 8 ? 2 : EIGHT ? 3 : 4) adamw_kernel(const __grid_constant__ Table<CAP> table, const Step set) {
    using A = Acc<T>;
    __shared__ double shared[ADAM_THREADS / 32];
    A clip = A(1);
    if (set.partials != nullptr) {
        double s = 0.0;
        for (int i = threadIdx.x; i < set.partial_count; i += ADAM_THREADS) s += set.partials[i];
        const double norm = sqrt(block_sum(s, shared));
        if (blockIdx.x == 0 && threadIdx.x == 0 && set.norm != nullptr) *set.norm = (float)norm;
        const double ratio = set.max_norm / (norm + 1e-6);
        clip = (A)(ratio > 1.0 ? 1.0 : ratio);  // (a norm that is NaN stays one)
    }
    const A b1 = (A)set.beta1, b2 = (A)set.beta2, c1 = (A)(1.0 - set.beta1),
            c2 = (A)(1.0 - set.beta2), eps = (A)set.eps;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int tensor = -1, done = 0;
    A keep = A(1), rate = A(0), inverse_root2 = A(0);
    uint32_t before = 0;
    Philox words(0);
    const auto report = [&] {  // the chunks of `tensor` that this block has finished
        __syncthreads();
        if (threadIdx.x == 0 && done) {
            const Entry &e = table.entry[tensor];
            const unsigned long long seen = atomicAdd(e.step, (unsigned long long)done << 32);
            if ((int)(seen >> 32) + done == e.chunks) *e.step = (unsigned long long)(before + 1);
        }
        done = 0;
    };
    for (int chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
        const int owner = tensor_of(table, chunk);
        const Entry &e = table.entry[owner];
        if (owner != tensor) {
            if (tensor >= 0) report();
            tensor = owner;
            before = (uint32_t)*reinterpret_cast<volatile unsigned long long *>(e.step);
            const double t = (double)(before + 1u);
            const double lr = e.device_lr != nullptr ? (double)*e.device_lr : e.lr;
            keep = (A)(1.0 - lr * e.decay);
            rate = (A)lr / expm1_of((A)(t * set.ln_beta1));  // - lr / (1 - beta1^t)
            inverse_root2 = A(1) / root_of(-expm1_of((A)(t * set.ln_beta2)));
            if constexpr (EIGHT) words = Philox(set.seed + (uint64_t)e.index * TENSOR_KEY + (uint64_t)before * STEP_KEY);
        }
        const int64_t base = (int64_t)(chunk - e.first_chunk) * ADAM_CHUNK + warp * ADAM_GROUP;
        ++done;
        if (base >= e.n) continue;  // (a whole warp, and no barrier lies ahead in this round)
        const Rates<A> rates{clip, b1, b2, c1, c2, eps, keep, rate, inverse_root2};
        if (e.whole && base + ADAM_GROUP <= e.n) update<T, EIGHT, true>(e, base, lane, rates, words);
        else update<T, EIGHT, false>(e, base, lane, rates, words);
    }
    if (tensor >= 0) report();
}

struct Launch {
    int dtype;
    bool eight;
    std::vector<int> which;
    int64_t chunks = 0;
};

int64_t chunks_of(int64_t n) { return std::max<int64_t>(1, ceil_div(n, ADAM_CHUNK)); }

// Tensors of one type and kind together, as many as a launch's argument takes.
std::vector<Launch> launches_of(const cgnn_adamw_tensor *tensors, int64_t count) {
    std::vector<Launch> launches;
    for (int64_t i = 0; i < count; ++i) {
        const bool eight = tensors[i].exp_avg_scale != nullptr;
        const int64_t chunks = chunks_of(tensors[i].n);
        Launch *room = nullptr;
        for (Launch &l : launches)
            if (l.dtype == tensors[i].dtype && l.eight == eight && (int)l.which.size() < MANY && l.chunks + chunks <= INT32_MAX / 2) room = &l;
        if (room == nullptr) {
            launches.push_back({tensors[i].dtype, eight, {}, 0});
            room = &launches.back();
        }
        room->which.push_back((int)i);
        room->chunks += chunks;
    }
    return launches;
}

int64_t blocks_of_squares(int64_t chunks) { return std::min<int64_t>(chunks, SMS * 8); }

template <int CAP>
void fill(Table<CAP> &table, const Launch &l, const cgnn_adamw_tensor *tensors) {
    int64_t chunk = 0;
    table.count = (int32_t)l.which.size();
    for (int i = 0; i < table.count; ++i) {
        const cgnn_adamw_tensor &t = tensors[l.which[i]];
        Entry &e = table.entry[i];
        e.param = t.param;
        e.grad = t.grad;
        e.first = t.exp_avg;
        e.second = t.exp_avg_sq;
        e.first_scale = t.exp_avg_scale;
        e.second_scale = t.exp_avg_sq_scale;
        e.step = reinterpret_cast<unsigned long long *>(t.step);
        e.n = t.n;
        e.lr = t.lr;
        e.decay = t.weight_decay;
        e.device_lr = t.device_lr;
        e.first_chunk = (int32_t)chunk;
        e.chunks = (int32_t)chunks_of(t.n);
        e.index = l.which[i];
        const uintptr_t places = (uintptr_t)t.param | (uintptr_t)t.grad;
        const uintptr_t moments = (uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq;
        e.whole = places % 16 == 0 && moments % (l.eight ? 4 : 16) == 0;
        chunk += e.chunks;
    }
    table.chunks = (int32_t)chunk;
}

template <typename T, int CAP>
int squares(const Launch &l, const cgnn_adamw_tensor *tensors, double *partials, cudaStream_t stream) {
    Table<CAP> table;
    fill(table, l, tensors);
    squares_kernel<T, CAP><<<(unsigned)blocks_of_squares(l.chunks), ADAM_THREADS, 0, stream>>>(table, partials);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

template <typename T, bool EIGHT, int CAP>
int step(const Launch &l, const cgnn_adamw_tensor *tensors, const Step &set, cudaStream_t stream) {
    static const int resident = resident_blocks(adamw_kernel<T, EIGHT, CAP>, ADAM_THREADS);
    Table<CAP> table;
    fill(table, l, tensors);
    adamw_kernel<T, EIGHT, CAP><<<(unsigned)std::min<int64_t>(l.chunks, SMS * resident), ADAM_THREADS, 0, stream>>>(table, set);
    CGNN_LAUNCH_CHECK();
    return CGNN_OK;
}

template <typename F>
int of_type(const Launch &l, F &&call) {
    switch (l.dtype) {
        case CGNN_F32: return call(float());
        case CGNN_F64: return call(double());
        case CGNN_BF16: return call(__nv_bfloat16());
        default: return call(__half());
    }
}

}  // namespace
}  // namespace cgnn

using namespace cgnn;

extern "C" {

size_t cgnn_adamw_scratch_bytes(const cgnn_adamw_tensor *tensors, int64_t count) {
    if (tensors == nullptr || count <= 0) return 0;
    try {
        int64_t blocks = 0;
        for (const Launch &l : launches_of(tensors, count)) blocks += blocks_of_squares(l.chunks);
        return (size_t)blocks * sizeof(double);
    } catch (...) {
        return 0;
    }
}

int cgnn_adamw(const cgnn_adamw_tensor *tensors, int64_t count, double beta1, double beta2, double eps, double max_norm, uint64_t seed,
               float *norm, void *scratch, size_t scratch_bytes, cgnn_stream_t stream_) {
    cudaStream_t stream = (cudaStream_t)stream_;
    CGNN_REQUIRE(count >= 0 && count <= INT32_MAX, "adamw: bad number of tensors");
    CGNN_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw: the betas must lie in [0, 1)");
    CGNN_REQUIRE(eps >= 0.0, "adamw: eps must not be negative");
    const bool clipped = max_norm >= 0.0;  // negative: no clipping
    CGNN_REQUIRE(max_norm == max_norm, "adamw: max_norm is NaN");
    if (count == 0) return CGNN_OK;
    CGNN_REQUIRE(tensors != nullptr, "adamw: null pointer");
    for (int64_t i = 0; i < count; ++i) {
        const cgnn_adamw_tensor &t = tensors[i];
        CGNN_REQUIRE(t.dtype >= CGNN_F32 && t.dtype <= CGNN_F16, "adamw: unknown dtype");
        CGNN_REQUIRE(t.n >= 0 && t.n <= (int64_t)1 << 40, "adamw: bad number of elements");
        CGNN_REQUIRE((t.device_lr != nullptr || t.lr >= 0.0) && t.weight_decay >= 0.0, "adamw: lr and weight_decay must not be negative");
        CGNN_REQUIRE(t.step != nullptr && ((uintptr_t)t.step & 7) == 0, "adamw: every tensor has an aligned step count");
        CGNN_REQUIRE(t.n == 0 || (t.param != nullptr && t.grad != nullptr && t.exp_avg != nullptr && t.exp_avg_sq != nullptr),
                     "adamw: null pointer");
        CGNN_REQUIRE((t.exp_avg_scale == nullptr) == (t.exp_avg_sq_scale == nullptr), "adamw: both moments have scales, or none");
        CGNN_REQUIRE(t.exp_avg_scale == nullptr || t.dtype != CGNN_F64, "adamw: moments of fp64 parameters are fp64");
    }
    try {
        const std::vector<Launch> launches = launches_of(tensors, count);
        Step set{};
        set.beta1 = beta1;
        set.beta2 = beta2;
        set.ln_beta1 = std::log(beta1);
        set.ln_beta2 = std::log(beta2);
        set.eps = eps;
        set.max_norm = max_norm;
        set.seed = seed;
        if (clipped) {
            CGNN_REQUIRE(scratch != nullptr && scratch_bytes >= cgnn_adamw_scratch_bytes(tensors, count) &&
                             ((uintptr_t)scratch & 7) == 0,
                         "adamw: scratch too small or not on an 8-byte boundary");
            double *partials = static_cast<double *>(scratch);
            set.partials = partials;
            for (const Launch &l : launches) {
                const int rc = of_type(l, [&](auto zero) {
                    using T = decltype(zero);
                    return l.which.size() <= FEW ? squares<T, FEW>(l, tensors, partials, stream)
                                                 : squares<T, MANY>(l, tensors, partials, stream);
                });
                if (rc != CGNN_OK) return rc;
                partials += blocks_of_squares(l.chunks);
                set.partial_count += (int32_t)blocks_of_squares(l.chunks);
            }
        }
        set.norm = norm;
        for (const Launch &l : launches) {
            const int rc = of_type(l, [&](auto zero) {
                using T = decltype(zero);
                const bool few = l.which.size() <= FEW;
                if constexpr (sizeof(T) < 8)
                    if (l.eight) return few ? step<T, true, FEW>(l, tensors, set, stream) : step<T, true, MANY>(l, tensors, set, stream);
                return few ? step<T, false, FEW>(l, tensors, set, stream) : step<T, false, MANY>(l, tensors, set, stream);
            });
            if (rc != CGNN_OK) return rc;
            set.norm = nullptr;
        }
        return CGNN_OK;
    } catch (...) {
        set_error("adamw: out of host memory");
        return CGNN_ERR_INVALID;
    }
}

}  // extern "C"
