// One AdamW step over many tensors, with fp32 states or states in 8 bits.
//
//   g' = f g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
//   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Two launches over one list of chunks in the kernel's parameters: one thread counts the step and works out what
// all elements share (in fp64: t, the bias corrections, f), then a warp takes a block of 256 elements, 8 a lane.
// The second launch starts while the first runs and waits for it when its first loads are on their way
// (programmatic dependent launch).  Bound by HBM: every array passes once.  On a B200 400 million bf16 parameters with
// masters and 8-bit states take 992 us (6.5 TB/s), 200 million in fp32 with fp32 states 818 us (6.8 TB/s).
//
// 8 bits: e4m3 codes of m and of sqrt(v) with a scale for each 256 elements (largest magnitude / 448).  The root
// halves v's range of exponents, so e4m3's 2^17 between the largest and the smallest code are 2^34 of v; a v above
// zero keeps at least the smallest code, so that no later step divides an m that was kept by a v that was lost.
// Scales are fp32, not powers of two: a block whose values all shrink by the same factor keeps its codes and
// shrinks its scale, where rounding each value to its old code would stop v's decay of 0.1 % a step.
//
// With 8-bit states a warp computes for longer than its loads take, at 51 instructions an element; loads held in registers
// for the next block left too few warps (3 blocks of threads an SM, 1.55 ms).  So bulk copies bring the next stages
// into a ring of three in shared memory.  fp32 states compute less: there the next block in registers suffices.
//
// m and v are rounded to fp32 at every operation as it is written, and their codes are those of the correctly rounded
// quotients, so that any fp32 program computes the same states bit for bit.  The change of p takes the approximate
// root and quotient (2^-20 of the change): with the exact ones, 3 quotients and a root an element, the kernel was bound
// by instructions.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include <cuda_fp8.h>

#include "common.cuh"
#include "internal.h"
#include "rows.cuh"

namespace hb {
namespace adamw {

constexpr int kThreads = 256, kBlock = 256;            // kBlock: elements of a scale, a warp's
constexpr int kStage = kThreads / 32 * kBlock;          // elements of a block of threads at a time
constexpr int kRing = 3;                                // 8-bit states: stages of a block in shared memory
// Elements of a block of threads: one stage, so that small calls take all SMs, or from kLongLeast elements on several.
constexpr int kChunk = kStage, kLongChunk = 8192;
constexpr int64_t kLongLeast = 148 * 8 * (int64_t)kLongChunk;
constexpr float kLeastBy = 0x1p-63f;                   // least divisor of a change: the root of the least normal v
constexpr int kFew = 24, kMany = 360;                  // tensors of a launch: 2 KB or 31 KB of parameters

struct Entry {  // one tensor; its fields lie together, as a block reads those of one
    void* param;
    const void* grad;
    void *first, *second;
    float *first_scale, *second_scale, *master;
    int64_t size;
    int32_t chunk;                    // its first
    uint8_t type, grad_type, aligned; // aligned: all of its arrays lie on 16 bytes
};
template <int MOST>
struct List {
    Entry e[MOST];
    int count, chunk;  // tensors, elements a chunk
};
static_assert(sizeof(List<kMany>) < 32000, "kernel parameters");

struct Shared {  // what all elements share, in device memory
    float factor, keep, rate, over_root;  // over_root: 1 / sqrt(1 - b2^t)
};
struct Fixed {
    float beta1, beta2, less1, less2, eps;
};

__global__ void begin_kernel(int* step, const float* norm, const float* rate, double lr, double beta1, double beta2, double decay,
                             double max_norm, Shared* shared) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int t = *step + 1;
    *step = t;
    if (rate) lr = *rate;
    double f = 1.0;
    if (norm) {
        f = max_norm / ((double)*norm + 1e-6);
        f = f >= 1.0 ? 1.0 : f;  // a NaN stays
    }
    shared->factor = (float)f;
    shared->keep = (float)(1.0 - lr * decay);
    shared->rate = (float)(lr / (1.0 - pow(beta1, (double)t)));
    shared->over_root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
}

template <int MOST>
__device__ __forceinline__ int tensor_of(const List<MOST>& l, int chunk) {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.e[mid].chunk <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Two fp32 values in one operation, each rounded like the scalar one: half the instructions of the multiply-add pipe.
union Pair {
    uint64_t both;
    float2 f;
    __device__ __forceinline__ Pair() {}
    __device__ __forceinline__ explicit Pair(float a) : f{a, a} {}
    __device__ __forceinline__ Pair(float a, float b) : f{a, b} {}
};
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.both) : "l"(a.both), "l"(b.both));
    return r;
}
// Scalar: of a product and a sum in pairs the assembler makes one fused operation, .rn or not.
__device__ __forceinline__ Pair operator+(Pair a, Pair b) { return Pair(__fadd_rn(a.f.x, b.f.x), __fadd_rn(a.f.y, b.f.y)); }
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.both) : "l"(a.both), "l"(b.both), "l"(c.both));
    return r;
}
// A lane has 8 values of a block of 256: 4 from lane * 4 on and 4 from 128 further, so that neighbouring lanes' words are
// neighbours in memory.  Writes 4 of them; WHOLE: all are there, on 16 bytes, else `left`.
template <typename T, bool WHOLE>
__device__ __forceinline__ void write4(const Pair* f, T* p, int left) {
    rows::Vec<T, 4 * (int)sizeof(T)> v;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) reinterpret_cast<__nv_bfloat162*>(v.v)[k] = __float22bfloat162_rn(f[k].f);
        else if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2*>(v.v)[k] = __float22half2_rn(f[k].f);
        else v.v[2 * k] = f[k].f.x, v.v[2 * k + 1] = f[k].f.y;
    }
    if (WHOLE) {
        v.store_once(p);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < left) p[j] = v.v[j];
    }
}
__device__ __forceinline__ Pair of_codes(uint32_t two) {  // the lower two bytes
    Pair r;
    r.f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
    return r;
}
__device__ __forceinline__ float root_near(float v) {  // within 2^-23 of the root, 0 for v below 2^-126
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float inverse_near(float v) {  // within 2^-23 of 1 / v, v 0 or a normal number below 2^126
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// v / 448, correctly rounded: the quotient by the constant's inverse and one correction by its residual, both fused, are
// exact for every 24-bit significand (a quotient by a constant after Brisebarre, Muller and Raina; all 2^23 were
// checked), as long as nothing on the way is subnormal.
__device__ __forceinline__ float by_448(float v) {
    if (!(v >= 0x1p-80f && v <= 0x1p120f)) return __fdiv_rn(v, 448.0f);
    const float q = v * (1.0f / 448.0f);
    return fmaf(fmaf(-448.0f, q, v), 1.0f / 448.0f, q);
}
__device__ __forceinline__ float larger(float a, float b) {  // a NaN stays
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The block's values (ROOT: their roots, which are >= 0) in 8 bits: the warp's largest magnitude by 448 is the scale (a NaN
// makes it one), the codes are those of the correctly rounded root and quotient.  Both are approximated first, to within
// 2^-21 together with the scale's inverse, once from below and once from above: where the two codes differ, a border
// between codes is that near (one value in some 10^5), and the exact operations are run.  ROOT: values above
// zero keep at least the smallest code; so where a code is 0, they are run too.
template <bool ROOT, bool WHOLE>
__device__ __forceinline__ void hold(const Pair (&f)[4], uint8_t* codes, float* scale, int left) {
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int j = (k >> 1) * 128 + (k & 1) * 2;
        if (WHOLE || j < left) top = larger(top, fabsf(f[k].f.x));
        if (WHOLE || j + 1 < left) top = larger(top, fabsf(f[k].f.y));
    }
    const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    uint32_t c[4] = {0, 0, 0, 0};
    const float s = by_448(ROOT ? __fsqrt_rn(most) : most);
    if (most != 0.0f) {  // the same for the warp
        const float inverse = inverse_near(s);
        uint32_t differ = s >= 0x1p-50f && s <= 0x1p100f ? 0 : 1;  // outside, the approximations leave the normal numbers
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Pair near = ROOT ? Pair(root_near(f[k].f.x), root_near(f[k].f.y)) : f[k];
            const Pair below = near * Pair(inverse * (1.0f - 0x1p-21f)), above = near * Pair(inverse * (1.0f + 0x1p-21f));
            c[k] = __nv_cvt_float2_to_fp8x2(below.f, __NV_SATFINITE, __NV_E4M3);
            differ |= c[k] ^ __nv_cvt_float2_to_fp8x2(above.f, __NV_SATFINITE, __NV_E4M3);
        }
        if (ROOT) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t word = c[2 * q] | c[2 * q + 1] << 16;
                differ |= (word - 0x01010101u) & ~word & 0x80808080u;  // a byte that is 0
            }
        }
        if (differ) {
            const float by = s > 0.0f ? s : 1.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 q = f[k].f;
                if (ROOT) q = make_float2(__fsqrt_rn(q.x), __fsqrt_rn(q.y));
                c[k] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(q.x, by), __fdiv_rn(q.y, by)), __NV_SATFINITE, __NV_E4M3);
                if (ROOT && (c[k] & 0xff) == 0 && f[k].f.x > 0.0f) c[k] |= 1;
                if (ROOT && c[k] >> 8 == 0 && f[k].f.y > 0.0f) c[k] |= 0x100;
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const uint32_t word = c[2 * q] | c[2 * q + 1] << 16;
        if (WHOLE) {
            __stcs(reinterpret_cast<uint32_t*>(codes + q * 128), word);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (q * 128 + j < left) codes[q * 128 + j] = (uint8_t)(word >> (8 * j));
        }
    }
    if ((threadIdx.x & 31) == 0) *scale = s;
}

// The arrays of a chunk: uniform for a block of threads, who add 32-bit offsets.  TS: what parameters are read from, their
// own type or the fp32 masters.
template <typename T, typename TS, typename TG>
struct Chunk {
    const TS* source;
    T* param;
    float* master;
    const TG* grad;
    void *first, *second;
    float *first_scale, *second_scale;
};

// What a lane reads of a whole block, raw: the next block's is on its way while this one is computed.
template <int BITS, typename TS, typename TG>
struct Lane {
    template <typename V>
    using Words = rows::Vec<V, 4 * (int)sizeof(V)>;
    Words<TS> source[2];
    Words<TG> grad[2];
    Words<float> first[BITS == 32 ? 2 : 1], second[BITS == 32 ? 2 : 1];
    uint32_t first_code[2], second_code[2];
    float first_scale, second_scale;
    template <typename V>
    static __device__ __forceinline__ void words(Words<V>& to, const V* p) {
        to.raw = *reinterpret_cast<const typename Words<V>::Raw*>(p);
    }
    template <typename C>
    __device__ __forceinline__ void load(const C& c, uint32_t block) {
        const uint32_t i = block * kBlock + (threadIdx.x & 31) * 4;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            words<TS>(source[q], c.source + i + q * 128);
            words<TG>(grad[q], c.grad + i + q * 128);
            if constexpr (BITS == 32) {
                words<float>(first[q], static_cast<const float*>(c.first) + i + q * 128);
                words<float>(second[q], static_cast<const float*>(c.second) + i + q * 128);
            } else {
                first_code[q] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c.first) + i + q * 128);
                second_code[q] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c.second) + i + q * 128);
            }
        }
        if constexpr (BITS == 8) first_scale = c.first_scale[block], second_scale = c.second_scale[block];
    }
    // Of a block whose end is the tensor's, or off the 16-byte grid: `left` elements from the lane's first on.
    template <typename C>
    __device__ __forceinline__ void load_some(const C& c, uint32_t block, int left) {
        const uint32_t i = block * kBlock + (threadIdx.x & 31) * 4;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if constexpr (BITS == 8) first_code[q] = second_code[q] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool there = q * 128 + j < left;
                const uint32_t at = i + q * 128 + j;
                source[q].v[j] = there ? c.source[at] : rows::from_float<TS>(0.0f);
                grad[q].v[j] = there ? c.grad[at] : rows::from_float<TG>(0.0f);
                if constexpr (BITS == 32) {
                    first[q].v[j] = there ? static_cast<const float*>(c.first)[at] : 0.0f;
                    second[q].v[j] = there ? static_cast<const float*>(c.second)[at] : 0.0f;
                } else if (there) {
                    first_code[q] |= (uint32_t)static_cast<const uint8_t*>(c.first)[at] << (8 * j);
                    second_code[q] |= (uint32_t)static_cast<const uint8_t*>(c.second)[at] << (8 * j);
                }
            }
        }
        if constexpr (BITS == 8) first_scale = c.first_scale[block], second_scale = c.second_scale[block];
    }
};
template <typename V>
__device__ __forceinline__ Pair pair_of(const V& words, int k) {
    return Pair(rows::to_float(words.v[2 * k]), rows::to_float(words.v[2 * k + 1]));
}

// The step of a lane's 8 values of a block, 4 at a time up to the states.
template <int BITS, bool WHOLE, typename T, typename TS, typename TG>
__device__ __forceinline__ void advance(const Chunk<T, TS, TG>& c, uint32_t block, int left, const Lane<BITS, TS, TG>& lane,
                                        const Fixed& fixed, const Shared& now) {
    const uint32_t i = block * kBlock + (threadIdx.x & 31) * 4;
    Pair m[4], v[4];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        Pair p[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            Pair &mk = m[q * 2 + k], &vk = v[q * 2 + k];
            if constexpr (BITS == 8) {
                mk = of_codes(lane.first_code[q] >> (16 * k)) * Pair(lane.first_scale);
                vk = of_codes(lane.second_code[q] >> (16 * k)) * Pair(lane.second_scale);
                vk = vk * vk;
            } else {
                mk = pair_of(lane.first[q], k);
                vk = pair_of(lane.second[q], k);
            }
            const Pair g = pair_of(lane.grad[q], k) * Pair(now.factor);
            mk = mk * Pair(fixed.beta1) + g * Pair(fixed.less1);
            vk = vk * Pair(fixed.beta2) + (g * g) * Pair(fixed.less2);
            const Pair root(root_near(vk.f.x), root_near(vk.f.y));
            Pair by = fma(root, Pair(now.over_root), Pair(fixed.eps));
            by = Pair(larger(by.f.x, kLeastBy), larger(by.f.y, kLeastBy));
            p[k] = fma(Pair(-now.rate), mk * Pair(inverse_near(by.f.x), inverse_near(by.f.y)), pair_of(lane.source[q], k) * Pair(now.keep));
        }
        if (c.master) write4<float, WHOLE>(p, c.master + i + q * 128, left - q * 128);
        write4<T, WHOLE>(p, c.param + i + q * 128, left - q * 128);
        if constexpr (BITS == 32) {
            write4<float, WHOLE>(m + q * 2, static_cast<float*>(c.first) + i + q * 128, left - q * 128);
            write4<float, WHOLE>(v + q * 2, static_cast<float*>(c.second) + i + q * 128, left - q * 128);
        }
    }
    if constexpr (BITS == 8) {
        hold<false, WHOLE>(m, static_cast<uint8_t*>(c.first) + i, c.first_scale + block, left);
        hold<true, WHOLE>(v, static_cast<uint8_t*>(c.second) + i, c.second_scale + block, left);
    }
}

// The stages of a block's ring: every array's piece of a stage, brought by bulk copies that need neither registers nor
// warps while they are on their way.
struct Ring {
    uint64_t full[kRing], empty[kRing];
    int abort, status;
};
extern __shared__ __align__(128) uint8_t ring_memory[];

template <typename TS, typename TG>
constexpr int stage_bytes() { return kStage * ((int)sizeof(TS) + (int)sizeof(TG) + 2) + 2 * (kStage / kBlock) * (int)sizeof(float); }

// A block of threads' chunk [from, to).
template <int BITS, typename T, typename TS, typename TG>
__device__ __forceinline__ void step_chunk(const Entry& e, int64_t from, int64_t to, const Fixed& fixed, const Shared* shared) {
    constexpr uint32_t kWarps = kThreads / 32;
    T* const param = static_cast<T*>(e.param) + from;
    float* const master = e.master ? e.master + from : nullptr;
    Chunk<T, TS, TG> c{};
    if constexpr (!std::is_same<T, TS>::value) c.source = master;
    else if constexpr (std::is_same<T, float>::value) c.source = master ? master : param;  // an fp32 parameter may have one too
    else c.source = param;
    c.param = param;
    c.master = master;
    c.grad = static_cast<const TG*>(e.grad) + from;
    c.first = static_cast<char*>(e.first) + from * (BITS / 8);
    c.second = static_cast<char*>(e.second) + from * (BITS / 8);
    if constexpr (BITS == 8) c.first_scale = e.first_scale + from / kBlock, c.second_scale = e.second_scale + from / kBlock;
    const uint32_t length = (uint32_t)(to - from), whole = e.aligned ? length / kBlock : 0, blocks = (length + kBlock - 1) / kBlock;
    Shared now;
    auto read_shared = [&] {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // also where no block is left: not to end before the launch it overlaps
        const volatile Shared* const written = shared;
        now = {written->factor, written->keep, written->rate, written->over_root};
    };
    uint32_t block = threadIdx.x >> 5;
    if constexpr (BITS == 8) {
        const uint32_t stages = whole / kWarps;
        __shared__ Ring ring;
        uint8_t* const memory = ring_memory;
        auto piece = [&](uint32_t stage) {  // the stage's arrays in shared memory
            uint8_t* at = memory + stage % kRing * stage_bytes<TS, TG>();
            Chunk<T, TS, TG> r = c;
            r.source = reinterpret_cast<const TS*>(at);
            at += kStage * sizeof(TS);
            r.grad = reinterpret_cast<const TG*>(at);
            at += kStage * sizeof(TG);
            r.first = at;
            r.second = at + kStage;
            r.first_scale = reinterpret_cast<float*>(at + 2 * kStage);
            r.second_scale = r.first_scale + kWarps;
            return r;
        };
        auto bring = [&](uint32_t stage) {  // one thread
            const Chunk<T, TS, TG> r = piece(stage);
            uint64_t* const bar = &ring.full[stage % kRing];
            const uint32_t i = stage * kStage;
            mbar_arrive_expect_tx(bar, stage_bytes<TS, TG>());
            bulk_load_1d(const_cast<TS*>(r.source), c.source + i, kStage * sizeof(TS), bar);
            bulk_load_1d(const_cast<TG*>(r.grad), c.grad + i, kStage * sizeof(TG), bar);
            bulk_load_1d(r.first, static_cast<const uint8_t*>(c.first) + i, kStage, bar);
            bulk_load_1d(r.second, static_cast<const uint8_t*>(c.second) + i, kStage, bar);
            bulk_load_1d(r.first_scale, c.first_scale + stage * kWarps, kWarps * sizeof(float), bar);
            bulk_load_1d(r.second_scale, c.second_scale + stage * kWarps, kWarps * sizeof(float), bar);
        };
        if (stages) {
            if (threadIdx.x == 0) {
                for (int i = 0; i < kRing; ++i) mbar_init(&ring.full[i], 1), mbar_init(&ring.empty[i], kWarps);
                ring.abort = ring.status = 0;
                fence_barrier_init();
                for (uint32_t stage = 0; stage < min(stages, (uint32_t)kRing); ++stage) bring(stage);
            }
            __syncthreads();
        }
        read_shared();
        for (uint32_t stage = 0; stage < stages; ++stage) {
            const uint32_t slot = stage % kRing, turn = stage / kRing & 1;
            // a wait that gave up makes the parameters NaN
            if (!mbar_wait_timed<false>(&ring.full[slot], turn, &ring.abort, &ring.status)) now.rate = __int_as_float(0x7fc00000);
            Lane<BITS, TS, TG> here;
            here.load(piece(stage), block);
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive(&ring.empty[slot]);
            advance<BITS, true>(c, stage * kWarps + block, kBlock, here, fixed, now);
            // refilled a turn late, when the other warps have long read it
            if (threadIdx.x == 0 && stage > 0 && stage - 1 + kRing < stages) {
                const uint32_t last = stage - 1;
                if (mbar_wait_timed<false>(&ring.empty[last % kRing], last / kRing & 1, &ring.abort, &ring.status)) bring(last + kRing);
            }
        }
        for (block += stages * kWarps; block < whole; block += kWarps) {
            Lane<BITS, TS, TG> here;
            here.load(c, block);
            advance<BITS, true>(c, block, kBlock, here, fixed, now);
        }
    } else {
        Lane<BITS, TS, TG> here, next;
        if (block < whole) here.load(c, block);
        read_shared();
        for (; block < whole; block += kWarps) {
            if (block + kWarps < whole) next.load(c, block + kWarps);
            advance<BITS, true>(c, block, kBlock, here, fixed, now);
            here = next;
        }
    }
    for (; block < blocks; block += kWarps) {
        const int left = (int)(length - block * kBlock) - (int)(threadIdx.x & 31) * 4;  // may be <= 0
        Lane<BITS, TS, TG> here;
        here.load_some(c, block, left);
        advance<BITS, false>(c, block, left, here, fixed, now);
    }
}
template <int BITS, typename T>
__device__ __forceinline__ void step_typed(const Entry& e, int64_t from, int64_t to, const Fixed& fixed, const Shared* shared) {
    if (e.grad_type == HB_F32) {
        if (e.master) step_chunk<BITS, T, float, float>(e, from, to, fixed, shared);
        else step_chunk<BITS, T, T, float>(e, from, to, fixed, shared);
    } else {
        if (e.master) step_chunk<BITS, T, float, T>(e, from, to, fixed, shared);
        else step_chunk<BITS, T, T, T>(e, from, to, fixed, shared);
    }
}

template <int BITS, int MOST>
__global__ void __launch_bounds__(kThreads, BITS == 8 ? 3 : 2) step_kernel(const __grid_constant__ List<MOST> l, const Fixed fixed, const Shared* shared) {
    const Entry& e = l.e[tensor_of(l, blockIdx.x)];
    const int64_t from = (int64_t)((int)blockIdx.x - e.chunk) * l.chunk, to = min(e.size, from + l.chunk);
    if (e.type == HB_F32) step_chunk<BITS, float, float, float>(e, from, to, fixed, shared);
    else if (e.type == HB_F16) step_typed<BITS, __half>(e, from, to, fixed, shared);
    else step_typed<BITS, __nv_bfloat16>(e, from, to, fixed, shared);
}

// ---------------------------------------------------------------- m and v of 8-bit states
constexpr int kHeld = 400;
struct Held {
    const uint8_t *first[kHeld], *second[kHeld];
    const float *first_scale[kHeld], *second_scale[kHeld];
    float *out_first[kHeld], *out_second[kHeld];
    int64_t size[kHeld];
    int32_t chunk[kHeld];
    int count;
};
static_assert(sizeof(Held) < 32000, "kernel parameters");

__global__ void __launch_bounds__(kThreads) moments_kernel(const __grid_constant__ Held l) {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.chunk[mid] <= (int)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const int64_t at = (int64_t)(blockIdx.x - l.chunk[lo]) * kChunk + (threadIdx.x >> 5) * kBlock;
    if (at >= l.size[lo]) return;
    const int64_t i = at + (threadIdx.x & 31) * 4;
    const int left = (int)min((int64_t)kBlock, l.size[lo] - i);
    const uint64_t bits = reinterpret_cast<uintptr_t>(l.first[lo]) | reinterpret_cast<uintptr_t>(l.second[lo]) |
                          reinterpret_cast<uintptr_t>(l.out_first[lo]) | reinterpret_cast<uintptr_t>(l.out_second[lo]);
    const float ms = l.first_scale[lo][at / kBlock], vs = l.second_scale[lo][at / kBlock];
    auto go = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value != 0;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            uint32_t mc = 0, vc = 0;
            const uint8_t *first = l.first[lo] + i + q * 128, *second = l.second[lo] + i + q * 128;
            if (WHOLE) {
                mc = *reinterpret_cast<const uint32_t*>(first);
                vc = *reinterpret_cast<const uint32_t*>(second);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (q * 128 + j < left) mc |= (uint32_t)first[j] << (8 * j), vc |= (uint32_t)second[j] << (8 * j);
            }
            Pair m[2], v[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                m[k] = of_codes(mc >> (16 * k)) * Pair(ms);
                v[k] = of_codes(vc >> (16 * k)) * Pair(vs);
                v[k] = v[k] * v[k];
            }
            write4<float, WHOLE>(m, l.out_first[lo] + i + q * 128, left - q * 128);
            write4<float, WHOLE>(v, l.out_second[lo] + i + q * 128, left - q * 128);
        }
    };
    if (at + kBlock <= l.size[lo] && (bits & 15) == 0) go(rows::Bytes<1>{});
    else go(rows::Bytes<0>{});
}

int finish(cudaError_t e, const char* what) {
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
}

constexpr int kMostStage = stage_bytes<float, float>();
template <int BITS, int MOST>
cudaError_t run(int64_t count, void* const* params, const void* const* grads, void* const* first, void* const* second,
                float* const* first_scale, float* const* second_scale, float* const* master, const int64_t* sizes,
                const int32_t* types, const int32_t* grad_types, int chunk, const Fixed& fixed, const Shared* shared, cudaStream_t st) {
    List<MOST> l;
    l.chunk = chunk;
    bool overlap = true;  // the first launch follows begin_kernel, the others a launch that writes
    for (int64_t from = 0; from < count; from += MOST) {
        l.count = 0;
        int64_t chunks = 0;
        int ring = 0;  // bytes of a stage
        for (int64_t i = from; i < std::min(count, from + MOST); ++i) {
            if (sizes[i] == 0) continue;
            Entry& e = l.e[l.count++];
            e.param = params[i];
            e.grad = grads[i];
            e.first = first[i];
            e.second = second[i];
            e.first_scale = BITS == 8 ? first_scale[i] : nullptr;
            e.second_scale = BITS == 8 ? second_scale[i] : nullptr;
            e.master = master ? master[i] : nullptr;
            e.size = sizes[i];
            e.chunk = (int32_t)chunks;
            e.type = (uint8_t)types[i];
            e.grad_type = (uint8_t)grad_types[i];
            e.aligned = ((rows::address_bits(e.param) | rows::address_bits(e.grad) | rows::address_bits(e.first) |
                          rows::address_bits(e.second) | rows::address_bits(e.master) | rows::address_bits(e.first_scale) |
                          rows::address_bits(e.second_scale)) & 15) == 0;
            ring = std::max(ring, kStage * ((e.master ? 4 : rows::type_bytes(e.type)) + rows::type_bytes(e.grad_type) + 2) +
                                      2 * (kStage / kBlock) * (int)sizeof(float));
            chunks += (sizes[i] + chunk - 1) / chunk;
        }
        if (l.count == 0) continue;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3((unsigned)chunks);
        config.blockDim = dim3(kThreads);
        config.dynamicSmemBytes = BITS == 8 ? (size_t)kRing * ring : 0;
        config.stream = st;
        config.attrs = &attr;
        config.numAttrs = overlap ? 1 : 0;
        overlap = false;
        cudaError_t e = cudaSuccess;
        if (BITS == 8) e = cudaFuncSetAttribute(step_kernel<BITS, MOST>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing * kMostStage);
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&config, step_kernel<BITS, MOST>, l, fixed, shared);
        count_launches(1);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

bool bad(const void* p, size_t size) { return !p || rows::address_bits(p) % size; }

}  // namespace adamw
}  // namespace hb

using namespace hb;
using namespace hb::adamw;

extern "C" size_t hb_adamw_workspace(void) { return sizeof(Shared); }

extern "C" int hb_adamw_step(int64_t count, void* const* params, const void* const* grads, void* const* first, void* const* second,
                             float* const* first_scale, float* const* second_scale, float* const* master, const int64_t* sizes,
                             const int32_t* types, const int32_t* grad_types, int bits, const hb_adamw_rule* rule, int32_t* step,
                             void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "hb_adamw_step";
    if (count < 0 || count > INT32_MAX || (bits != 8 && bits != 32)) return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: number of tensors or bits");
    if (!rule || bad(step, 4) || (count > 0 && (!params || !grads || !first || !second || !sizes || !types || !grad_types ||
                                                (bits == 8 && (!first_scale || !second_scale)))))
        return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: null pointer, or misaligned step");
    if (!(rule->beta1 >= 0.0 && rule->beta1 < 1.0 && rule->beta2 >= 0.0 && rule->beta2 < 1.0) || !(rule->eps >= 0.0 && rule->eps <= 1e30) ||
        !(rule->decay >= 0.0) || (!rule->rate && !(rule->lr >= 0.0)) || (rule->norm && !(rule->max_norm >= 0.0)))
        return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: betas in [0, 1), eps in [0, 1e30], the other numbers >= 0");
    if ((rule->rate && bad(rule->rate, 4)) || (rule->norm && bad(rule->norm, 4)))
        return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: misaligned rate or norm");
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (sizes[i] < 0 || !rows::valid_type(types[i]) || (grad_types[i] != types[i] && grad_types[i] != HB_F32))
            return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: size of a tensor, or a gradient neither of its type nor fp32");
        if (sizes[i] == 0) continue;
        if (bad(params[i], rows::type_bytes(types[i])) || bad(grads[i], rows::type_bytes(grad_types[i])) ||
            bad(first[i], bits == 8 ? 1 : 4) || bad(second[i], bits == 8 ? 1 : 4) || (master && rows::address_bits(master[i]) % 4) ||
            (bits == 8 && (bad(first_scale[i], 4) || bad(second_scale[i], 4))))
            return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: null or misaligned pointer of a tensor");
        if (sizes[i] > INT32_MAX * (int64_t)kChunk || (chunks += (sizes[i] + kChunk - 1) / kChunk) > INT32_MAX)
            return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: too many elements");
    }
    if (!workspace || rows::address_bits(workspace) % 16) return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: the workspace must be 16-byte aligned");
    if (workspace_bytes < sizeof(Shared)) return abi_fail(HB_WORKSPACE, "workspace smaller than hb_adamw_workspace()");
    const auto st = static_cast<cudaStream_t>(stream);
    Shared* shared = static_cast<Shared*>(workspace);
    begin_kernel<<<1, 1, 0, st>>>(step, rule->norm, rule->rate, rule->lr, rule->beta1, rule->beta2, rule->decay, rule->max_norm, shared);
    count_launches(1);
    cudaError_t e = cudaGetLastError();
    const Fixed fixed{(float)rule->beta1, (float)rule->beta2, (float)(1.0 - rule->beta1), (float)(1.0 - rule->beta2), (float)rule->eps};
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) total += sizes[i];
    const auto go = bits == 8 ? (count <= kFew ? run<8, kFew> : run<8, kMany>) : (count <= kFew ? run<32, kFew> : run<32, kMany>);
    if (e == cudaSuccess)
        e = go(count, params, grads, first, second, first_scale, second_scale, master, sizes, types, grad_types,
               total < kLongLeast ? kChunk : kLongChunk, fixed, shared, st);
    return finish(e, what);
}

extern "C" int hb_adamw_moments(int64_t count, const void* const* first, const void* const* second, const float* const* first_scale,
                                const float* const* second_scale, const int64_t* sizes, float* const* out_first,
                                float* const* out_second, void* stream) {
    const char* what = "hb_adamw_moments";
    if (count < 0 || count > INT32_MAX ||
        (count > 0 && (!first || !second || !first_scale || !second_scale || !sizes || !out_first || !out_second)))
        return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_moments: number of tensors or null pointer");
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (sizes[i] < 0 || sizes[i] > INT32_MAX * (int64_t)kChunk || (chunks += (sizes[i] + kChunk - 1) / kChunk) > INT32_MAX)
            return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_moments: size of a tensor");
        if (sizes[i] > 0 && (bad(first[i], 1) || bad(second[i], 1) || bad(first_scale[i], 4) || bad(second_scale[i], 4) ||
                             bad(out_first[i], 4) || bad(out_second[i], 4)))
            return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_moments: null or misaligned pointer of a tensor");
    }
    const auto st = static_cast<cudaStream_t>(stream);
    for (int64_t from = 0; from < count; from += kHeld) {
        Held l;
        l.count = 0;
        int32_t at = 0;
        for (int64_t i = from; i < std::min(count, from + kHeld); ++i) {
            if (sizes[i] == 0) continue;
            const int t = l.count++;
            l.first[t] = static_cast<const uint8_t*>(first[i]);
            l.second[t] = static_cast<const uint8_t*>(second[i]);
            l.first_scale[t] = first_scale[i];
            l.second_scale[t] = second_scale[i];
            l.out_first[t] = out_first[i];
            l.out_second[t] = out_second[i];
            l.size[t] = sizes[i];
            l.chunk[t] = at;
            at += (int32_t)((sizes[i] + kChunk - 1) / kChunk);
        }
        if (l.count == 0) continue;
        moments_kernel<<<(unsigned)at, kThreads, 0, st>>>(l);
        count_launches(1);
    }
    return finish(cudaGetLastError(), what);
}
