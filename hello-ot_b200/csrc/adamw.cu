// One AdamW step over many tensors, with fp32 states or states in 8 bits.
//
//   g' = f g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
//   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Two launches over one list of chunks in the kernel's parameters: one thread counts the step and works out what
// all elements share (in fp64: t, the bias corrections, f), then warps go through blocks of 256 elements, 8 a lane.
// The second launch starts while the first runs and waits for it when its first loads are on their way
// (programmatic dependent launch).  Bound by HBM: every array passes once.
//
// 8 bits: e4m3 codes of m and of sqrt(v) with a scale for each 256 elements (largest magnitude / 448).  The root
// halves v's range of exponents, so e4m3's 2^17 between the largest and the smallest code are 2^34 of v; a v above
// zero keeps at least the smallest code, so that no later step divides an m that was kept by a v that was lost.
// Scales are fp32, not powers of two: a block whose values all shrink by the same factor keeps its codes and
// shrinks its scale, where rounding each value to its old code would stop v's decay of 0.1 % a step.
//
// m and v are rounded to fp32 at every operation as it is written, and their codes are those of the correctly rounded
// quotients, so that any fp32 program computes the same states bit for bit.  The change of p takes the approximate
// root and quotient (2^-20 of the change): with the exact ones, 3 quotients and a root an element, the kernel was bound
// by instructions (400 million bf16 parameters, 8 bits: 2.46 ms of 0.86 at the copy rate).
#include <algorithm>
#include <cmath>
#include <string>

#include <cuda_fp8.h>

#include "internal.h"
#include "rows.cuh"

namespace hb {
namespace adamw {

constexpr int kThreads = 256, kBlock = 256, kChunk = 2048;  // elements: of a scale, of a block of threads (a scale a warp)
constexpr int kMost8 = 280, kMost32 = 330;                   // tensors of a launch: 32 KB of parameters

template <int MOST>
struct List {
    void* param[MOST];
    const void* grad[MOST];
    void *first[MOST], *second[MOST];
    float* master[MOST];
    int64_t size[MOST];
    int32_t chunk[MOST + 1];  // first chunk of each tensor
    uint8_t type[MOST], grad_type[MOST];
    int count;
};
struct Scales {  // of a list's tensors; 8-bit states
    float *first[kMost8], *second[kMost8];
};
struct NoScales {};
static_assert(sizeof(List<kMost8>) + sizeof(Scales) < 32000 && sizeof(List<kMost32>) < 32000, "kernel parameters");

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
        if (l.chunk[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// A lane's 8 values, `left` of them there; VECTORS: all of them, on 16 bytes.
template <typename T>
__device__ __forceinline__ void read8(float (&f)[8], const T* p, int left, bool vectors) {
    if (vectors) {
        constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
        for (int q = 0; q < 8 / N; ++q) {
            rows::Vec<T, 16> v;
            v.raw = *reinterpret_cast<const uint4*>(p + q * N);
#pragma unroll
            for (int j = 0; j < N; ++j) f[q * N + j] = rows::to_float(v.v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = j < left ? rows::to_float(p[j]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void write8(const float (&f)[8], T* p, int left, bool vectors) {
    if (vectors) {
        constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
        for (int q = 0; q < 8 / N; ++q) {
            rows::Vec<T, 16> v;
#pragma unroll
            for (int j = 0; j < N; ++j) v.v[j] = rows::from_float<T>(f[q * N + j]);
            v.store_once(p + q * N);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = rows::from_float<T>(f[j]);
    }
}
__device__ __forceinline__ void read_codes(uint8_t (&c)[8], const uint8_t* p, int left, bool vectors) {
    if (vectors) {
        rows::Vec<uint8_t, 8> v;
        v.raw = *reinterpret_cast<const uint2*>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = v.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = j < left ? p[j] : 0;
    }
}
__device__ __forceinline__ void of_codes(float (&f)[8], const uint8_t (&c)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c[j] | c[j + 1] << 8), __NV_E4M3);
        const float2 v = __half22float2(__half2(h));
        f[j] = v.x, f[j + 1] = v.y;
    }
}
// a / b within 2^-21, for any b >= 0 of the range: __fdividef's divisors end at 2^126.
__device__ __forceinline__ float quotient(float a, float b) { return b < 0x1p126f ? __fdividef(a, b) : a / b; }
__device__ __forceinline__ float root_near(float v) {  // within 2^-23 of the root
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// The block's values (ROOT: their roots, which are >= 0) in 8 bits: the warp's largest magnitude by 448 is the scale (a NaN
// makes it one), the codes are those of the correctly rounded root and quotient.  Both are approximated first, to
// within 2^-22 with the scale's inverse: where the codes a little below and above are the same, that is the code, and
// only next to a border between two codes (one value in some 10^5) the exact operations are run.  ROOT: values above
// zero keep at least the smallest code.
template <bool ROOT>
__device__ __forceinline__ void hold(const float (&f)[8], const float (&near)[8], uint8_t* codes, float* scale, int left, bool vectors) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, j < left ? __float_as_uint(fabsf(f[j])) : 0u);
    most = __reduce_max_sync(0xffffffffu, most);
    const float largest = ROOT ? __fsqrt_rn(__uint_as_float(most)) : __uint_as_float(most);
    const float s = __fdiv_rn(largest, 448.0f);
    const float by = s > 0.0f ? s : 1.0f, inverse = __fdiv_rn(1.0f, by);
    const bool plain = by >= 0x1p-100f && by <= 0x1p100f;  // nothing below leaves the normal numbers
    rows::Vec<uint8_t, 8> v;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float q = near[j] * inverse;
        const uint32_t both = __nv_cvt_float2_to_fp8x2(make_float2(fmaf(q, -0x1p-21f, q), fmaf(q, 0x1p-21f, q)), __NV_SATFINITE, __NV_E4M3);
        uint32_t code = both & 0xff;
        if (code != both >> 8 || !plain)
            code = __nv_cvt_float_to_fp8(__fdiv_rn(ROOT ? __fsqrt_rn(f[j]) : f[j], by), __NV_SATFINITE, __NV_E4M3);
        if (ROOT && code == 0 && f[j] > 0.0f) code = 1;
        v.v[j] = (uint8_t)code;
    }
    if (vectors) {
        v.store_once(codes);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) codes[j] = v.v[j];
    }
    if ((threadIdx.x & 31) == 0) *scale = s;
}

// A lane's share of a block of 256 elements that begins at `at`.
template <int BITS, typename T, typename TG, int MOST, typename S>
__device__ __forceinline__ void step_block(const List<MOST>& l, const S& scales, int t, int64_t at, const Fixed& fixed,
                                           const Shared* shared) {
    const int64_t i = at + (threadIdx.x & 31) * 8;
    const int left = (int)min((int64_t)8, l.size[t] - i);  // may be <= 0
    T* param = static_cast<T*>(l.param[t]);
    const TG* grad = static_cast<const TG*>(l.grad[t]);
    float* master = l.master[t];
    const uint64_t bits = reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(master) |
                          reinterpret_cast<uintptr_t>(l.first[t]) | reinterpret_cast<uintptr_t>(l.second[t]);
    const bool vectors = left == 8 && (bits & 15) == 0;
    float p[8], g[8], m[8], v[8];
    uint8_t mc[8], vc[8];
    float ms = 0.0f, vs = 0.0f;
    if (master) read8(p, master + i, left, vectors);
    else read8(p, param + i, left, vectors);
    read8(g, grad + i, left, vectors);
    if constexpr (BITS == 32) {
        read8(m, static_cast<const float*>(l.first[t]) + i, left, vectors);
        read8(v, static_cast<const float*>(l.second[t]) + i, left, vectors);
    } else {
        read_codes(mc, static_cast<const uint8_t*>(l.first[t]) + i, left, vectors);
        read_codes(vc, static_cast<const uint8_t*>(l.second[t]) + i, left, vectors);
        ms = scales.first[t][at / kBlock];
        vs = scales.second[t][at / kBlock];
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const volatile Shared* now = shared;
    const float factor = now->factor, keep = now->keep, rate = now->rate, over_root = now->over_root;
    if constexpr (BITS == 8) {
        of_codes(m, mc);
        of_codes(v, vc);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m[j] = __fmul_rn(m[j], ms);
            v[j] = __fmul_rn(v[j], vs);
            v[j] = __fmul_rn(v[j], v[j]);
        }
    }
    float root[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float gj = __fmul_rn(g[j], factor);
        m[j] = __fadd_rn(__fmul_rn(m[j], fixed.beta1), __fmul_rn(gj, fixed.less1));
        v[j] = __fadd_rn(__fmul_rn(v[j], fixed.beta2), __fmul_rn(__fmul_rn(gj, gj), fixed.less2));
        root[j] = root_near(v[j]);
        p[j] = fmaf(-rate, quotient(m[j], fmaf(root[j], over_root, fixed.eps)), __fmul_rn(p[j], keep));
    }
    if (master) write8(p, master + i, left, vectors);
    write8(p, param + i, left, vectors);
    if constexpr (BITS == 32) {
        write8(m, static_cast<float*>(l.first[t]) + i, left, vectors);
        write8(v, static_cast<float*>(l.second[t]) + i, left, vectors);
    } else {
        hold<false>(m, m, static_cast<uint8_t*>(l.first[t]) + i, scales.first[t] + at / kBlock, left, vectors);
        hold<true>(v, root, static_cast<uint8_t*>(l.second[t]) + i, scales.second[t] + at / kBlock, left, vectors);
    }
}

template <int BITS, int MOST, typename S>
__global__ void __launch_bounds__(kThreads) step_kernel(const __grid_constant__ List<MOST> l, const __grid_constant__ S scales,
                                                        const Fixed fixed, const Shared* shared) {
    const int t = tensor_of(l, blockIdx.x);
    const int64_t at = (int64_t)(blockIdx.x - l.chunk[t]) * kChunk + (threadIdx.x >> 5) * kBlock;
    if (at >= l.size[t]) {  // the launch does not end before the one it overlaps
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const int type = l.type[t], grad = l.grad_type[t];
    if (type == HB_F32) step_block<BITS, float, float>(l, scales, t, at, fixed, shared);
    else if (type == HB_F16 && grad == HB_F16) step_block<BITS, __half, __half>(l, scales, t, at, fixed, shared);
    else if (type == HB_F16) step_block<BITS, __half, float>(l, scales, t, at, fixed, shared);
    else if (grad == HB_BF16) step_block<BITS, __nv_bfloat16, __nv_bfloat16>(l, scales, t, at, fixed, shared);
    else step_block<BITS, __nv_bfloat16, float>(l, scales, t, at, fixed, shared);
}

// ---------------------------------------------------------------- m and v of 8-bit states
struct Held {
    const uint8_t *first[kMost8], *second[kMost8];
    const float *first_scale[kMost8], *second_scale[kMost8];
    float *out_first[kMost8], *out_second[kMost8];
    int64_t size[kMost8];
    int32_t chunk[kMost8 + 1];
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
    const int64_t i = at + (threadIdx.x & 31) * 8;
    const int left = (int)min((int64_t)8, l.size[lo] - i);
    const uint64_t bits = reinterpret_cast<uintptr_t>(l.first[lo]) | reinterpret_cast<uintptr_t>(l.second[lo]) |
                          reinterpret_cast<uintptr_t>(l.out_first[lo]) | reinterpret_cast<uintptr_t>(l.out_second[lo]);
    const bool vectors = left == 8 && (bits & 15) == 0;
    uint8_t mc[8], vc[8];
    float m[8], v[8];
    read_codes(mc, l.first[lo] + i, left, vectors);
    read_codes(vc, l.second[lo] + i, left, vectors);
    const float ms = l.first_scale[lo][at / kBlock], vs = l.second_scale[lo][at / kBlock];
    of_codes(m, mc);
    of_codes(v, vc);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        m[j] = __fmul_rn(m[j], ms);
        v[j] = __fmul_rn(v[j], vs);
        v[j] = __fmul_rn(v[j], v[j]);
    }
    write8(m, l.out_first[lo] + i, left, vectors);
    write8(v, l.out_second[lo] + i, left, vectors);
}

int finish(cudaError_t e, const char* what) {
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
}

template <int BITS, int MOST, typename S>
cudaError_t run(int64_t count, void* const* params, const void* const* grads, void* const* first, void* const* second,
                float* const* first_scale, float* const* second_scale, float* const* master, const int64_t* sizes,
                const int32_t* types, const int32_t* grad_types, const Fixed& fixed, const Shared* shared, cudaStream_t st) {
    List<MOST> l;
    S scales;
    bool overlap = true;  // the first launch follows begin_kernel, the others a launch that writes
    for (int64_t from = 0; from < count; from += MOST) {
        l.count = 0;
        int64_t chunks = 0;
        for (int64_t i = from; i < std::min(count, from + MOST); ++i) {
            if (sizes[i] == 0) continue;
            const int t = l.count++;
            l.param[t] = params[i];
            l.grad[t] = grads[i];
            l.first[t] = first[i];
            l.second[t] = second[i];
            l.master[t] = master ? master[i] : nullptr;
            if constexpr (BITS == 8) scales.first[t] = first_scale[i], scales.second[t] = second_scale[i];
            l.size[t] = sizes[i];
            l.type[t] = (uint8_t)types[i];
            l.grad_type[t] = (uint8_t)grad_types[i];
            l.chunk[t] = (int32_t)chunks;
            chunks += (sizes[i] + kChunk - 1) / kChunk;
        }
        if (l.count == 0) continue;
        l.chunk[l.count] = (int32_t)chunks;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3((unsigned)chunks);
        config.blockDim = dim3(kThreads);
        config.stream = st;
        config.attrs = &attr;
        config.numAttrs = overlap ? 1 : 0;
        overlap = false;
        const cudaError_t e = cudaLaunchKernelEx(&config, step_kernel<BITS, MOST, S>, l, scales, fixed, shared);
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
    if (!(rule->beta1 >= 0.0 && rule->beta1 < 1.0 && rule->beta2 >= 0.0 && rule->beta2 < 1.0) || !(rule->eps >= 0.0) ||
        !(rule->decay >= 0.0) || (!rule->rate && !(rule->lr >= 0.0)) || (rule->norm && !(rule->max_norm >= 0.0)))
        return abi_fail(HB_BAD_ARGUMENT, "hb_adamw_step: betas in [0, 1), the other numbers >= 0");
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
    if (e == cudaSuccess)
        e = bits == 8 ? run<8, kMost8, Scales>(count, params, grads, first, second, first_scale, second_scale, master, sizes, types,
                                               grad_types, fixed, shared, st)
                      : run<32, kMost32, NoScales>(count, params, grads, first, second, first_scale, second_scale, master, sizes, types,
                                                   grad_types, fixed, shared, st);
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
    for (int64_t from = 0; from < count; from += kMost8) {
        Held l;
        l.count = 0;
        int32_t at = 0;
        for (int64_t i = from; i < std::min(count, from + kMost8); ++i) {
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
        l.chunk[l.count] = at;
        moments_kernel<<<(unsigned)at, kThreads, 0, st>>>(l);
        count_launches(1);
    }
    return finish(cudaGetLastError(), what);
}
