// The global norm of many gradients, and the gradients scaled down to a limit.
//
//   norm = sqrt(sum over all tensors of g^2),  f = min(1, limit / (norm + 1e-6)),  out = f g
//
// Two launches over one list of chunks: the first leaves one fp64 sum of squares a
// block, the second adds those in order in every block, so nothing waits on an
// atomic and the result does not depend on the launch.  Bound by HBM: g is read
// twice and written once.  The second launch goes through the chunks backwards, so
// that it finds in L2 what the first read last.  Up to half a million elements the
// time is launches: one cluster of blocks does both steps in one, with its hardware
// barrier between them.  From 8 million on the second launch has a block a chunk: blocks
// that start in the order of memory keep HBM's pages open, where resident blocks that
// stride through it drift apart (1.6 GB copied and scaled: 471 us against 541).  The
// norm is then a launch of its own, so that a block begins with its loads.
//
// Measured on a B200: 800 million bf16 values 711 us (2 reads and a write: 6.7 TB/s), their
// norm alone 258 us (6.2 TB/s); 200 thousand f32 values 7 us.
//
// Squares are added in fp32 over at most 32 values and in fp64 from there on.  A
// group whose fp32 sum is so small or so large that squares were lost or overflowed
// is added again in fp64, so the norm of finite gradients is finite wherever fp32
// can hold it.
#include <algorithm>
#include <cmath>
#include <string>

#include <cooperative_groups.h>

#include "internal.h"
#include "rows.cuh"

namespace hb {
namespace clip {

constexpr int kThreads = 256, kSmallThreads = 512;
constexpr int64_t kChunk = 8192, kSmallChunk = 8192;  // elements; small: 4 loads a thread of fp32
// Elements of the one-launch form.  A call waited for, and a call among others (us): 2^18 f32 values 20.7 and 8.3 in one
// launch, 20.7 and 11.3 in two; 2^19 23.5 and 12.3 against 20.5 and 11.3; 2^20 28.8 and 17.3 against 20.6 and 11.3.
constexpr int64_t kSmallMost = 1 << 19;
constexpr int kCluster = 16;
// Elements from which a block scales one chunk.  As above, without and with it: 2^22 f32 25.0 and 12.4 against 27.2 and
// 14.6; 2^23 31.5 and 18.5 against 31.7 and 20.5 in f32, 28.7 and 16.4 against 28.2 and 15.7 in bf16.  On the device alone
// 2^25 bf16 values take 38 us without and 30 with it.
constexpr int64_t kLargeLeast = 1 << 23, kLargeChunk = 16384;
constexpr int kMostBlocks = 148 * 8;
constexpr double kEps = 1e-6;

// A list of tensors in the kernel's parameters: no copy to the device.
template <int MOST>
struct List {
    const void* in[MOST];
    void* out[MOST];
    int64_t size[MOST];
    int32_t first[MOST + 1];  // first chunk of each tensor
    uint8_t type[MOST], out_type[MOST];
    int count, chunk;  // tensors, elements a chunk
};
constexpr int kFew = 64, kMany = 1024;  // 1.9 KB and 30 KB of parameters (32 KB is the most)

template <int MOST>
__device__ __forceinline__ int tensor_of(const List<MOST>& l, int chunk) {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / 32];
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double r = 0.0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) r += part[i];
    return r;
}

// Sum of squares of n values: fp32, or fp64 where fp32 would lose them.
template <int N>
__device__ __forceinline__ double squares(const float (&f)[N]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(f[i], f[i], s);
    if (s >= 1e-24f && s <= 3e38f) return (double)s;
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) d = fma((double)f[i], (double)f[i], d);
    return d;
}

// WRITTEN: the kernel writes the values in place later, which rules out the read-only path (800 million bf16 values
// take 258 us through it against 269).
template <int THREADS, bool WRITTEN, typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int n) {
    using V = rows::Vec<T, 16>;
    constexpr int U = 4;
    double sum = 0.0;
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        const int whole = n / V::N;
        for (int i = threadIdx.x; i < whole; i += THREADS * U) {
            V v[U];
            float f[U * V::N];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const T* at = p + (int64_t)(i + u * THREADS) * V::N;
                if (i + u * THREADS >= whole) v[u].zero();
                else if (WRITTEN) v[u].raw = *reinterpret_cast<const uint4*>(at);
                else v[u].load(at);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < V::N; ++j) f[u * V::N + j] = rows::to_float(v[u].v[j]);
            sum += squares(f);
        }
        done = whole * V::N;
    }
    for (int i = done + threadIdx.x; i < n; i += THREADS) {
        const float f[1] = {rows::to_float(p[i])};
        sum += squares(f);
    }
    return sum;
}

// This block's sum of squares.
template <int THREADS, bool WRITTEN, int MOST>
__device__ __forceinline__ double list_squares(const List<MOST>& l) {
    double sum = 0.0;
    for (int chunk = blockIdx.x; chunk < l.first[l.count]; chunk += gridDim.x) {
        const int t = tensor_of(l, chunk);
        const int64_t at = (int64_t)(chunk - l.first[t]) * l.chunk;
        const int n = (int)min((int64_t)l.chunk, l.size[t] - at);
        if (l.type[t] == HB_F32) sum += chunk_squares<THREADS, WRITTEN>(static_cast<const float*>(l.in[t]) + at, n);
        else if (l.type[t] == HB_F16) sum += chunk_squares<THREADS, WRITTEN>(static_cast<const __half*>(l.in[t]) + at, n);
        else sum += chunk_squares<THREADS, WRITTEN>(static_cast<const __nv_bfloat16*>(l.in[t]) + at, n);
    }
    return block_sum<THREADS>(sum);
}

template <int MOST>
__global__ void __launch_bounds__(kThreads) square_kernel(const __grid_constant__ List<MOST> l, double* __restrict__ partial) {
    const double sum = list_squares<kThreads, false>(l);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__device__ __forceinline__ double total_norm(const double* partial, int partials) {
    double s = 0.0;
    for (int i = threadIdx.x; i < partials; i += kThreads) s += partial[i];
    return sqrt(block_sum<kThreads>(s));
}

__device__ __forceinline__ float factor_of(double norm, double limit) {
    const double r = limit / (norm + kEps);
    return r >= 1.0 ? 1.0f : (float)r;  // a NaN stays
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* __restrict__ partial, int partials, double limit,
                                                        float* __restrict__ norm, float* __restrict__ factor) {
    const double n = total_norm(partial, partials);
    if (threadIdx.x == 0) {
        *norm = (float)n;
        *factor = factor_of(n, limit);
    }
}

template <int THREADS, typename T, typename TO>
__device__ __forceinline__ void scale_chunk(const T* p, TO* out, int n, float f) {
    constexpr int N = 16 / (int)sizeof(T), kPieces = N * (int)sizeof(TO) / 16;
    using V = rows::Vec<T, 16>;
    using O = rows::Vec<TO, 16>;
    constexpr int U = 4;
    int done = 0;
    if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(out)) & 15) == 0) {
        const int whole = n / N;
        for (int i = threadIdx.x; i < whole; i += THREADS * U) {
            V v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * THREADS < whole) v[u].raw = *reinterpret_cast<const uint4*>(p + (int64_t)(i + u * THREADS) * N);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * THREADS < whole) {
#pragma unroll
                    for (int q = 0; q < kPieces; ++q) {
                        O o;
#pragma unroll
                        for (int j = 0; j < O::N; ++j)
                            o.v[j] = rows::from_float<TO>(f * rows::to_float(v[u].v[q * O::N + j]));
                        o.store_once(out + (int64_t)(i + u * THREADS) * N + q * O::N);
                    }
                }
        }
        done = whole * N;
    }
    for (int i = done + threadIdx.x; i < n; i += THREADS) out[i] = rows::from_float<TO>(f * rows::to_float(p[i]));
}

template <int THREADS, int MOST>
__device__ __forceinline__ void scale_one(const List<MOST>& l, int chunk, float f) {
    const int t = tensor_of(l, chunk);
    if (f == 1.0f && l.in[t] == l.out[t]) return;
    const int64_t at = (int64_t)(chunk - l.first[t]) * l.chunk;
    const int m = (int)min((int64_t)l.chunk, l.size[t] - at);
    const int type = l.type[t], to = l.out_type[t];
    if (type == HB_F32) {
        scale_chunk<THREADS>(static_cast<const float*>(l.in[t]) + at, static_cast<float*>(l.out[t]) + at, m, f);
    } else if (type == HB_F16) {
        const __half* p = static_cast<const __half*>(l.in[t]) + at;
        if (to == HB_F32) scale_chunk<THREADS>(p, static_cast<float*>(l.out[t]) + at, m, f);
        else scale_chunk<THREADS>(p, static_cast<__half*>(l.out[t]) + at, m, f);
    } else {
        const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(l.in[t]) + at;
        if (to == HB_F32) scale_chunk<THREADS>(p, static_cast<float*>(l.out[t]) + at, m, f);
        else scale_chunk<THREADS>(p, static_cast<__nv_bfloat16*>(l.out[t]) + at, m, f);
    }
}

template <int MOST>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ List<MOST> l,
                                                         const double* __restrict__ partial, int partials, double limit,
                                                         float* __restrict__ norm) {
    const double n = total_norm(partial, partials);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const float f = factor_of(n, limit);
    for (int chunk = l.first[l.count] - 1 - blockIdx.x; chunk >= 0; chunk -= gridDim.x) scale_one<kThreads>(l, chunk, f);
}

// A block a chunk; the factor is norm_kernel's.
template <int MOST>
__global__ void __launch_bounds__(kThreads) scale_large_kernel(const __grid_constant__ List<MOST> l,
                                                               const float* __restrict__ factor) {
    scale_one<kThreads>(l, l.first[l.count] - 1 - blockIdx.x, *factor);
}

// Both steps in one cluster.  A block takes the same chunks in both, and no other block's, so nothing that it writes in
// place is another block's to read.
__global__ void __launch_bounds__(kSmallThreads) clip_small_kernel(const __grid_constant__ List<kFew> l, int scale, double limit,
                                                              float* __restrict__ norm) {
    namespace cg = cooperative_groups;
    __shared__ double mine, all;
    cg::cluster_group cluster = cg::this_cluster();
    const double sum = list_squares<kSmallThreads, true>(l);
    if (threadIdx.x == 0) mine = sum;
    cluster.sync();
    if (threadIdx.x < 32) {
        double s = threadIdx.x < kCluster ? *cluster.map_shared_rank(&mine, threadIdx.x) : 0.0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (threadIdx.x == 0) all = s;
    }
    __syncthreads();
    // a block stays until the others have read its sum; nothing else is handed over
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const double n = sqrt(all);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    if (scale) {
        const float f = factor_of(n, limit);
        for (int chunk = blockIdx.x; chunk < l.first[l.count]; chunk += gridDim.x) scale_one<kSmallThreads>(l, chunk, f);
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// The tensors from..to of the caller's list that hold elements.
template <int MOST>
int fill(List<MOST>& l, int64_t chunk, int64_t from, int64_t to, const void* const* in, const int64_t* size,
         const int32_t* type, void* const* out, const int32_t* out_type) {
    l.count = 0;
    l.chunk = (int)chunk;
    int64_t chunks = 0;
    for (int64_t i = from; i < to; ++i) {
        if (size[i] == 0) continue;
        const int t = l.count++;
        l.in[t] = in[i];
        l.out[t] = out ? out[i] : nullptr;
        l.size[t] = size[i];
        l.type[t] = (uint8_t)type[i];
        l.out_type[t] = (uint8_t)(out ? out_type[i] : type[i]);
        l.first[t] = (int32_t)chunks;
        chunks += (size[i] + chunk - 1) / chunk;
    }
    l.first[l.count] = (int32_t)chunks;
    return (int)chunks;
}

inline int blocks_of(int chunks) { return std::max(1, std::min(chunks, kMostBlocks)); }

template <int MOST>
cudaError_t run(int64_t count, const void* const* in, const int64_t* size, const int32_t* type, void* const* out,
                const int32_t* out_type, double limit, bool large, float* norm, float* factor, double* partial,
                cudaStream_t st) {
    List<MOST> l;
    const int64_t chunk = large ? kLargeChunk : kChunk;
    int partials = 0;
    for (int64_t from = 0; from < count || from == 0; from += MOST) {
        const int blocks = blocks_of(fill(l, chunk, from, std::min(count, from + MOST), in, size, type, out, out_type));
        square_kernel<MOST><<<blocks, kThreads, 0, st>>>(l, partial + partials);
        count_launches(1);
        partials += blocks;
    }
    if (!out || large) {
        norm_kernel<<<1, kThreads, 0, st>>>(partial, partials, limit, norm, factor);
        count_launches(1);
        if (!out) return cudaGetLastError();
    }
    for (int64_t from = 0; from < count || from == 0; from += MOST) {
        if (count > MOST) fill(l, chunk, from, std::min(count, from + MOST), in, size, type, out, out_type);
        const int chunks = l.first[l.count];
        if (chunks == 0 && large) continue;
        if (large) scale_large_kernel<MOST><<<chunks, kThreads, 0, st>>>(l, factor);
        else scale_kernel<MOST><<<blocks_of(chunks), kThreads, 0, st>>>(l, partial, partials, limit, norm);
        count_launches(1);
    }
    return cudaGetLastError();
}

int check(int64_t count, const void* const* in, const int64_t* size, const int32_t* type, const float* norm,
          const void* ws, size_t ws_bytes) {
    if (count < 0 || count > INT32_MAX) return abi_fail(HB_BAD_ARGUMENT, "gradient norm: number of tensors out of range");
    if (!norm || !ws || (count > 0 && (!in || !size || !type)))
        return abi_fail(HB_BAD_ARGUMENT, "gradient norm: null pointer");
    if (rows::address_bits(norm) % sizeof(float)) return abi_fail(HB_BAD_ARGUMENT, "gradient norm: misaligned pointer");
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (size[i] < 0 || !rows::valid_type(type[i]) || (size[i] > 0 && !in[i]) ||
            rows::address_bits(in[i]) % rows::type_bytes(type[i]))
            return abi_fail(HB_BAD_ARGUMENT, "gradient norm: size, type or pointer of a tensor");
        if (size[i] > INT32_MAX * kChunk || (chunks += (size[i] + kChunk - 1) / kChunk) > INT32_MAX)
            return abi_fail(HB_BAD_ARGUMENT, "gradient norm: too many elements");
    }
    if (rows::address_bits(ws) % 256) return abi_fail(HB_BAD_ARGUMENT, "gradient norm: the workspace must be 256-byte aligned");
    if (ws_bytes < hb_clip_workspace(count)) return abi_fail(HB_WORKSPACE, "workspace smaller than hb_clip_workspace()");
    return HB_OK;
}

int start(int64_t count, const void* const* in, const int64_t* size, const int32_t* type, void* const* out,
          const int32_t* out_type, double limit, float* norm, void* ws, void* stream) {
    const auto st = static_cast<cudaStream_t>(stream);
    double* partial = static_cast<double*>(ws) + 1;  // after the factor
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) total += size[i];
    cudaError_t e = cudaSuccess;
    if (count <= kFew && total <= kSmallMost) {
        List<kFew> l;
        fill(l, kSmallChunk, 0, count, in, size, type, out, out_type);
        e = cudaFuncSetAttribute(clip_small_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = kCluster;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(kCluster);
        config.blockDim = dim3(kSmallThreads);
        config.stream = st;
        config.attrs = &attr;
        config.numAttrs = 1;
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&config, clip_small_kernel, l, out != nullptr ? 1 : 0, limit, norm);
        count_launches(1);
        return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("gradient norm: ") + cudaGetErrorString(e));
    }
    const auto go = count <= kFew ? run<kFew> : run<kMany>;
    float* factor = static_cast<float*>(ws);
    e = go(count, in, size, type, out, out_type, limit, total >= kLargeLeast, norm, factor, partial, st);
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("gradient norm: ") + cudaGetErrorString(e));
}

}  // namespace clip
}  // namespace hb

using namespace hb;
using namespace hb::clip;

extern "C" size_t hb_clip_workspace(int64_t count) {
    if (count < 0) return 0;
    return sizeof(double) * (1 + kMostBlocks * (size_t)std::max<int64_t>(1, (count + kMany - 1) / kMany));
}

extern "C" int hb_grad_norm(int64_t count, const void* const* grads, const int64_t* sizes, const int32_t* types,
                            float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check(count, grads, sizes, types, norm, workspace, workspace_bytes);
    if (rc) return rc;
    return start(count, grads, sizes, types, nullptr, nullptr, 0.0, norm, workspace, stream);
}

extern "C" int hb_clip_grad_norm(int64_t count, const void* const* grads, const int64_t* sizes, const int32_t* types,
                                 void* const* outs, const int32_t* out_types, double limit, float* norm,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check(count, grads, sizes, types, norm, workspace, workspace_bytes);
    if (rc) return rc;
    if (!(limit >= 0.0)) return abi_fail(HB_BAD_ARGUMENT, "gradient clipping: the limit must be a number >= 0");
    if (count > 0 && (!outs || !out_types)) return abi_fail(HB_BAD_ARGUMENT, "gradient clipping: null pointer");
    for (int64_t i = 0; i < count; ++i)
        if (sizes[i] > 0 && (!outs[i] || (out_types[i] != types[i] && out_types[i] != HB_F32) ||
                             rows::address_bits(outs[i]) % rows::type_bytes(out_types[i])))
            return abi_fail(HB_BAD_ARGUMENT, "gradient clipping: an output has its gradient's type or is fp32");
    static void* const none[1] = {nullptr};
    static const int32_t any[1] = {HB_F32};
    return start(count, grads, sizes, types, count > 0 ? outs : none, count > 0 ? out_types : any, limit, norm, workspace,
                 stream);
}
