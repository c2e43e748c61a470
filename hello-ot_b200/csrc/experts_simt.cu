// Products of rows sorted by expert on the CUDA cores: fp32 rows, and few rows of any type.
//
// fp32 (product_f32): every form of experts.cu in tiles of 128 x 128, 8 of the summed length a step, two steps in
// shared memory; a thread holds 8 x 8 sums and adds products in pairs (fma.rn.f32x2), each rounded like the scalar
// instruction, so the sums are plain fp32 sums.  The tensor cores would need three bf16 parts of each operand and
// cut off the low bits of their running sums, which fp32 results do not allow.  In the gated forms a tile's
// columns are 64 of g and the same 64 of u, and one thread holds both of a place.
//
// Few rows (few_rows, at most 16 of all experts together): one token's step of a decode batch reads the named
// experts' weights once and is bound by that.  A warp streams the weight rows of one output column and multiplies
// them with up to 8 rows of x, which stay in L1; a block of 8 warps takes 8 columns for the rows of one expert,
// which the expert's first row finds out for itself.
#include <algorithm>
#include <string>

#include "experts.cuh"
#include "internal.h"

namespace hb {
namespace experts {
namespace {

// ---------------------------------------------------------------- fp32 tiles
constexpr int BM = 128, BN = 128, BK = 8, kPitch = 132, kThreads = 256;

struct Params {
    const int32_t* offsets;
    int groups, rows, n, k, segments, splits, activation;
    Operand a[2], b[2], dh;
    float* out[2];
    int64_t out_row;
    float* partial;
};

__device__ __forceinline__ uint64_t pack(float a, float b) {
    return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
__device__ __forceinline__ void fma2(uint64_t& c, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}
__device__ __forceinline__ float half_of(uint64_t v, int hi) { return __uint_as_float((uint32_t)(hi ? v >> 32 : v)); }

// Four of an operand tile's 128 x 8 values for this thread: LONG rows run along the summed length, else across it.
// Place i of the tile's 128 is at base + i * row (LONG) or base + i; `lim` of them and `left` of the length are there.
template <bool LONG>
__device__ __forceinline__ void fetch(float (&r)[4], const float* base, int64_t row, int lim, int k0, int left) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = LONG ? t & 7 : (t >> 7) + 2 * i, m = LONG ? (t >> 3) + 32 * i : t & 127;
        r[i] = m < lim && k < left ? __ldg(LONG ? base + m * row + k0 + k : base + (int64_t)(k0 + k) * row + m) : 0.0f;
    }
}
template <bool LONG>
__device__ __forceinline__ void stage(float (*to)[kPitch], const float (&r)[4]) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = LONG ? t & 7 : (t >> 7) + 2 * i, m = LONG ? (t >> 3) + 32 * i : t & 127;
        to[k][m] = r[i];
    }
}

template <int FORM>
__global__ void __launch_bounds__(kThreads, 2) f32_kernel(const __grid_constant__ Params p) {
    constexpr bool HALVES = FORM == kGated || FORM == kGatedGrad;
    constexpr bool A_LONG = FORM != kWeights, B_LONG = FORM != kWeights && FORM != kBack;
    constexpr int COLS = HALVES ? BN / 2 : BN;
    __shared__ __align__(16) float as[2][BK][kPitch], bs[2][BK][kPitch];
    __shared__ int start[kMostGroups + 2], tile[kMostGroups + 2];
    read_groups(p.offsets, p.groups, p.rows, BM, start, tile);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int col = blockIdx.x * COLS;
    int row, lim, length, group, part = 0, split = 0;  // lim: rows of the tile that are the output's
    const float *a0, *b0;
    if (FORM == kWeights) {
        part = blockIdx.z % p.segments;
        group = blockIdx.z / p.segments;
        split = group % p.splits;
        group /= p.splits;
        row = blockIdx.y * BM;
        lim = min(BM, p.n - row);
        int begin, end;
        split_rows(start[group + 1] - start[group], p.splits, split, begin, end);
        length = end - begin;
        begin += start[group];
        a0 = static_cast<const float*>(p.a[part].p) + begin * p.a[part].row + row;
        b0 = static_cast<const float*>(p.b[0].p) + begin * p.b[0].row + col;
    } else {
        if ((int)blockIdx.y >= tile[p.groups + 1]) return;
        group = group_of(tile, p.groups, blockIdx.y);
        row = start[group] + ((int)blockIdx.y - tile[group]) * BM;
        lim = min(BM, start[group + 1] - row);
        length = group == p.groups ? 0 : p.k;
        a0 = b0 = nullptr;
    }
    uint64_t acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0;
    for (int seg = 0; seg < (FORM == kBack ? p.segments : 1) && length > 0; ++seg) {
        int64_t arow, brow;
        int blim = min(COLS, (FORM == kWeights ? p.k : p.n) - col);
        const float* b1 = nullptr;
        if (FORM == kWeights) {
            arow = p.a[part].row;
            brow = p.b[0].row;
        } else {
            arow = p.a[seg].row;
            a0 = static_cast<const float*>(p.a[seg].p) + row * arow;
            brow = p.b[seg].row;
            b0 = static_cast<const float*>(p.b[seg].p) + group * p.b[seg].group + (B_LONG ? col * brow : col);
            if (HALVES) b1 = static_cast<const float*>(p.b[1].p) + group * p.b[1].group + col * p.b[1].row;
        }
        float ra[4], rb[4];
        auto load = [&](int k0) {
            fetch<A_LONG>(ra, a0, arow, lim, k0, length - k0);
            if (HALVES) {  // places 0-63 of the tile are g's columns, 64-127 u's
                const int t = threadIdx.x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = t & 7, m = (t >> 3) + 32 * i, c = m & 63;
                    rb[i] = c < blim && k0 + k < length ? __ldg((m < 64 ? b0 + c * brow : b1 + c * p.b[1].row) + k0 + k) : 0.0f;
                }
            } else {
                fetch<B_LONG>(rb, b0, brow, blim, k0, length - k0);
            }
        };
        load(0);
        stage<A_LONG>(as[0], ra);
        stage<B_LONG>(bs[0], rb);
        __syncthreads();
        int buf = 0;
        for (int k0 = 0; k0 < length; k0 += BK) {
            const bool more = k0 + BK < length;
            if (more) load(k0 + BK);
#pragma unroll
            for (int k = 0; k < BK; ++k) {
                const float4 a_lo = *reinterpret_cast<const float4*>(&as[buf][k][ty * 4]);
                const float4 a_hi = *reinterpret_cast<const float4*>(&as[buf][k][64 + ty * 4]);
                const ulonglong2 b_lo = *reinterpret_cast<const ulonglong2*>(&bs[buf][k][tx * 4]);
                const ulonglong2 b_hi = *reinterpret_cast<const ulonglong2*>(&bs[buf][k][64 + tx * 4]);
                const float av[8] = {a_lo.x, a_lo.y, a_lo.z, a_lo.w, a_hi.x, a_hi.y, a_hi.z, a_hi.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint64_t aa = pack(av[i], av[i]);
                    fma2(acc[i][0], aa, b_lo.x);
                    fma2(acc[i][1], aa, b_lo.y);
                    fma2(acc[i][2], aa, b_hi.x);
                    fma2(acc[i][3], aa, b_hi.y);
                }
            }
            if (more) {
                stage<A_LONG>(as[buf ^ 1], ra);
                stage<B_LONG>(bs[buf ^ 1], rb);
            }
            __syncthreads();
            buf ^= 1;
        }
    }
    float* out = p.out[FORM == kWeights ? part : 0];
    int64_t out_row = p.out_row;
    if (FORM == kWeights) {
        if (p.splits > 1) {
            out = p.partial + (((int64_t)split * p.segments + part) * p.groups + group) * p.n * p.k;
            out_row = p.k;
        } else {
            out += (int64_t)group * p.n * out_row;
        }
    }
    const int width = FORM == kWeights ? p.k : p.n;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int m = (i < 4 ? 0 : 60) + ty * 4 + i;
        if (m >= lim) continue;
        const int64_t r = (int64_t)(row + m) * out_row;
#pragma unroll
        for (int j = 0; j < (HALVES ? 4 : 8); ++j) {
            const int c = col + (j < 4 ? 0 : 60) + tx * 4 + j;
            if (c >= width) continue;
            const float v = half_of(acc[i][j / 2], j & 1);
            if (HALVES) {
                const float u = half_of(acc[i][2 + j / 2], j & 1);
                float slope;
                const float act = activate<true, FORM == kGatedGrad>(p.activation, v, slope);
                if (FORM == kGated) {
                    out[r + c] = length ? act * u : 0.0f;
                } else if (length == 0) {
                    out[r + c] = p.out[1][r + c] = 0.0f;
                } else {
                    const float d = static_cast<const float*>(p.dh.p)[(int64_t)(row + m) * p.dh.row + c];
                    out[r + c] = d * u * slope;
                    p.out[1][r + c] = d * act;
                }
            } else {
                out[r + c] = v;
            }
        }
    }
}

template <int FORM>
cudaError_t launch_f32(const Params& p, cudaStream_t st) {
    const int width = FORM == kWeights ? p.k : p.n, cols = FORM == kGated || FORM == kGatedGrad ? BN / 2 : BN;
    dim3 grid((width + cols - 1) / cols, FORM == kWeights ? (p.n + BM - 1) / BM : p.rows / BM + p.groups + 1,
              FORM == kWeights ? p.splits * p.segments * p.groups : 1);
    if (grid.y > 65535 || grid.z > 65535) return cudaErrorInvalidConfiguration;
    f32_kernel<FORM><<<grid, kThreads, 0, st>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

// ---------------------------------------------------------------- parts of the weights' gradients
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ partial, int splits, int64_t each, int64_t part,
                                                   T* __restrict__ out0, T* __restrict__ out1) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // of segments x part values
    if (i >= each) return;
    float sum = 0.0f;
    for (int s = 0; s < splits; ++s) sum += partial[s * each + i];
    (i < part ? out0 : out1)[i < part ? i : i - part] = rows::from_float<T>(sum);
}

// ---------------------------------------------------------------- few rows
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32, kPass = 8;

struct FewParams {
    const int32_t* offsets;
    int groups, rows, n, k, activation;
    Operand x, w[2];
    void* out;
};

// The first expert whose rows end behind row r (groups: none): with offsets read as their running maximum, the row's.
__device__ __forceinline__ int expert_of(const int32_t* offsets, int groups, int r, int* shared) {
    if (threadIdx.x == 0) *shared = groups;
    __syncthreads();
    for (int e = threadIdx.x; e < groups; e += kFewThreads)
        if (offsets[e + 1] > r) {
            atomicMin(shared, e);
            break;
        }
    __syncthreads();
    const int e = *shared;
    __syncthreads();
    return e;
}

template <typename T, int VB, bool GATED>
__global__ void __launch_bounds__(kFewThreads) few_kernel(const __grid_constant__ FewParams p) {
    using V = rows::Vec<T, VB>;
    __shared__ int found;
    const int r0 = blockIdx.y, lane = threadIdx.x & 31;
    const int col = blockIdx.x * kFewWarps + (threadIdx.x >> 5);
    int e = 0, count = p.rows - r0;
    if (p.offsets) {
        e = expert_of(p.offsets, p.groups, r0, &found);
        if (r0 > 0 && expert_of(p.offsets, p.groups, r0 - 1, &found) == e) return;  // the expert's first row does the work
        if (e < p.groups) count = min(count, p.offsets[e + 1] - r0);
    } else if (r0 > 0) {
        return;
    }
    if (col >= p.n) return;
    T* out = static_cast<T*>(p.out) + (int64_t)r0 * p.n + col;
    if (e == p.groups) {
        for (int r = lane; r < count; r += 32) out[(int64_t)r * p.n] = rows::from_float<T>(0.0f);
        return;
    }
    const T* w0 = static_cast<const T*>(p.w[0].p) + e * p.w[0].group + col * p.w[0].row;
    const T* w1 = GATED ? static_cast<const T*>(p.w[1].p) + e * p.w[1].group + col * p.w[1].row : nullptr;
    for (int r = 0; r < count; r += kPass) {
        const int here = min(kPass, count - r);
        const T* x = static_cast<const T*>(p.x.p) + (r0 + r) * p.x.row;
        float g[kPass], u[kPass];
#pragma unroll
        for (int i = 0; i < kPass; ++i) g[i] = u[i] = 0.0f;
        constexpr int U = 4;  // vectors of each weight row in flight
        for (int k = lane * V::N; k < p.k; k += 32 * V::N * U) {
            V a[U], b[U];
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int at = k + q * 32 * V::N;
                if (at < p.k) {
                    a[q].load_once(w0 + at);
                    if (GATED) b[q].load_once(w1 + at);
                }
            }
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int at = k + q * 32 * V::N;
                if (at >= p.k) break;
#pragma unroll
                for (int i = 0; i < kPass; ++i) {
                    if (i >= here) break;
                    V xv;
                    xv.load(x + i * p.x.row + at);
#pragma unroll
                    for (int j = 0; j < V::N; ++j) {
                        const float xf = rows::to_float(xv.v[j]);
                        g[i] = fmaf(xf, rows::to_float(a[q].v[j]), g[i]);
                        if (GATED) u[i] = fmaf(xf, rows::to_float(b[q].v[j]), u[i]);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
            if (i >= here) break;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                g[i] += __shfl_xor_sync(0xffffffffu, g[i], d);
                if (GATED) u[i] += __shfl_xor_sync(0xffffffffu, u[i], d);
            }
            if (lane == 0) {
                float slope;
                const float v = GATED ? activate<sizeof(T) == 4, false>(p.activation, g[i], slope) * u[i] : g[i];
                out[(int64_t)(r + i) * p.n] = rows::from_float<T>(v);
            }
        }
    }
}

template <typename T>
void launch_few(const FewParams& p, bool vectors, bool gated, cudaStream_t st) {
    const dim3 grid((p.n + kFewWarps - 1) / kFewWarps, p.rows);
    constexpr int B = (int)sizeof(T);
    if (vectors) {
        if (gated) few_kernel<T, 16, true><<<grid, kFewThreads, 0, st>>>(p);
        else few_kernel<T, 16, false><<<grid, kFewThreads, 0, st>>>(p);
    } else {
        if (gated) few_kernel<T, B, true><<<grid, kFewThreads, 0, st>>>(p);
        else few_kernel<T, B, false><<<grid, kFewThreads, 0, st>>>(p);
    }
}

}  // namespace

cudaError_t product_f32(const Job& job, cudaStream_t st) {
    Params p{};
    p.offsets = job.offsets;
    p.groups = job.groups;
    p.rows = job.rows;
    p.n = job.n;
    p.k = job.k;
    p.segments = job.segments;
    p.splits = job.splits;
    p.activation = job.activation;
    p.dh = job.dh;
    p.out_row = job.out_row;
    p.partial = job.partial;
    for (int i = 0; i < 2; ++i) p.a[i] = job.a[i], p.b[i] = job.b[i], p.out[i] = static_cast<float*>(job.out[i]);
    switch (job.form) {
        case kProduct: return launch_f32<kProduct>(p, st);
        case kGated: return launch_f32<kGated>(p, st);
        case kGatedGrad: return launch_f32<kGatedGrad>(p, st);
        case kBack: return launch_f32<kBack>(p, st);
        default: return launch_f32<kWeights>(p, st);
    }
}

cudaError_t join_parts(const Job& job, cudaStream_t st) {
    const int64_t part = (int64_t)job.groups * job.n * job.k, each = part * job.segments;
    const unsigned blocks = (unsigned)((each + 255) / 256);
    rows::for_type(job.type, 16, [&](auto type, auto) {
        using T = decltype(type);
        join_kernel<T><<<blocks, 256, 0, st>>>(job.partial, job.splits, each, part, static_cast<T*>(job.out[0]), static_cast<T*>(job.out[1]));
    });
    count_launches(1);
    return cudaGetLastError();
}

cudaError_t few_rows(const Job& job, cudaStream_t st) {
    FewParams p{};
    p.offsets = job.offsets;
    p.groups = job.groups;
    p.rows = job.rows;
    p.n = job.n;
    p.k = job.k;
    p.activation = job.activation;
    p.x = job.a[0];
    p.w[0] = job.b[0];
    p.w[1] = job.b[1];
    p.out = job.out[0];
    const bool gated = job.form == kGated;
    uint64_t bits = rows::address_bits(p.x.p) | rows::address_bits(p.w[0].p);
    const uint64_t size = rows::type_bytes(job.type);
    bits |= (uint64_t)(p.x.row | p.w[0].row | p.w[0].group | job.k) * size;
    if (gated) bits |= rows::address_bits(p.w[1].p) | (uint64_t)(p.w[1].row | p.w[1].group) * size;
    const bool vectors = bits % 16 == 0;
    if (job.type == HB_F32) launch_few<float>(p, vectors, gated, st);
    else if (job.type == HB_F16) launch_few<__half>(p, vectors, gated, st);
    else launch_few<__nv_bfloat16>(p, vectors, gated, st);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace experts
}  // namespace hb
