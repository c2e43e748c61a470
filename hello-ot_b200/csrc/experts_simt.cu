// Products of rows sorted by expert on the CUDA cores: fp32 rows, and few rows of any type.
//
// fp32 (product_f32): every form of experts.cu in tiles of 128 x 128 or 64 x 64, 8 of the summed length a step.  Each
// thread copies its elements straight to shared memory (asynchronous copies of 4 bytes, which take any alignment and
// order and write zeros for what is not there), three steps ahead; it holds 8 x 16 or 8 x 4 sums and adds products in
// pairs (fma.rn.f32x2), each rounded like the scalar instruction, so the sums are plain fp32 sums.  Shared memory
// returns 128 bytes a cycle, whatever the lanes share, and 8 x 8 sums want just that for 128 products a cycle: with
// them 32768 x 2048 x 1024 ran at 47 TFLOP/s, now at 53 (2603 us).  The tensor cores
// would need three bf16 parts of each operand and cut off the low bits of their running sums, which fp32 results do
// not allow.  In the gated forms half of a tile's columns are g's and half the same places of u, and one thread
// holds both of a place.
//
// Few rows (few_rows): one token's step of a decode batch reads the named experts' weights once and is bound by that.
// A warp streams the weight rows of one output column and multiplies them with up to 8 rows of x, which
// stay in L1; a block of 8 warps takes 8 columns for the rows of one expert, which the expert's first row finds out for
// itself.
#include <algorithm>
#include <string>

#include "experts.cuh"
#include "internal.h"

namespace hb {
namespace experts {
namespace {

// ---------------------------------------------------------------- fp32 tiles
constexpr int BK = 8, kStages = 4, kThreads = 128;

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
// 4 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy4(uint32_t to, const float* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}

// What a thread copies of an operand's TILE x 8 values each step.  LONG: the operand's rows run along the summed length,
// and 8 threads take 8 neighbours of a row; else across it, and the threads take neighbours of one place of the length.
template <int TILE, bool LONG>
struct Source {
    static constexpr int EACH = TILE * BK / kThreads, APART = kThreads / 8, ACROSS = kThreads / TILE;  // LONG: rows apart; else places of the length
    const float* at[LONG ? EACH : 1];
    int64_t step;  // from one step to the next
    int64_t row;
    uint32_t to;   // the first element's place in a stage, bytes
    uint32_t live; // which of the rows are there
    int k;         // the first element's place in the summed length
    // Place 0 of the tile at `base`, `lim` of them there; HALVES: places from TILE / 2 on at `other`, by its own stride.
    template <bool HALVES>
    __device__ __forceinline__ void start(const float* base, const float* other, int64_t stride, int64_t other_stride, int lim, int pitch) {
        const int t = threadIdx.x;
        row = stride;
        live = 0;
        if (LONG) {
            const int m0 = t >> 3;
            k = t & 7;
            step = BK;
            to = (k * pitch + m0) * 4;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int m = m0 + APART * i, place = HALVES ? m % (TILE / 2) : m;
                const int there = place < lim ? place : 0;
                at[i] = (HALVES && m >= TILE / 2 ? other + there * other_stride : base + there * stride) + k;
                live |= (place < lim ? 1u : 0u) << i;
            }
        } else {
            const int m = t % TILE;
            k = t / TILE;
            step = BK * stride;
            to = (k * pitch + m) * 4;
            at[0] = base + (m < lim ? m : 0) + k * stride;
            live = m < lim ? ~0u : 0u;
        }
    }
    // The next step's elements; `left` of the length are left.
    __device__ __forceinline__ void copy(uint32_t stage, int left, int pitch) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (LONG) {
                const bool there = (live >> i & 1) && k < left;
                copy4(stage + to + APART * i * 4, there ? at[i] : at[0], there);
                if (k + BK < left) at[i] += step;
            } else {
                const bool there = live && k + ACROSS * i < left;
                copy4(stage + to + ACROSS * i * pitch * 4, there ? at[0] + ACROSS * i * row : at[0], there);
            }
        }
        if (!LONG && k + BK < left) at[0] += step;
    }
};

template <int FORM, int TILE>
__global__ void __launch_bounds__(kThreads, TILE == 128 ? 2 : 5) f32_kernel(const __grid_constant__ Params p) {
    constexpr bool HALVES = FORM == kGated || FORM == kGatedGrad;
    constexpr bool A_LONG = FORM != kWeights, B_LONG = FORM != kWeights && FORM != kBack;
    constexpr int COLS = HALVES ? TILE / 2 : TILE, PITCH = TILE + 4;
    constexpr int NR = 8, NQ = TILE / 32, QW = TILE / 32, NP = NQ * QW / 2;  // a thread's rows, its blocks of QW columns, 32 apart, pairs
    constexpr int STAGE = BK * PITCH;           // floats of an operand
    union Memory {
        float stage[kStages][2][STAGE];
        int groups[2][kMostGroups + 2];  // until the block knows its rows
    };
    __shared__ __align__(16) Memory memory;
    const int tid = threadIdx.x, tx = tid % (32 / QW), ty = tid / (32 / QW);
    const int col = blockIdx.y * COLS;
    int row, lim, length, group, part = 0, split = 0, first = 0;  // lim: rows of the tile that are the output's
    {
        int *start = memory.groups[0], *tile = memory.groups[1];
        read_groups(p.offsets, p.groups, p.rows, TILE, start, tile);
        if (FORM == kWeights) {
            part = blockIdx.z % p.segments;
            group = blockIdx.z / p.segments;
            split = group % p.splits;
            group /= p.splits;
            row = blockIdx.x * TILE;
            lim = min(TILE, p.n - row);
            int end;
            split_rows(start[group + 1] - start[group], p.splits, split, first, end);
            length = end - first;
            first += start[group];
        } else {
            if ((int)blockIdx.x >= tile[p.groups + 1]) return;
            group = group_of(tile, p.groups, blockIdx.x);
            row = start[group] + ((int)blockIdx.x - tile[group]) * TILE;
            lim = min(TILE, start[group + 1] - row);
            length = group == p.groups ? 0 : p.k;
        }
        __syncthreads();  // the stages lie over the groups
    }
    const int width = FORM == kWeights ? p.k : p.n;
    uint64_t acc[NR][NP];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < NP; ++j) acc[i][j] = 0;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(&memory.stage[0][0][0]);
    for (int seg = 0; seg < (FORM == kBack ? p.segments : 1) && length > 0; ++seg) {
        Source<TILE, A_LONG> a;
        Source<TILE, B_LONG> b;
        const int blim = min(COLS, width - col);
        if (FORM == kWeights) {
            const Operand &x = p.a[part], &y = p.b[0];
            a.template start<false>(static_cast<const float*>(x.p) + first * x.row + row, nullptr, x.row, 0, lim, PITCH);
            b.template start<false>(static_cast<const float*>(y.p) + first * y.row + col, nullptr, y.row, 0, blim, PITCH);
        } else {
            const Operand &x = p.a[seg], &y = p.b[seg];
            a.template start<false>(static_cast<const float*>(x.p) + row * x.row, nullptr, x.row, 0, lim, PITCH);
            const float* from = static_cast<const float*>(y.p) + group * y.group;
            if (HALVES) {
                const Operand& z = p.b[1];
                b.template start<true>(from + col * y.row, static_cast<const float*>(z.p) + group * z.group + col * z.row, y.row, z.row, blim, PITCH);
            } else {
                b.template start<false>(from + (B_LONG ? col * y.row : col), nullptr, y.row, 0, blim, PITCH);
            }
        }
        const int steps = (length + BK - 1) / BK;
        auto bring = [&](int step) {
            if (step < steps) {
                const uint32_t to = base + step % kStages * 2 * STAGE * 4;
                a.copy(to, length - step * BK, PITCH);
                b.copy(to + STAGE * 4, length - step * BK, PITCH);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int step = 0; step < kStages - 1; ++step) bring(step);
        for (int step = 0; step < steps; ++step) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncthreads();  // this step's elements are there, and the step before is read
            bring(step + kStages - 1);
            const float *as = memory.stage[step % kStages][0], *bs = memory.stage[step % kStages][1];
#pragma unroll
            for (int k = 0; k < BK; ++k) {
                float av[NR];
                uint64_t bv[NP];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 f = *reinterpret_cast<const float4*>(as + k * PITCH + h * (TILE / 2) + ty * 4);
                    av[h * 4] = f.x, av[h * 4 + 1] = f.y, av[h * 4 + 2] = f.z, av[h * 4 + 3] = f.w;
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    const float* from = bs + k * PITCH + q * 32 + tx * QW;
                    if constexpr (QW == 4) {
                        const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(from);
                        bv[2 * q] = u.x, bv[2 * q + 1] = u.y;
                    } else {
                        bv[q] = *reinterpret_cast<const uint64_t*>(from);
                    }
                }
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const uint64_t aa = pack(av[i], av[i]);
#pragma unroll
                    for (int j = 0; j < NP; ++j) fma2(acc[i][j], aa, bv[j]);
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the next segment writes the stages
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
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int m = i / 4 * (TILE / 2) + ty * 4 + i % 4;
        if (m >= lim) continue;
        const int64_t r = (int64_t)(row + m) * out_row;
#pragma unroll
        for (int j = 0; j < (HALVES ? NP : 2 * NP); ++j) {  // HALVES: the second half of the blocks is u's
            const int c = col + j / QW * 32 + tx * QW + j % QW;
            if (c >= width) continue;
            const float v = half_of(acc[i][j / 2], j & 1);
            if (HALVES) {
                const float u = half_of(acc[i][NP / 2 + j / 2], j & 1);
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

template <int FORM, int TILE>
cudaError_t launch_f32(const Params& p, cudaStream_t st) {
    const int width = FORM == kWeights ? p.k : p.n, cols = FORM == kGated || FORM == kGatedGrad ? TILE / 2 : TILE;
    const dim3 grid(FORM == kWeights ? (p.n + TILE - 1) / TILE : p.rows / TILE + p.groups + 1, (width + cols - 1) / cols,
                    FORM == kWeights ? p.splits * p.segments * p.groups : 1);
    f32_kernel<FORM, TILE><<<grid, kThreads, 0, st>>>(p);
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

// The expert of row r (the first whose rows end behind it, with offsets read as their running maximum; groups: none), or
// -1 where the row before has the same: the expert's first row does the work.
__device__ __forceinline__ int expert_of(const int32_t* offsets, int groups, int r, int (&found)[2]) {
    if (threadIdx.x < 2) found[threadIdx.x] = groups;
    __syncthreads();
    int here = groups, before = groups;
    for (int e = threadIdx.x; e < groups && here == groups; e += kFewThreads) {
        const int end = offsets[e + 1];
        if (end > r) here = e;
        if (end >= r && before == groups) before = e;
    }
    if (here < groups) atomicMin(&found[0], here);
    if (before < groups) atomicMin(&found[1], before);
    __syncthreads();
    return r > 0 && found[0] == found[1] ? -1 : found[0];
}

// 16 bytes of a row from element k on, zeros behind its end; VECTORS: rows lie on 16 bytes and end there.  Either way a
// lane has the same elements, so the sums do not depend on where the rows lie.
template <bool VECTORS, typename T>
__device__ __forceinline__ void load_piece(rows::Vec<T, 16>& v, const T* row, int k, int end, bool once) {
    if (VECTORS) {
        if (k >= end) v.zero();
        else if (once) v.load_once(row + k);
        else v.load(row + k);
    } else {
#pragma unroll
        for (int j = 0; j < rows::Vec<T, 16>::N; ++j) v.v[j] = k + j < end ? row[k + j] : rows::from_float<T>(0.0f);
    }
}

// Four blocks an SM and two pieces of a row in flight; two blocks with four pieces took 33 us where this takes 25, and 51 where
// it takes 37 (16 rows of 16 experts, 2048 x 1024 bf16, on two machines).
template <typename T, bool VECTORS, bool GATED>
__global__ void __launch_bounds__(kFewThreads, 4) few_kernel(const __grid_constant__ FewParams p) {
    using V = rows::Vec<T, 16>;
    __shared__ int found[2];
    const int r0 = blockIdx.y, lane = threadIdx.x & 31;
    const int col = blockIdx.x * kFewWarps + (threadIdx.x >> 5);
    int e = 0, count = p.rows - r0;
    if (p.offsets) {
        e = expert_of(p.offsets, p.groups, r0, found);
        if (e < 0) return;
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
        constexpr int U = 2;  // pieces of each weight row in flight
        for (int k = lane * V::N; k < p.k; k += 32 * V::N * U) {
            V a[U], b[U];
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int at = k + q * 32 * V::N;
                load_piece<VECTORS>(a[q], w0, at, p.k, true);
                if (GATED) load_piece<VECTORS>(b[q], w1, at, p.k, true);
            }
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int at = k + q * 32 * V::N;
                if (at >= p.k) break;
#pragma unroll
                for (int i = 0; i < kPass; ++i) {
                    if (i >= here) break;
                    V xv;
                    load_piece<VECTORS>(xv, x + i * p.x.row, at, p.k, false);
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
    const dim3 grid((p.n + kFewWarps - 1) / kFewWarps, p.rows);  // rows: at most 4 an expert, 8192
    if (vectors) {
        if (gated) few_kernel<T, true, true><<<grid, kFewThreads, 0, st>>>(p);
        else few_kernel<T, true, false><<<grid, kFewThreads, 0, st>>>(p);
    } else {
        if (gated) few_kernel<T, false, true><<<grid, kFewThreads, 0, st>>>(p);
        else few_kernel<T, false, false><<<grid, kFewThreads, 0, st>>>(p);
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
    const bool wide = f32_tile(job) == 128;
    switch (job.form) {
        case kProduct: return wide ? launch_f32<kProduct, 128>(p, st) : launch_f32<kProduct, 64>(p, st);
        case kGated: return wide ? launch_f32<kGated, 128>(p, st) : launch_f32<kGated, 64>(p, st);
        case kGatedGrad: return wide ? launch_f32<kGatedGrad, 128>(p, st) : launch_f32<kGatedGrad, 64>(p, st);
        case kBack: return wide ? launch_f32<kBack, 128>(p, st) : launch_f32<kBack, 64>(p, st);
        default: return wide ? launch_f32<kWeights, 128>(p, st) : launch_f32<kWeights, 64>(p, st);
    }
}

int f32_tile(const Job& job) {
    const int64_t cols = job.form == kGated || job.form == kGatedGrad ? 64 : 128, width = job.form == kWeights ? job.k : job.n;
    const int64_t tiles = (width + cols - 1) / cols *
                          (job.form == kWeights ? job.segments * (int64_t)job.groups * ((job.n + 127) / 128) : job.rows / 128 + job.groups / 2);
    return tiles * (job.form == kWeights ? std::max<int64_t>(1, job.rows / job.groups / 1024) : 1) < 222 ? 64 : 128;
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
