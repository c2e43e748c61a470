// Root-mean-square norm of rows with the residual's addition, its 8-bit output, and its gradients.
//
//   t = x + residual,  r = 1 / sqrt(mean(t^2) + eps),  y = t r w
//   dx = r w dy - x r^3 mean(w dy x) + dtotal,  dw = sum over rows of dy x r
//
// Bound by HBM: each array passes once.  A row is held in the registers of 8 to 512 threads, 8 to 32 columns each, so
// its sum and its scaling need one read, and the next row comes meanwhile; rows of more than 16384 columns are read
// a second time, from L2.  The gradient of w is summed over a block's rows in registers, every block leaves one row of
// fp32 partial sums, and a second launch adds those in order: no atomics, the result does not depend on the launch.
// On a B200 65536 x 2048 bf16 with residual takes 164 us (6.5 TB/s), in 8 bits 167 (5.7 TB/s), rows in 8 bits read
// back 69 (5.9 TB/s), the gradients 187 (5.7 TB/s): calls one after the other; one that is waited for takes 5 us more.
//
// Sums are fp32; t is rounded for the output alone.  In 8 bits 32 columns share a power of two: the exponent is that
// of the group's largest magnitude by 448, rounded up, so nothing saturates and the group's largest value keeps
// 4 significant bits.
#include <algorithm>
#include <cmath>
#include <string>

#include <cuda_fp8.h>

#include "internal.h"
#include "rows.cuh"

namespace hb {
namespace norm8 {

constexpr int kGroup = 32;  // columns that share a scale

// ---------------------------------------------------------------- 8 bits
// Exponent byte of the smallest power of two by which a magnitude (its bits) fits 448 = 0.875 * 2^9.
__device__ __forceinline__ int scale_byte(uint32_t bits) {
    if (bits >= 0x7f800000u) return 255;
    if (bits == 0) return 0;
    const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);  // 1.75 * 2^8 fits 2^0
    return max(e, 1);  // 2^-126: no subnormal scale
}
__device__ __forceinline__ float scale_value(int byte) {
    return byte == 255 ? __int_as_float(0x7fc00000) : byte == 0 ? 0x1p-127f : __uint_as_float((uint32_t)byte << 23);
}
__device__ __forceinline__ uint8_t to_code(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float of_code(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// ---------------------------------------------------------------- forward
struct Forward {
    const void *x, *residual, *weight;
    int64_t x_row, residual_row, rows;
    int width, weight_type, weight_whole;
    float eps;
    void *y, *total;
    int turns;
    uint8_t *codes, *scales;
};

// Sum over the THREADS threads of a row: a part of a warp, a warp, or a whole block.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* shared) {
#pragma unroll
    for (int d = (THREADS < 32 ? THREADS : 32) / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (THREADS <= 32) return v;
    __syncthreads();  // the last row's sums have been read
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) s += shared[i];
    return s;
}

// N values of the weight from column c, a multiple of N; whole: the weight begins on 16 bytes.
template <int N, typename T>
__device__ __forceinline__ void load_values(float (&w)[N], const T* p, bool whole) {
    constexpr int BYTES = N * (int)sizeof(T) < 16 ? N * (int)sizeof(T) : 16, M = BYTES / (int)sizeof(T);
    if (whole) {
#pragma unroll
        for (int q = 0; q < N / M; ++q) {
            rows::Vec<T, BYTES> v;
            v.load(p + q * M);
#pragma unroll
            for (int j = 0; j < M; ++j) w[q * M + j] = rows::to_float(v.v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = rows::to_float(p[j]);
    }
}
template <int N, typename P>
__device__ __forceinline__ void load_weights(float (&w)[N], const P& p, int c) {
    if (p.weight_type == HB_F32) load_values<N>(w, static_cast<const float*>(p.weight) + c, p.weight_whole);
    else if (p.weight_type == HB_F16) load_values<N>(w, static_cast<const __half*>(p.weight) + c, p.weight_whole);
    else load_values<N>(w, static_cast<const __nv_bfloat16*>(p.weight) + c, p.weight_whole);
}

// N values of row r from column c in 8 bits; the lanes of a group hold neighbouring vectors.  Called by whole warps;
// `there` false: columns behind the row.
template <int N>
__device__ __forceinline__ void write_8bit(const Forward& p, int64_t r, int c, const float (&y)[N], bool there) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) most = max(most, there ? __float_as_uint(fabsf(y[j])) : 0u);
    if (N == 1) {
        most = __reduce_max_sync(0xffffffffu, most);
    } else {
#pragma unroll
        for (int d = 1; d < kGroup / N; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
    }
    if (!there) return;
    const int byte = scale_byte(most);
    // 2^(127 - byte); the largest byte of finite magnitudes is 247
    const float inverse = byte == 0 ? 0.0f : byte == 255 ? __int_as_float(0x7fc00000) : __uint_as_float((uint32_t)(254 - byte) << 23);
    rows::Vec<uint8_t, N> code;
#pragma unroll
    for (int j = 0; j < N; ++j) code.v[j] = to_code(y[j] * inverse);
    code.store(p.codes + r * p.width + c);
    if (c % kGroup == 0) p.scales[r * ((p.width + kGroup - 1) / kGroup) + c / kGroup] = (uint8_t)byte;
}

// A row's raw values, COLUMNS of each thread; the next row's come while this one is summed.
template <typename T, int VB, int THREADS, int COLUMNS>
struct Raw {
    using V = rows::Vec<T, VB>;
    static constexpr int HELD = COLUMNS / V::N;
    V v[HELD];
    __device__ __forceinline__ void load(const T* row, int width, bool there) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int c = (i * THREADS + (int)threadIdx.x % THREADS) * V::N;
            if (there && c < width) v[i].load_once(row + c);
            else v[i].zero();
        }
    }
};

constexpr int block_of(int threads) { return threads < 128 ? 128 : threads; }

// THREADS threads hold a row, COLUMNS each; a block takes some rows in order (`turns`).
template <typename T, int VB, int THREADS, int COLUMNS, bool ADD, bool BITS8>
__global__ void __launch_bounds__(block_of(THREADS)) forward_kernel(const __grid_constant__ Forward p) {
    using R = Raw<T, VB, THREADS, COLUMNS>;
    using V = typename R::V;
    constexpr int ROWS = block_of(THREADS) / THREADS;
    __shared__ float shared[THREADS < 32 ? 1 : THREADS / 32];
    const int t = threadIdx.x % THREADS;
    const int64_t step = ROWS;
    const int64_t base = (int64_t)blockIdx.x * ROWS * p.turns;
    const int64_t end = min(p.rows, base + ROWS * p.turns);
    const T *x = static_cast<const T*>(p.x), *residual = static_cast<const T*>(p.residual);
    R a, b;
    int64_t r = base + threadIdx.x / THREADS;
    a.load(x + r * p.x_row, p.width, r < end);
    if (ADD) b.load(residual + r * p.residual_row, p.width, r < end);
    // every thread of a block makes the same turns: the rows of a warp or block are summed together
    for (int64_t first = base; first < end; first += step, r += step) {
        const bool there = r < end;
        float f[R::HELD][V::N], squares = 0.0f;
#pragma unroll
        for (int i = 0; i < R::HELD; ++i)
#pragma unroll
            for (int j = 0; j < V::N; ++j) {
                f[i][j] = rows::to_float(a.v[i].v[j]);
                if (ADD) f[i][j] += rows::to_float(b.v[i].v[j]);
                squares = fmaf(f[i][j], f[i][j], squares);
            }
        const int64_t next = r + step;
        a.load(x + next * p.x_row, p.width, next < end);
        if (ADD) b.load(residual + next * p.residual_row, p.width, next < end);
        if (p.total && there) {
#pragma unroll
            for (int i = 0; i < R::HELD; ++i) {
                const int c = (i * THREADS + t) * V::N;
                V o;
#pragma unroll
                for (int j = 0; j < V::N; ++j) o.v[j] = rows::from_float<T>(f[i][j]);
                if (c < p.width) o.store_once(static_cast<T*>(p.total) + r * p.width + c);
            }
        }
        const float scale = 1.0f / sqrtf(row_sum<THREADS>(squares, shared) / (float)p.width + p.eps);
#pragma unroll
        for (int i = 0; i < R::HELD; ++i) {
            const int c = (i * THREADS + t) * V::N;
            if (i * THREADS * V::N >= p.width) break;  // the same for all
            const bool inside = there && c < p.width;
            float w[V::N];
            if (inside) load_weights(w, p, c);
#pragma unroll
            for (int j = 0; j < V::N; ++j) f[i][j] = inside ? f[i][j] * scale * w[j] : 0.0f;
            if constexpr (BITS8) {
                write_8bit<V::N>(p, r, c, f[i], inside);
            } else if (inside) {
                V o;
#pragma unroll
                for (int j = 0; j < V::N; ++j) o.v[j] = rows::from_float<T>(f[i][j]);
                o.store_once(static_cast<T*>(p.y) + r * p.width + c);
            }
        }
    }
}

// Rows wider than 512 threads hold: a block a row, read twice.
template <typename T, int VB, bool BITS8>
__global__ void __launch_bounds__(512) wide_forward_kernel(const __grid_constant__ Forward p) {
    using V = rows::Vec<T, VB>;
    __shared__ float shared[16];
    const int64_t r = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + r * p.x_row;
    const T* residual = p.residual ? static_cast<const T*>(p.residual) + r * p.residual_row : nullptr;
    auto load = [&](float (&f)[V::N], int c) {
        V a, b;
        a.load(x + c);
        if (residual) b.load(residual + c);
#pragma unroll
        for (int j = 0; j < V::N; ++j) f[j] = residual ? rows::to_float(a.v[j]) + rows::to_float(b.v[j]) : rows::to_float(a.v[j]);
    };
    float squares = 0.0f, f[V::N];
    for (int c = threadIdx.x * V::N; c < p.width; c += 512 * V::N) {
        load(f, c);
#pragma unroll
        for (int j = 0; j < V::N; ++j) squares = fmaf(f[j], f[j], squares);
    }
    const float scale = 1.0f / sqrtf(row_sum<512>(squares, shared) / (float)p.width + p.eps);
    for (int from = 0; from < p.width; from += 512 * V::N) {
        const int c = from + threadIdx.x * V::N;
        const bool inside = c < p.width;
        V o;
        float w[V::N];
        if (inside) {
            load(f, c);
            load_weights(w, p, c);
#pragma unroll
            for (int j = 0; j < V::N; ++j) o.v[j] = rows::from_float<T>(f[j]);
            if (p.total) o.store_once(static_cast<T*>(p.total) + r * p.width + c);
        }
#pragma unroll
        for (int j = 0; j < V::N; ++j) f[j] = inside ? f[j] * scale * w[j] : 0.0f;
        if constexpr (BITS8) {
            write_8bit<V::N>(p, r, c, f, inside);
        } else if (inside) {
#pragma unroll
            for (int j = 0; j < V::N; ++j) o.v[j] = rows::from_float<T>(f[j]);
            o.store_once(static_cast<T*>(p.y) + r * p.width + c);
        }
    }
}

template <typename T, int VB, int THREADS, int COLUMNS, bool BITS8>
void launch_forward(const Forward& p, cudaStream_t st) {
    constexpr int BLOCK = block_of(THREADS), ROWS = BLOCK / THREADS;
    if constexpr (COLUMNS == 0) {
        wide_forward_kernel<T, VB, BITS8><<<(unsigned)p.rows, 512, 0, st>>>(p);
    } else {
        // A block's rows come one after the other in memory: enough to hide its start, few enough that blocks which start
        // in order keep HBM's pages open (65536 x 2048 bf16 with residual 172 us at 1, 160 at 2, 164 at 4, 183 where
        // resident blocks stride; without residual 103, 95, 92 and 93; 32768 x 2048 fp32 157, 161, 162 and 171).
        Forward q = p;
        q.turns = sizeof(T) == 4 ? 1 : p.residual ? 2 : 4;
        while (q.turns > 1 && p.rows < (int64_t)ROWS * q.turns * 148 * 8) q.turns /= 2;  // few rows: all SMs first
        const unsigned blocks = (unsigned)((p.rows + ROWS * q.turns - 1) / (ROWS * q.turns));
        if (p.residual) forward_kernel<T, VB, THREADS, COLUMNS, true, BITS8><<<blocks, BLOCK, 0, st>>>(q);
        else forward_kernel<T, VB, THREADS, COLUMNS, false, BITS8><<<blocks, BLOCK, 0, st>>>(q);
    }
}

// ---------------------------------------------------------------- reading 8 bits back
// A warp a row: 16 columns a lane where rows lie on 16 bytes, else one.
template <typename TO, bool VECTORS>
__global__ void __launch_bounds__(256) read_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                   int64_t rows, int width, TO* __restrict__ out) {
    const int groups = (width + kGroup - 1) / kGroup, lane = threadIdx.x & 31;
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= rows) return;
    codes += r * width;
    scales += r * groups;
    out += r * width;
    if (VECTORS) {
        constexpr int V = 16 / (int)sizeof(TO);
#pragma unroll 2
        for (int c = lane * 16; c < width; c += 512) {
            rows::Vec<uint8_t, 16> in;
            in.load_once(codes + c);
            const float s = scale_value(scales[c / kGroup]);
#pragma unroll
            for (int q = 0; q < 16 / V; ++q) {
                rows::Vec<TO, 16> o;
#pragma unroll
                for (int j = 0; j < V; ++j) o.v[j] = rows::from_float<TO>(of_code(in.v[q * V + j]) * s);
                o.store(out + c + q * V);
            }
        }
    } else {
#pragma unroll 4
        for (int c = lane; c < width; c += 32) out[c] = rows::from_float<TO>(of_code(codes[c]) * scale_value(scales[c / kGroup]));
    }
}

// ---------------------------------------------------------------- gradients
struct Backward {
    const void *dy, *x, *dtotal, *weight;
    int64_t dy_row, x_row, dtotal_row, rows;
    int width, weight_type, weight_whole;
    float eps;
    void* dx;
    float *partial, *stats;  // partial: [blocks][width]; stats: [rows][2] of wide rows
};

// Sums of w dy x and x^2 at once.
template <int THREADS>
__device__ __forceinline__ float2 row_sums(float a, float b, float2* shared) {
#pragma unroll
    for (int d = (THREADS < 32 ? THREADS : 32) / 2; d > 0; d >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, d);
        b += __shfl_xor_sync(0xffffffffu, b, d);
    }
    if (THREADS <= 32) return make_float2(a, b);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) s.x += shared[i].x, s.y += shared[i].y;
    return s;
}

// r^3 mean(w dy x), one factor at a time: the mean grows as the row does, while r^3 alone leaves fp32's normal numbers from
// rows of some 10^13 and 10^-13 on, whose squares it still sums.
__device__ __forceinline__ float row_pull(float inverse, float mean) { return inverse * (inverse * (inverse * mean)); }

// Resident blocks an SM: what the registers of a thread's columns leave (128 a thread, 80 with 8 columns).
constexpr int resident(int threads, int columns) {
    return (columns <= 8 ? 768 : 512) / block_of(threads) > 1 ? (columns <= 8 ? 768 : 512) / block_of(threads) : 1;
}

// Rows held in registers; a block strides over the rows and keeps its sums for dw.  Up to 16 columns a thread the
// weight's values are held too, and rows of 16-byte vectors of 16-bit values, which take half the registers, come while
// the row before is summed (65536 x 2048 bf16 219 -> 186 us; in fp32 it spills, 208 -> 225).
template <typename T, int VB, int THREADS, int COLUMNS>
__global__ void __launch_bounds__(block_of(THREADS), resident(THREADS, COLUMNS)) backward_kernel(const __grid_constant__ Backward p) {
    using R = Raw<T, VB, THREADS, COLUMNS>;
    using V = typename R::V;
    constexpr int ROWS = block_of(THREADS) / THREADS, HELD = R::HELD;
    constexpr bool KEEP = COLUMNS <= 16, AHEAD = KEEP && VB == 16 && sizeof(T) == 2;
    __shared__ float2 shared[THREADS < 32 ? 1 : THREADS / 32];
    __shared__ float joined[ROWS > 1 ? THREADS * COLUMNS : 1];
    const int t = threadIdx.x % THREADS, mine = threadIdx.x / THREADS;
    float dw[HELD][V::N], kept[KEEP ? HELD : 1][V::N];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int c = (i * THREADS + t) * V::N;
#pragma unroll
        for (int j = 0; j < V::N; ++j) {
            dw[i][j] = 0.0f;
            if (KEEP) kept[i][j] = 0.0f;
        }
        if (KEEP && c < p.width) load_weights(kept[i], p, c);
    }
    const T *x = static_cast<const T*>(p.x), *dy = static_cast<const T*>(p.dy);
    const T* dtotal = p.dx ? static_cast<const T*>(p.dtotal) : nullptr;
    R a, g, d;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t r = (int64_t)blockIdx.x * ROWS + mine;
    auto fetch = [&](R& ra, R& rg, R& rd, int64_t at) {
        const bool there = at < p.rows;
        ra.load(x + at * p.x_row, p.width, there);
        rg.load(dy + at * p.dy_row, p.width, there);
        if (dtotal) rd.load(dtotal + at * p.dtotal_row, p.width, there);
    };
    if (AHEAD) fetch(a, g, d, r);
    for (int64_t first = (int64_t)blockIdx.x * ROWS; first < p.rows; first += step, r += step) {
        R a_next, g_next, d_next;
        if (AHEAD) fetch(a_next, g_next, d_next, r + step);
        else fetch(a, g, d, r);
        float squares = 0.0f, along = 0.0f;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int c = (i * THREADS + t) * V::N;
            float w[V::N];
            if (!KEEP && c < p.width) load_weights(w, p, c);
#pragma unroll
            for (int j = 0; j < V::N; ++j) {
                const float xf = rows::to_float(a.v[i].v[j]), wj = KEEP ? kept[i][j] : c < p.width ? w[j] : 0.0f;
                squares = fmaf(xf, xf, squares);
                along = fmaf(wj * rows::to_float(g.v[i].v[j]), xf, along);
            }
        }
        const float2 sums = row_sums<THREADS>(along, squares, shared);
        const float inverse = 1.0f / sqrtf(sums.y / (float)p.width + p.eps);
        const float back = row_pull(inverse, sums.x / (float)p.width);
        if (r < p.rows) {
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                const int c = (i * THREADS + t) * V::N;
                if (c >= p.width) continue;
                float w[V::N];
                if (!KEEP) load_weights(w, p, c);
                V o;
#pragma unroll
                for (int j = 0; j < V::N; ++j) {
                    const float xf = rows::to_float(a.v[i].v[j]), gf = rows::to_float(g.v[i].v[j]);
                    dw[i][j] = fmaf(gf * xf, inverse, dw[i][j]);
                    float v = fmaf(inverse, (KEEP ? kept[i][j] : w[j]) * gf, -xf * back);
                    if (dtotal) v += rows::to_float(d.v[i].v[j]);
                    o.v[j] = rows::from_float<T>(v);
                }
                if (p.dx) o.store_once(static_cast<T*>(p.dx) + r * p.width + c);
            }
        }
        if (AHEAD) a = a_next, g = g_next, d = d_next;
    }
    if (!p.partial) return;
    float* to = p.partial + (int64_t)blockIdx.x * p.width;
    if constexpr (ROWS > 1) {  // the block's rows side by side, added in order
        for (int turn = 0; turn < ROWS; ++turn) {
            __syncthreads();
            if (mine != turn) continue;
#pragma unroll
            for (int i = 0; i < HELD; ++i)
#pragma unroll
                for (int j = 0; j < V::N; ++j) {
                    float& s = joined[(i * THREADS + t) * V::N + j];
                    s = turn == 0 ? dw[i][j] : s + dw[i][j];
                }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < p.width; c += block_of(THREADS)) to[c] = joined[c];
    } else {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int c = (i * THREADS + t) * V::N;
#pragma unroll
            for (int j = 0; j < V::N; ++j)
                if (c + j < p.width) to[c + j] = dw[i][j];
        }
    }
}

// Wide rows: the two sums of each row first, then columns by blocks of 256 vectors over slabs of rows.
template <typename T, int VB>
__global__ void __launch_bounds__(512) wide_sums_kernel(const __grid_constant__ Backward p) {
    using V = rows::Vec<T, VB>;
    __shared__ float2 shared[16];
    const int64_t r = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + r * p.x_row;
    const T* dy = static_cast<const T*>(p.dy) + r * p.dy_row;
    float squares = 0.0f, along = 0.0f;
    for (int c = threadIdx.x * V::N; c < p.width; c += 512 * V::N) {
        V a, g;
        float w[V::N];
        a.load(x + c);
        g.load(dy + c);
        load_weights(w, p, c);
#pragma unroll
        for (int j = 0; j < V::N; ++j) {
            const float xf = rows::to_float(a.v[j]);
            squares = fmaf(xf, xf, squares);
            along = fmaf(w[j] * rows::to_float(g.v[j]), xf, along);
        }
    }
    const float2 sums = row_sums<512>(squares, along, shared);
    if (threadIdx.x == 0) {
        const float inverse = 1.0f / sqrtf(sums.x / (float)p.width + p.eps);
        p.stats[2 * r] = inverse;
        p.stats[2 * r + 1] = row_pull(inverse, sums.y / (float)p.width);
    }
}
template <typename T, int VB>
__global__ void __launch_bounds__(256) wide_kernel(const __grid_constant__ Backward p) {
    using V = rows::Vec<T, VB>;
    const int c = (blockIdx.x * 256 + threadIdx.x) * V::N;
    if (c >= p.width) return;
    float w[V::N], dw[V::N];
    load_weights(w, p, c);
#pragma unroll
    for (int j = 0; j < V::N; ++j) dw[j] = 0.0f;
    for (int64_t r = blockIdx.y; r < p.rows; r += gridDim.y) {
        const float inverse = p.stats[2 * r], back = p.stats[2 * r + 1];
        V a, g, d, o;
        a.load(static_cast<const T*>(p.x) + r * p.x_row + c);
        g.load(static_cast<const T*>(p.dy) + r * p.dy_row + c);
        if (p.dtotal) d.load(static_cast<const T*>(p.dtotal) + r * p.dtotal_row + c);
#pragma unroll
        for (int j = 0; j < V::N; ++j) {
            const float xf = rows::to_float(a.v[j]), gf = rows::to_float(g.v[j]);
            dw[j] = fmaf(gf * xf, inverse, dw[j]);
            float v = fmaf(inverse, w[j] * gf, -xf * back);
            if (p.dtotal) v += rows::to_float(d.v[j]);
            o.v[j] = rows::from_float<T>(v);
        }
        if (p.dx) o.store(static_cast<T*>(p.dx) + r * p.width + c);
    }
    if (p.partial)
#pragma unroll
        for (int j = 0; j < V::N; ++j) p.partial[(int64_t)blockIdx.y * p.width + c + j] = dw[j];
}

// dw: the blocks' sums added, 8 chains a column in a fixed order.
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ partial, int parts, int width, void* dw, int type) {
    __shared__ float shared[8][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), chain = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < width)
#pragma unroll 4
        for (int i = chain; i < parts; i += 8) s += partial[(int64_t)i * width + c];
    shared[chain][threadIdx.x & 31] = s;
    __syncthreads();
    if (chain == 0 && c < width) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += shared[i][threadIdx.x];
        rows::store_weight(dw, type, c, s);
    }
}

// Threads a row and columns a thread: the smallest form that holds the row.  Rows of up to 128 columns lie 16 to a
// block, where a vector is a quarter of a scale's group at least.  Off the 16-byte grid a thread's loads are short, and up to
// 1024 columns it holds 8, so that more threads are resident (bf16, 16 and 8 columns a thread: norm of 40000 x 1002 with
// residual 87 and 72 us, in 8 bits 158 and 91, gradients 158 and 99; 200000 x 131 125 and 82; but 65536 x 1091 226
// and 238, gradients of 20000 x 3333 172 and 323).
template <int N, typename F>
void for_width(int64_t width, F&& f) {
    if (N < 4 && width <= 256) f(rows::Bytes<32>{}, rows::Bytes<N < 4 ? 8 : 16>{});
    else if (N < 4 && width <= 1024) f(rows::Bytes<128>{}, rows::Bytes<N < 4 ? 8 : 16>{});
    else if (N >= 4 && width <= 128) f(rows::Bytes<N >= 4 ? 8 : 32>{}, rows::Bytes<16>{});
    else if (width <= 512) f(rows::Bytes<32>{}, rows::Bytes<16>{});
    else if (width <= 2048) f(rows::Bytes<128>{}, rows::Bytes<16>{});
    else if (width <= 4096) f(rows::Bytes<256>{}, rows::Bytes<16>{});
    else if (width <= 8192) f(rows::Bytes<512>{}, rows::Bytes<16>{});
    else if (width <= 16384) f(rows::Bytes<512>{}, rows::Bytes<32>{});
    else f(rows::Bytes<512>{}, rows::Bytes<0>{});
}
constexpr int64_t kMostHeld = 16384;  // columns of a row that for_width holds
constexpr int kParts = 148 * 8;       // most blocks that sum dw

// Blocks that sum dw: as many as are resident, or a row each.
inline int parts_of(int64_t rows, int threads, int columns) {
    const int64_t side = block_of(threads) / threads, blocks = 148 * resident(threads, columns);
    return (int)std::max<int64_t>(1, std::min(blocks, (rows + side - 1) / side));
}

inline bool bad_rows(const void* p, int64_t stride, int type) {
    return !p || rows::address_bits(p) % rows::type_bytes(type) || stride < 0;
}
// Vector bytes of all rows together: 16, 4 or an element.
inline int vector_of(uint64_t bits, int type) {
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : rows::type_bytes(type);
}
template <typename F>
void for_vectors(int type, int vb, F&& f) {
    if (type == HB_F32) {
        if (vb == 16) f(float{}, rows::Bytes<16>{});
        else f(float{}, rows::Bytes<4>{});
    } else if (type == HB_F16) {
        if (vb == 16) f(__half{}, rows::Bytes<16>{});
        else if (vb == 4) f(__half{}, rows::Bytes<4>{});
        else f(__half{}, rows::Bytes<2>{});
    } else {
        if (vb == 16) f(__nv_bfloat16{}, rows::Bytes<16>{});
        else if (vb == 4) f(__nv_bfloat16{}, rows::Bytes<4>{});
        else f(__nv_bfloat16{}, rows::Bytes<2>{});
    }
}
int finish(cudaError_t e, const char* what) {
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace norm8
}  // namespace hb

using namespace hb;
using namespace hb::norm8;

extern "C" int hb_rms_norm(int type, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, int64_t rows,
                           int64_t width, const void* weight, int weight_type, double eps, void* y, void* codes, void* scales,
                           void* total, void* stream) {
    if (!rows::valid_type(type) || !rows::valid_type(weight_type)) return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm: element type");
    if (rows < 0 || rows > INT32_MAX || width < 1 || width > (1 << 30)) return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm: rows or width out of range");
    if (!(eps >= 0.0)) return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm: eps must be a number >= 0");
    if (rows == 0) return HB_OK;
    const int size = rows::type_bytes(type);
    if (bad_rows(x, x_stride, type) || (residual && bad_rows(residual, residual_stride, type)) || !weight ||
        rows::address_bits(weight) % rows::type_bytes(weight_type) || (codes ? !scales || y : !y) || rows::address_bits(y) % size ||
        rows::address_bits(total) % size)
        return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm: null or misaligned pointer, or bad stride");
    Forward p{x, residual, weight, x_stride, residual_stride, rows, (int)width, weight_type, rows::address_bits(weight) % 16 == 0, (float)eps, y, total, 1,
              static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales)};
    uint64_t bits = rows::address_bits(x) | rows::address_bits(residual) | rows::address_bits(y) | rows::address_bits(total) |
                    (uint64_t)(width | (rows > 1 ? x_stride : 0) | (rows > 1 && residual ? residual_stride : 0)) * size;
    if (codes) bits |= rows::address_bits(codes) % (16 / size) ? 1 : 0;  // a vector's codes lie on their own size
    const auto st = static_cast<cudaStream_t>(stream);
    for_vectors(type, vector_of(bits, type), [&](auto t, auto vb) {
        using T = decltype(t);
        constexpr int VB = decltype(vb)::value, N = VB / (int)sizeof(T);
        for_width<N>(width, [&](auto threads, auto columns) {
            constexpr int THREADS = decltype(threads)::value, COLUMNS = decltype(columns)::value;
            if (p.codes) launch_forward<T, VB, THREADS, COLUMNS, true>(p, st);
            else launch_forward<T, VB, THREADS, COLUMNS, false>(p, st);
        });
    });
    count_launches(1);
    return finish(cudaGetLastError(), "hb_rms_norm");
}

extern "C" int hb_rows_of_8bit(const void* codes, const void* scales, int64_t rows, int64_t width, int out_type, void* out, void* stream) {
    if (!rows::valid_type(out_type)) return abi_fail(HB_BAD_ARGUMENT, "hb_rows_of_8bit: element type");
    if (rows < 0 || rows > INT32_MAX || width < 1 || width > (1 << 30))
        return abi_fail(HB_BAD_ARGUMENT, "hb_rows_of_8bit: rows or width out of range");
    if (rows == 0) return HB_OK;
    if (!codes || !scales || !out || rows::address_bits(out) % rows::type_bytes(out_type))
        return abi_fail(HB_BAD_ARGUMENT, "hb_rows_of_8bit: null or misaligned pointer");
    const bool vector = width % 16 == 0 && ((rows::address_bits(codes) | rows::address_bits(out)) & 15) == 0;
    const unsigned blocks = (unsigned)((rows + 7) / 8);
    const auto st = static_cast<cudaStream_t>(stream);
    const auto *c = static_cast<const uint8_t*>(codes), *s = static_cast<const uint8_t*>(scales);
    rows::for_type(out_type, 16, [&](auto t, auto) {
        using T = decltype(t);
        if (vector) read_kernel<T, true><<<blocks, 256, 0, st>>>(c, s, rows, (int)width, static_cast<T*>(out));
        else read_kernel<T, false><<<blocks, 256, 0, st>>>(c, s, rows, (int)width, static_cast<T*>(out));
    });
    count_launches(1);
    return finish(cudaGetLastError(), "hb_rows_of_8bit");
}

extern "C" size_t hb_rms_norm_grad_workspace(int64_t rows, int64_t width) {
    if (rows < 0 || rows > INT32_MAX || width < 1 || width > (1 << 30)) return 0;
    // the blocks' sums, and two sums a row of those that no block holds
    const size_t sums = width > kMostHeld ? (size_t)rows * 2 * sizeof(float) : 0;
    return (sums + 255) / 256 * 256 + (size_t)std::min<int64_t>(kParts, std::max<int64_t>(rows, 1)) * width * sizeof(float);
}

extern "C" int hb_rms_norm_grad(int type, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* dtotal,
                                int64_t dtotal_stride, int64_t rows, int64_t width, const void* weight, int weight_type, double eps,
                                void* dx, void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "hb_rms_norm_grad";
    if (!rows::valid_type(type) || !rows::valid_type(weight_type)) return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm_grad: element type");
    if (rows < 0 || rows > INT32_MAX || width < 1 || width > (1 << 30))
        return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm_grad: rows or width out of range");
    if (!(eps >= 0.0)) return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm_grad: eps must be a number >= 0");
    const int size = rows::type_bytes(type);
    if (!weight || rows::address_bits(weight) % rows::type_bytes(weight_type) || rows::address_bits(dweight) % rows::type_bytes(weight_type) ||
        rows::address_bits(dx) % size ||
        (rows > 0 && (bad_rows(dy, dy_stride, type) || bad_rows(x, x_stride, type) || (dtotal && bad_rows(dtotal, dtotal_stride, type)))))
        return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm_grad: null or misaligned pointer, or bad stride");
    const auto st = static_cast<cudaStream_t>(stream);
    if (rows == 0)
        return dweight ? finish(cudaMemsetAsync(dweight, 0, (size_t)width * rows::type_bytes(weight_type), st), what) : HB_OK;
    if (!dx && !dweight) return HB_OK;
    if (!workspace || rows::address_bits(workspace) % 256)
        return abi_fail(HB_BAD_ARGUMENT, "hb_rms_norm_grad: the workspace must be 256-byte aligned");
    if (workspace_bytes < hb_rms_norm_grad_workspace(rows, width))
        return abi_fail(HB_WORKSPACE, "workspace smaller than hb_rms_norm_grad_workspace()");
    const size_t sums = width > kMostHeld ? ((size_t)rows * 2 * sizeof(float) + 255) / 256 * 256 : 0;
    float* const stats = static_cast<float*>(workspace);
    float* const partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + sums);
    Backward p{dy, x, dtotal, weight, dy_stride, x_stride, dtotal_stride, rows, (int)width, weight_type, rows::address_bits(weight) % 16 == 0, (float)eps, dx,
               dweight ? partial : nullptr, stats};
    uint64_t bits = rows::address_bits(dy) | rows::address_bits(x) | rows::address_bits(dtotal) | rows::address_bits(dx) |
                    (uint64_t)(width | (rows > 1 ? x_stride | dy_stride : 0) | (rows > 1 && dtotal ? dtotal_stride : 0)) * size;
    int parts = 0;
    for_vectors(type, vector_of(bits, type), [&](auto t, auto vb) {
        using T = decltype(t);
        constexpr int VB = decltype(vb)::value, N = VB / (int)sizeof(T);
        if (width <= kMostHeld) {
            for_width<N>(width, [&](auto threads, auto columns) {
                constexpr int THREADS = decltype(threads)::value, COLUMNS = decltype(columns)::value;
                if constexpr (COLUMNS > 0) {
                    parts = parts_of(rows, THREADS, COLUMNS);
                    backward_kernel<T, VB, THREADS, COLUMNS><<<parts, block_of(THREADS), 0, st>>>(p);
                }
            });
            count_launches(1);
            return;
        }
        wide_sums_kernel<T, VB><<<(unsigned)rows, 512, 0, st>>>(p);
        const unsigned columns = (unsigned)((width + 256 * N - 1) / (256 * N));
        parts = (int)std::min<int64_t>(rows, std::max<int64_t>(1, 148 * 8 / columns));
        wide_kernel<T, VB><<<dim3(columns, parts), 256, 0, st>>>(p);
        count_launches(2);
    });
    if (dweight) {
        join_kernel<<<(unsigned)((width + 31) / 32), 256, 0, st>>>(partial, parts, (int)width, dweight, weight_type);
        count_launches(1);
    }
    return finish(cudaGetLastError(), what);
}
