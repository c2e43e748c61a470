// What the kernels of the experts' products share: the rows of each expert, the
// activations, and the forms that experts.cu hands to experts_simt.cu.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "rows.cuh"

namespace hb {
namespace experts {

// Forms of a product.  Row forms go over the rows of each expert, kWeights over each expert's weight.
//   kProduct    out = a b^T                    kGated      out = act(a b0^T) * (a b1^T)
//   kGatedGrad  out0 = dh u act'(g), out1 = dh act(g), g = a b0^T, u = a b1^T
//   kBack       out = sum over segments a b    kWeights    out = a^T b over the expert's rows
enum Form { kProduct, kGated, kGatedGrad, kBack, kWeights };
constexpr int kSilu = 0, kGelu = 1;
constexpr int kMostGroups = 2048;  // experts of a call: their first rows and tiles lie in shared memory

struct Operand {
    const void* p;
    int64_t row, group;  // distance of rows and of experts in elements (group: weights alone)
};

// One product, types and sizes as the C entry checked them.
struct Job {
    int type, form, activation;
    const int32_t* offsets;  // null: all rows are the only expert's
    int groups, rows;
    int n, k;                // columns of the output; summed length (kWeights: n x k columns of a and b: out is [n][k])
    Operand a[2], b[2];
    Operand dh;              // kGatedGrad
    void* out[2];
    int64_t out_row;         // distance of the outputs' rows in elements
    int segments;            // kBack: products added up; kWeights: products side by side (a[i], out[i])
    int splits;              // kWeights: parts of the expert's rows that are summed apart; above 1 they go to `partial`,
    float* partial;          // fp32 [splits][segments][groups][n][k], and are added in order
};

// The part `split` of an expert's `length` rows: whole stages of 64.
__host__ __device__ inline void split_rows(int length, int splits, int split, int& begin, int& end) {
    const int stages = ((length + 63) / 64 + splits - 1) / splits;
    begin = (int)(length < (int64_t)split * stages * 64 ? length : (int64_t)split * stages * 64);
    end = (int)(length < (int64_t)begin + stages * 64 ? length : (int64_t)begin + stages * 64);
}

// The expert's rows [begin, end): offsets are read as their running maximum inside 0..rows, so that whatever they hold
// the experts' rows are apart and inside.  Group `groups` is the rows behind the last expert.  Fills start[0..groups+1]
// and tile[0..groups+1], the number of tiles of TILE rows before each group; called by a whole block.
__device__ inline void read_groups(const int32_t* offsets, int groups, int rows, int tile_rows, int* start, int* tile) {
    const int t = threadIdx.x;
    if (!offsets) {
        if (t == 0) start[0] = 0, start[1] = start[2] = rows;
    } else if (t < 32) {  // running maximum, 32 at a time
        int most = 0;
        for (int base = 0; base <= groups; base += 32) {
            const int i = base + t;
            int v = i == 0 || i > groups ? 0 : min(max(offsets[i], 0), rows);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, v, d);
                if (t >= d) v = max(v, o);
            }
            v = max(v, most);
            if (i <= groups) start[i] = v;
            most = __shfl_sync(0xffffffffu, v, 31);
        }
        if (t == 0) start[groups + 1] = rows;
    }
    __syncthreads();
    if (t < 32) {  // sums of tiles
        int before = 0;
        for (int base = 0; base <= groups; base += 32) {
            const int i = base + t;
            const int own = i <= groups ? (start[i + 1] - start[i] + tile_rows - 1) / tile_rows : 0;
            int v = own;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, v, d);
                if (t >= d) v += o;
            }
            if (i <= groups) tile[i] = before + v - own;
            before += __shfl_sync(0xffffffffu, v, 31);
        }
        if (t == 0) tile[groups + 1] = before;
    }
    __syncthreads();
}

// The group of a tile: the last one whose first tile is at or before it and that has tiles.
__device__ inline int group_of(const int* tile, int groups, int t) {
    int lo = 0, hi = groups;  // groups + 1 of them
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tile[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// act(g) and, with SLOPE, act'(g).  PRECISE: results that are held in 32 bits.  Otherwise approximate exponentials and
// inverses, each within 2^-22 of itself, below them the rounding of the exponential's argument: silu is within
// (4 + 2 |g|) 2^-23 of itself (0 from g = -87 on, where its inverse leaves the normal numbers), gelu within
// 2^-19 + g^2 2^-23, and a 16-bit result is rounded by 2^-11 or 2^-8.
__device__ __forceinline__ float power_of_two(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float inverse_of(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <bool PRECISE>
__device__ __forceinline__ float sigmoid(float g) {
    if (PRECISE) return 1.0f / (1.0f + expf(-g));
    return inverse_of(1.0f + power_of_two(g * -1.4426950408889634f));
}
template <bool PRECISE, bool SLOPE>
__device__ __forceinline__ float activate(int kind, float g, float& slope) {
    if (kind == kSilu) {
        const float s = sigmoid<PRECISE>(g);
        if (SLOPE) slope = s * fmaf(g, 1.0f - s, 1.0f);
        return g * s;
    }
    float cdf, bell = 0.0f;
    if (PRECISE) {
        cdf = normcdff(g);  // relative on the left too, where 1 + erf cancels (4 % off at -5, 0 from -6 on)
        if (SLOPE) bell = expf(-0.5f * g * g);
    } else {
        // The normal distribution's tail as t P(t) exp(-g^2 / 2) with t = 1 / (1 + 0.26 |g|).  P is a least-maximum fit of
        // the relative error up to |g| = 14, there 1.2e-6 and at 0 a fifth of that: a form with an absolute bound (1.5e-7)
        // is 1 % off at -8.  (The gated product of 73879 x 6 x 190 x 696 f16, which erff bound: 141 -> 104 us.)
        const float z = fabsf(g), t = inverse_of(fmaf(0.26f, z, 1.0f));
        bell = power_of_two(z * z * -0.72134752044448170f);
        float poly = fmaf(t, -0.07291857624580797f, 0.2288692421997913f);
        poly = fmaf(t, poly, -0.10639618748002432f);
        poly = fmaf(t, poly, 0.16648443600537696f);
        poly = fmaf(t, poly, 0.07324207014058234f);
        poly = fmaf(t, poly, 0.10720565848608428f);
        poly = fmaf(t, poly, 0.10351347417893313f);
        const float tail = t * poly * bell;
        cdf = g < 0.0f ? tail : 1.0f - tail;  // a NaN stays
    }
    if (SLOPE) slope = fmaf(g * 0.39894228040143268f, bell, cdf);
    return g * cdf;
}

// Whether a forward product streams the weights by warps (experts_simt.cu): few rows, or few for each expert in fp32 or where
// there is little work.  Gated, streamed and in tiles (us): 64 x 64 x 512 x 512 f32 29 and 125, 128 x 64 41 and 126,
// 273 x 73 x 25 x 24 f16 8.6 and 12.5; but 487 x 117 x 18 x 50 f16 18.7 and 14.7, 200 x 4 x 128 x 128 f16 29 and 8.
// The counts lie on the device, so the rule goes by their average: where one of 128 experts has all of 512 rows, 1024 x 1024
// f32 takes 860 us, and 210 in tiles.
constexpr int64_t kFewRows = 16, kFewEach = 4, kFewWork = 1 << 24;  // rows, rows an expert, products
inline bool is_few(int type, int64_t rows, int64_t experts, int64_t n, int64_t k, int weights) {
    return rows <= kFewRows || (rows <= kFewEach * experts && (type == HB_F32 || rows * n * k * weights <= kFewWork));
}
cudaError_t few_rows(const Job& job, cudaStream_t st);
cudaError_t product_f32(const Job& job, cudaStream_t st);
// The side of product_f32's tiles: 64 where those of 128 would be fewer than 1.5 an SM.  Product, with 64 and 128 (us):
// 8198 x 8 x 257 x 129 (136 tiles of 128) 31 and 37, 8192 x 8 x 512 x 512 (272 tiles) 117 and 103.
int f32_tile(const Job& job);
// Adds the parts of kWeights in order and rounds them once.
cudaError_t join_parts(const Job& job, cudaStream_t st);

}  // namespace experts
}  // namespace hb
