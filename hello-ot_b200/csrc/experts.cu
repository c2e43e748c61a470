// Products of rows sorted by expert with each expert's weight, on the tensor cores (fp16, bf16).
//
//   product   y[r] = x[r] W[e]^T                        e the expert of row r
//   gated     h[r] = act(x[r] Wg[e]^T) * (x[r] Wu[e]^T)
//   backward  dx[r] = dy[r] W[e],  dW[e] = sum over the expert's rows of dy[r]^T x[r]; of the gated form
//             dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//
// One persistent kernel per product: a TMA producer, one thread that issues tcgen05.mma, 16 warps that
// read the accumulators.  A CTA pair (cta_group::2) takes a tile of 256 x 256 of the output, each CTA with
// its own 128 rows of one operand and 128 of the other's 256, 64 of the summed length a stage, five stages;
// the accumulators are fp32 in TMEM, twice, so that a tile is written while the next one is summed.  Experts
// of up to 128 rows on average take single CTAs and tiles of 128 x 128, where half of a pair's rows
// would be foreign (64 x 128 rows x 2048 x 1024 gated: 105 us, in pairs 120; 64 x 256 rows in pairs 124).
// In the gated forms the even CTA brings 128 rows of Wg and the odd one the same rows of Wu: columns 0-127 of
// the accumulator are g, 128-255 are u, and one thread holds both of a place, so g and u never leave the
// chip.  The gradients compute g and u again: it costs 2 of 6 products, and saves two arrays of rows x hidden
// that, kept in 16 bits, would put two more roundings into every gradient.  dg and du do go through memory in
// 16 bits, as operands of kind::f16 have to be: one rounding more, and a bf16 gradient's error from 0.0017 to 0.0023.
//
// Bound by the tensor cores from some hundred rows an expert on: 65536 rows of 32 experts, 2048 x 1024 bf16,
// calls one after the other on three sets of inputs: product 206 us (1334 TFLOP/s), gated 396 (1388), dx 280 to 350
// (982 to 785), dW 222 (1238); 16384 x 8192 x 8192 product 1445 us (1522).  With fewer rows the weights' bytes: 64 x 128
// rows gated 105 us for 537 MB.  What one product writes comes out of the same SM that sums the next, so short
// sums (dx's, 1024) stay further from the rate.
//
// The rows of an expert begin anywhere: TMA boxes may (only the innermost coordinate has to lie on 16
// bytes), rows of the next expert that a tile's box brings along are summed and not written.  In the sum
// over an expert's rows (dW) they have to be zeros instead, of both operands (0 * NaN): the box that holds
// the expert's end completes on a barrier of its own CTA, a warp of its own zeroes the foreign rows and
// hands the stage on.
#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "experts.cuh"
#include "internal.h"

namespace hb {
namespace experts {

constexpr int BK = 64, kStages = 5, kEpiWarps = 16;
// producer, issuer, writers, and in kWeights a warp that zeroes foreign rows
constexpr int threads_of(int form) { return 64 + 32 * kEpiWarps + (form == kWeights ? 32 : 0); }
constexpr int kTileBytes = 128 * BK * 2, kStageBytes = 2 * kTileBytes;
constexpr int kBand = 8;  // row tiles that share a weight tile while it is in L2 (16384 x 8192 x 8192 1445 us, with 4 1480, with 16 1460)

struct Params {
    CUtensorMap a[2], b[2];
    const int32_t* offsets;
    int groups, rows, n, k, segments, activation;
    int col_tiles, row_tiles;  // row_tiles: kWeights alone
    int splits;                // kWeights
    int blocked[2];            // operands read across the summed length whose columns are whole boxes of 64: a, b
    float* partial;
    const void* dh;
    int64_t dh_row;
    void* out[2];
    int64_t out_row;  // distance of the outputs' rows in elements
};

struct __align__(1024) Smem {
    uint8_t stage[kStages][kStageBytes];
    __align__(16) uint8_t out[kEpiWarps][32 * 64];  // a warp's 32 rows x 64 bytes on their way out
    int start[kMostGroups + 2], tile[kMostGroups + 2];
    uint64_t full[kStages], empty[kStages], tail[kStages], tfull[2], tempty[2];
    uint32_t tmem_base;
    int abort, status;
};
constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
static_assert(kSmemBytes <= 227 * 1024, "dynamic shared memory above the 227 KB a CTA may use");

// ---------------------------------------------------------------- instructions
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
    tma_load_2d(dst, map, bar, c0, c1);
}
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
// Arrive, with bytes to come, on an mbarrier of either CTA of the cluster (address from peer_smem).  Relaxed: the stage's
// data are ordered by the copies' completion, and a release to the cluster would fence the thread at every stage
// (the products of 256-row tiles ran at 700 TFLOP/s with it).
__device__ __forceinline__ void arrive_expect_cluster(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
__device__ __forceinline__ void load_4d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
// Arrive on an mbarrier of the other CTA after reading TMEM (whose loads have been waited for): nothing in memory is
// handed over, so no release either.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Smem& s) {
    return mbar_wait_timed<PAIR>(bar, parity, &s.abort, &s.status);
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A tile stored with the 128-byte swizzle whose rows are the summed length (K rows of 64 columns of the output
// dimension, 128 bytes): 8 rows are 1024 bytes, the next 64 columns are a box of BK rows further.
__device__ __forceinline__ uint64_t desc_columns(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)((BK * 128) >> 4) << 16;  // leading byte offset: the next 64 columns
    d |= (uint64_t)(1024 >> 4) << 32;        // stride byte offset: the next 8 rows
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// Instruction descriptor of kind::f16: fp32 accumulators, both operands bf16 or both fp16, each read along the summed
// length or (columns) across it.
__host__ __device__ constexpr uint32_t idesc(bool bf16, bool a_columns, bool b_columns, int m, int n) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_columns ? 1u : 0u) << 15) |
           ((b_columns ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// ---------------------------------------------------------------- tiles
template <int FORM, bool PAIR>
struct Shape {
    static constexpr bool kHalves = FORM == kGated || FORM == kGatedGrad;  // the accumulator is [g | u]
    static constexpr bool kAColumns = FORM == kWeights, kBColumns = FORM == kWeights || FORM == kBack;
    static constexpr int M = PAIR ? 256 : 128, N = PAIR ? 256 : 128;  // of the accumulator, over the pair
    static constexpr int kCols = kHalves ? N / 2 : N;                 // output columns
    static constexpr uint32_t kTmemCols = 2 * N;
};

struct Tile {
    int group, row, rows;  // group; first row of this CTA in the output; rows of the group from there (may be <= 0)
    int col;               // first column
    int part, split;       // kWeights: which product, which part of the rows
    int begin, length;     // kWeights: the rows to sum over
    int blocks;            // stages; 0: the output is zeros
};

template <int FORM, bool PAIR>
__device__ __forceinline__ int tiles_of(const Params& p, const Smem& s) {
    if (FORM == kWeights) return p.splits * p.segments * p.groups * p.row_tiles * p.col_tiles;
    return s.tile[p.groups + 1] * p.col_tiles;
}

template <int FORM, bool PAIR>
__device__ __forceinline__ Tile tile_at(const Params& p, const Smem& s, int u, int rank) {
    using S = Shape<FORM, PAIR>;
    Tile t;
    int local, row_tiles;
    if (FORM == kWeights) {
        row_tiles = p.row_tiles;
        const int per = row_tiles * p.col_tiles;
        t.group = u / per;
        local = u - t.group * per;
        t.part = t.group % p.segments;
        t.group /= p.segments;
        t.split = t.group % p.splits;
        t.group /= p.splits;
        int end;
        split_rows(s.start[t.group + 1] - s.start[t.group], p.splits, t.split, t.begin, end);
        t.length = end - t.begin;
        t.begin += s.start[t.group];
        t.blocks = (t.length + BK - 1) / BK;
    } else {
        t.group = group_of(s.tile, p.groups, u / p.col_tiles);
        row_tiles = s.tile[t.group + 1] - s.tile[t.group];
        local = u - s.tile[t.group] * p.col_tiles;
        t.part = t.split = t.begin = t.length = 0;
        t.blocks = t.group == p.groups ? 0 : p.segments * ((p.k + BK - 1) / BK);
    }
    const int band = local / (kBand * p.col_tiles), in_band = local - band * kBand * p.col_tiles;
    const int deep = min(kBand, row_tiles - band * kBand);
    const int row = (band * kBand + in_band % deep) * S::M + (PAIR ? rank * 128 : 0);
    t.col = in_band / deep * S::kCols;
    if (FORM == kWeights) {
        t.row = row;
        t.rows = p.n - row;
    } else {
        t.row = s.start[t.group] + row;
        t.rows = s.start[t.group + 1] - t.row;
    }
    return t;
}

// ---------------------------------------------------------------- roles
// 128 columns x 64 rows of the summed length, two boxes of 64 columns.  Blocked: the tensor's 64-column blocks are a
// dimension of their own and one copy brings both boxes (two copies a stage and operand cost up to a tenth of the rate:
// 16384 x 8192 x 8192 in dW 1288 -> 1424 TFLOP/s).  `bar` this CTA's barrier, or `full` the pair's.
template <bool PAIR>
__device__ __forceinline__ void columns_2d(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, uint32_t full, int col, int row,
                                           int blocked) {
    if (blocked) {
        if (PAIR) load_3d_pair(dst, map, full, 0, row, col >> 6);
        else load_3d(dst, map, bar, 0, row, col >> 6);
        return;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (PAIR) tma_load_2d_pair(dst + i * BK * 128, map, full, col + i * 64, row);
        else load_2d(dst + i * BK * 128, map, bar, col + i * 64, row);
    }
}
template <bool PAIR>
__device__ __forceinline__ void columns_3d(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, uint32_t full, int col, int row,
                                           int group, int blocked) {
    if (blocked) {
        if (PAIR) load_4d_pair(dst, map, full, 0, row, col >> 6, group);
        else load_4d(dst, map, bar, 0, row, col >> 6, group);
        return;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (PAIR) load_3d_pair(dst + i * BK * 128, map, full, col + i * 64, row, group);
        else load_3d(dst + i * BK * 128, map, bar, col + i * 64, row, group);
    }
}

// Lane 0 waits for its warp, which goes on or gives up as one.
template <bool PAIR>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, Smem& s) {
    bool ok = true;
    if ((threadIdx.x & 31) == 0) ok = wait<PAIR>(bar, parity, s);
    return __shfl_sync(0xffffffffu, ok, 0);
}

// The producer's warp; lane 0 issues the loads.  Every stage brings 128 rows of each operand for this CTA.  With pairs
// the completions of both CTAs count on the even one's barrier.
template <int FORM, bool PAIR>
__device__ __forceinline__ void produce(const Params& p, Smem& s, int rank) {
    using S = Shape<FORM, PAIR>;
    const int lane = threadIdx.x & 31;
    uint32_t stage = 0, phase = 0;
    const int units = tiles_of<FORM, PAIR>(p, s);
    const int per_segment = (p.k + BK - 1) / BK;
    for (int u = blockIdx.x / (PAIR ? 2 : 1); u < units; u += gridDim.x / (PAIR ? 2 : 1)) {
        const Tile t = tile_at<FORM, PAIR>(p, s, u, rank);
        for (int kb = 0; kb < t.blocks; ++kb) {
            if (!warp_wait<PAIR>(&s.empty[stage], phase ^ 1, s)) return;
            uint8_t *a = s.stage[stage], *b = a + kTileBytes;
            const uint32_t full = PAIR ? peer_smem(&s.full[stage], 0) : 0u;
            if (FORM == kWeights) {
                const int row = t.begin + kb * BK, left = t.length - kb * BK;
                const int bcol = t.col + (PAIR ? rank * 128 : 0);
                const CUtensorMap* am = &p.a[t.part];
                if (left >= BK) {
                    if (lane == 0) {
                        if (PAIR) arrive_expect_cluster(full, kStageBytes);
                        else mbar_arrive_expect_tx(&s.full[stage], kStageBytes);
                        columns_2d<PAIR>(a, am, &s.full[stage], full, t.row, row, p.blocked[0]);
                        columns_2d<PAIR>(b, &p.b[0], &s.full[stage], full, bcol, row, p.blocked[1]);
                    }
                } else if (lane == 0) {  // rows of the next expert are in the box: clean_tails hands the stage on
                    mbar_arrive_expect_tx(&s.tail[stage], kStageBytes);
                    columns_2d<false>(a, am, &s.tail[stage], 0, t.row, row, p.blocked[0]);
                    columns_2d<false>(b, &p.b[0], &s.tail[stage], 0, bcol, row, p.blocked[1]);
                }
            } else if (lane == 0) {
                const int seg = FORM == kBack ? kb / per_segment : 0;
                const int k0 = (kb - seg * per_segment) * BK;
                if (PAIR) {
                    arrive_expect_cluster(full, kStageBytes);
                    tma_load_2d_pair(a, &p.a[seg], full, k0, t.row);
                    if (FORM == kBack) {
                        columns_3d<true>(b, &p.b[seg], nullptr, full, t.col + rank * 128, k0, t.group, p.blocked[1]);
                    } else if (S::kHalves) {
                        load_3d_pair(b, &p.b[rank], full, k0, t.col, t.group);
                    } else {
                        load_3d_pair(b, &p.b[0], full, k0, t.col + rank * 128, t.group);
                    }
                } else {
                    uint64_t* bar = &s.full[stage];
                    mbar_arrive_expect_tx(bar, kStageBytes);
                    load_2d(a, &p.a[seg], bar, k0, t.row);
                    if (FORM == kBack) {
                        columns_3d<false>(b, &p.b[seg], bar, 0, t.col, k0, t.group, p.blocked[1]);
                    } else if (S::kHalves) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) load_3d(b + i * 64 * 128, &p.b[i], bar, k0, t.col, t.group);
                    } else {
                        load_3d(b, &p.b[0], bar, k0, t.col, t.group);
                    }
                }
            }
            if (++stage == kStages) stage = 0, phase ^= 1;
        }
    }
}

// kWeights: a warp zeroes the rows behind the end of the summed ones in the stage that holds it, of both operands, and
// hands the stage on; the producer goes on meanwhile (one that waited for each end took twice as long where experts
// have few rows).
template <bool PAIR>
__device__ __forceinline__ void clean_tails(const Params& p, Smem& s, int rank) {
    const int lane = threadIdx.x & 31;
    uint32_t stage = 0, phases = 0;
    const int units = tiles_of<kWeights, PAIR>(p, s);
    for (int u = blockIdx.x / (PAIR ? 2 : 1); u < units; u += gridDim.x / (PAIR ? 2 : 1)) {
        const Tile t = tile_at<kWeights, PAIR>(p, s, u, rank);
        stage = (stage + t.blocks) % kStages;
        const int left = t.length % BK;
        if (left == 0) continue;
        const uint32_t last = (stage + kStages - 1) % kStages;
        if (!warp_wait<false>(&s.tail[last], phases >> last & 1, s)) return;
        phases ^= 1u << last;
        const int words = (BK - left) * 8;  // 16 bytes each, of every box
        for (int i = lane; i < words; i += 32)
#pragma unroll
            for (int box = 0; box < 4; ++box)
                *reinterpret_cast<uint4*>(s.stage[last] + box * BK * 128 + left * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
            if (PAIR) mbar_arrive_remote(peer_smem(&s.full[last], 0));
            else mbar_arrive(&s.full[last]);
        }
    }
}

// One thread (of the even CTA) issues the products; commits release the stages and hand over the accumulator.
template <int FORM, bool PAIR, bool BF16>
__device__ __forceinline__ void multiply(const Params& p, Smem& s, uint32_t tmem) {
    using S = Shape<FORM, PAIR>;
    constexpr uint32_t ID = idesc(BF16, S::kAColumns, S::kBColumns, S::M, S::N);
    auto commit = [](uint64_t* bar) {
        if (PAIR) mma_commit_pair(bar);
        else mma_commit(bar);
    };
    uint32_t stage = 0, phase = 0, done = 0;
    const int units = tiles_of<FORM, PAIR>(p, s), step = gridDim.x / (PAIR ? 2 : 1);
    // Stages of a tile; the next tile's are looked up while this one's products are under way.
    const int summed = FORM == kWeights ? 0 : s.tile[p.groups] * p.col_tiles, each = p.segments * ((p.k + BK - 1) / BK);
    auto blocks_of = [&](int u) {
        if (u >= units) return 0;
        if constexpr (FORM == kWeights) return tile_at<FORM, PAIR>(p, s, u, 0).blocks;
        else return u < summed ? each : 0;
    };
    int u = blockIdx.x / (PAIR ? 2 : 1), blocks = blocks_of(u);
    for (; u < units; u += step) {
        if (blocks == 0) {
            blocks = blocks_of(u + step);
            continue;
        }
        int next = 0;
        const uint32_t buf = done & 1;
        if (!wait<PAIR>(&s.tempty[buf], ((done >> 1) & 1) ^ 1, s)) return;
        tc_fence_after();
        const uint32_t d = tmem + buf * S::N;
        for (int kb = 0; kb < blocks; ++kb) {
            if (!wait<PAIR>(&s.full[stage], phase, s)) return;
            tc_fence_after();
            const uint32_t a = smem_u32(s.stage[stage]), b = a + kTileBytes;
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
                const uint64_t ad = S::kAColumns ? desc_columns(a + kk * 16 * 128) : smem_desc_sw128(a + kk * 32);
                const uint64_t bd = S::kBColumns ? desc_columns(b + kk * 16 * 128) : smem_desc_sw128(b + kk * 32);
                if (PAIR) mma_f16_pair(d, ad, bd, ID, (kb | kk) != 0);
                else mma_f16(d, ad, bd, ID, (kb | kk) != 0);
            }
            commit(&s.empty[stage]);
            if (++stage == kStages) stage = 0, phase ^= 1;
            if (kb == 0) next = blocks_of(u + step);
        }
        commit(&s.tfull[buf]);
        ++done;
        blocks = next;
    }
}

// 16 columns of a warp's 32 rows: lane l gets row l.  Waited for by tmem_wait16.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&r)[16]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
          "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait16(float (&r)[16]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]),
                   "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15])
                 ::"memory");
}

// A thread's 16 values of its row as the words of T that they round to: 32 or 64 bytes.
template <typename T>
union Row16 {
    uint4 word[sizeof(T)];
    T t[16];
    __device__ __forceinline__ Row16() {}
    __device__ __forceinline__ void hold(const float (&v)[16]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) t[i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(t + i) = __floats2half2_rn(v[i], v[i + 1]);
                else *reinterpret_cast<__nv_bfloat162*>(t + i) = __floats2bfloat162_rn(v[i], v[i + 1]);
            }
        }
    }
};

// Where a warp's chunk of 32 rows goes: 64 bytes of each (COLS values of T), through shared memory, so that rows leave in
// whole sectors.  The swizzle keeps 8 rows' 16-byte words in different banks.
template <typename T>
struct Writer {
    static constexpr int COLS = 64 / (int)sizeof(T), V = 16 / (int)sizeof(T);
    uint8_t* buf;
    int lane, unit;  // unit: bytes (16, 4 or a value) that rows lie on
    // Words first..first + N of this thread's row.
    template <int N>
    __device__ __forceinline__ void stage(const uint4 (&word)[N], int first) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            *reinterpret_cast<uint4*>(buf + lane * 64 + (((first + j) ^ ((lane >> 1) & 3)) << 4)) = word[j];
    }
    // The staged chunk to `to`, `stride` values between rows; `rows` and `cols` how many there are.
    __device__ __forceinline__ void write(T* to, int64_t stride, int rows, int cols) {
        __syncwarp();
        if (unit == 16) {
            const int j = lane & 3;
            to += (lane >> 2) * stride + j * V;
            if (j * V < cols) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = i * 8 + (lane >> 2);
                    if (row < rows)
                        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(buf + row * 64 + ((j ^ ((row >> 1) & 3)) << 4));
                    to += 8 * stride;
                }
            }
        } else if (unit == 4) {
            constexpr int W = 4 / (int)sizeof(T);  // rows are even, so the end cuts no word
            const int w = lane & 15, j = w >> 2;
            to += (lane >> 4) * stride + w * W;
            if (w * W < cols)
#pragma unroll 4
                for (int row = lane >> 4; row < rows; row += 2, to += 2 * stride)
                    *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(buf + row * 64 + ((j ^ ((row >> 1) & 3)) << 4) + (w & 3) * 4);
        } else {
            const int c = lane % COLS, j = c / V, in = c % V * (int)sizeof(T);
            to += lane / COLS * stride + c;
            if (c < cols)
#pragma unroll 4
                for (int row = lane / COLS; row < rows; row += 32 / COLS, to += 32 / COLS * stride)
                    *to = *reinterpret_cast<const T*>(buf + row * 64 + ((j ^ ((row >> 1) & 3)) << 4) + in);
        }
        __syncwarp();
    }
};

// A chunk of 32 rows x 32 values on its way in: 8 rows' 64 bytes an instruction, held in registers until the sums are
// there, then through the same shared memory to the thread of each row.
template <typename T>
struct Reader {
    uint4 word[4];
    bool vectors;
    int lane;
    __device__ __forceinline__ void load(const T* from, int64_t stride, int rows, int cols) {
        if (!vectors) return;
        const int j = lane & 3;
        from += (lane >> 2) * stride + j * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            word[i] = make_uint4(0, 0, 0, 0);
            if (i * 8 + (lane >> 2) < rows && j * 8 < cols) word[i] = __ldcs(reinterpret_cast<const uint4*>(from));
            from += 8 * stride;
        }
    }
    __device__ __forceinline__ void stage(uint8_t* buf, const T* from, int64_t stride, int rows, int cols) const {
        if (vectors) {
            const int j = lane & 3;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = i * 8 + (lane >> 2);
                *reinterpret_cast<uint4*>(buf + row * 64 + ((j ^ ((row >> 1) & 3)) << 4)) = word[i];
            }
        } else {
            const int j = lane >> 3, in = (lane & 7) * 2;
#pragma unroll 4
            for (int row = 0; row < 32; ++row)
                *reinterpret_cast<T*>(buf + row * 64 + ((j ^ ((row >> 1) & 3)) << 4) + in) =
                    row < rows && lane < cols ? from[row * stride + lane] : rows::from_float<T>(0.0f);
        }
        __syncwarp();
    }
    // This thread's row; the shared memory is free again.
    __device__ __forceinline__ void take(const uint8_t* buf) {
#pragma unroll
        for (int q = 0; q < 4; ++q) word[q] = *reinterpret_cast<const uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4));
        __syncwarp();
    }
    __device__ __forceinline__ void values(int h, float (&v)[16]) const {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            rows::Vec<T, 16> w;
            w.raw = word[2 * h + q];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[q * 8 + i] = rows::to_float(w.v[i]);
        }
    }
};

// g and u of 16 places to the outputs: h in v, or dg in v and du in w.
template <int FORM, int ACTIVATION>
__device__ __forceinline__ void combine(float (&v)[16], float (&w)[16], const float (&d)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float slope;
        const float a = activate<false, FORM == kGatedGrad>(ACTIVATION, v[i], slope);
        if (FORM == kGated) {
            v[i] = a * w[i];
        } else {
            v[i] = d[i] * w[i] * slope;
            w[i] = d[i] * a;
        }
    }
}

// Four warps a TMEM lane quarter, each on a quarter of the output's columns.  A wait that gave up leaves NaN.
template <int FORM, bool PAIR, typename T>
__device__ __forceinline__ void write_out(const Params& p, Smem& s, uint32_t tmem, int rank) {
    using S = Shape<FORM, PAIR>;
    constexpr int kSlice = S::kCols / 4, kChunk = kSlice < 32 ? kSlice : 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int quarter = warp & 3, slice = (warp - 2) >> 2;
    const uint32_t tempty = PAIR ? peer_smem(&s.tempty[0], 0) : 0u;
    const int width = FORM == kWeights ? p.k : p.n;
    // what all rows of the outputs lie on
    const uint64_t grid = (uint64_t)p.out_row * 2 | reinterpret_cast<uintptr_t>(p.out[0]) | reinterpret_cast<uintptr_t>(p.out[1]);
    Writer<T> writer{s.out[warp - 2], lane, grid % 16 == 0 ? 16 : grid % 4 == 0 ? 4 : 2};
    Writer<float> writer32{s.out[warp - 2], lane, p.k % 4 == 0 ? 16 : 4};
    Reader<T> reader;  // kGatedGrad
    reader.lane = lane;
    reader.vectors = p.dh_row % 8 == 0 && width % 8 == 0 && (reinterpret_cast<uintptr_t>(p.dh) & 15) == 0;
    uint32_t done = 0;
    bool good = true;
    const int units = tiles_of<FORM, PAIR>(p, s);
    for (int u = blockIdx.x / (PAIR ? 2 : 1); u < units; u += gridDim.x / (PAIR ? 2 : 1)) {
        const Tile t = tile_at<FORM, PAIR>(p, s, u, rank);
        const uint32_t acc = done & 1;
        const bool summed = t.blocks != 0;
        const T* dh = nullptr;
        if constexpr (FORM == kGatedGrad) {  // on its way while the tile is summed
            static_assert(kSlice == kChunk, "one chunk a warp");
            const int64_t first = (int64_t)(t.row + quarter * 32) * p.dh_row + t.col + slice * kSlice;
            dh = static_cast<const T*>(p.dh) + first;
            if (summed) reader.load(dh, p.dh_row, min(32, t.rows - quarter * 32), min(kChunk, width - t.col - slice * kSlice));
        }
        if (summed) {
            good = __all_sync(0xffffffffu, good && wait<PAIR>(&s.tfull[acc], (done >> 1) & 1, s));  // a warp goes on as one
            tc_fence_after();
        }
        const int row0 = quarter * 32, col0 = t.col + slice * kSlice;
        const int rows = min(32, t.rows - row0);  // of this warp; may be <= 0
        T* out = static_cast<T*>(p.out[FORM == kWeights ? t.part : 0]);
        float* partial = nullptr;
        if (FORM == kWeights) {
            out += (int64_t)t.group * p.n * p.out_row;
            if (p.splits > 1) partial = p.partial + (((int64_t)t.split * p.segments + t.part) * p.groups + t.group) * p.n * p.k;
        }
        const int64_t at = (int64_t)(t.row + row0) * p.out_row + col0;
        const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + acc * S::N + slice * kSlice;
#pragma unroll
        for (int c = 0; c < kSlice; c += kChunk) {
            const int cols = min(kChunk, width - col0 - c);
            if (rows <= 0 || cols <= 0) break;  // the same for the whole warp
            const bool filled = summed && good;
            float v[kChunk / 16][16], w[S::kHalves ? kChunk / 16 : 1][16];
            Row16<T> second[FORM == kGatedGrad ? kChunk / 16 : 1];
            if constexpr (FORM == kGatedGrad)
                if (filled) {
                    reader.stage(s.out[warp - 2], dh, p.dh_row, rows, cols);
                    reader.take(s.out[warp - 2]);
                }
            if (FORM != kGatedGrad && filled) {
#pragma unroll
                for (int h = 0; h < kChunk / 16; ++h) {
                    tmem_ld16(taddr + c + h * 16, v[h]);
                    if constexpr (S::kHalves) tmem_ld16(taddr + S::N / 2 + c + h * 16, w[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < kChunk / 16; ++h) {
                if (!filled) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[h][i] = good ? 0.0f : __int_as_float(0x7fc00000);
                    if constexpr (FORM == kGatedGrad) second[h].hold(v[h]);
                } else if constexpr (S::kHalves) {
                    float d[16];
                    if constexpr (FORM == kGatedGrad) {  // half a chunk at a time: registers
                        tmem_ld16(taddr + c + h * 16, v[h]);
                        tmem_ld16(taddr + S::N / 2 + c + h * 16, w[h]);
                        reader.values(h, d);
                    }
                    tmem_wait16(v[h]);
                    tmem_wait16(w[h]);
                    if (p.activation == kSilu) combine<FORM, kSilu>(v[h], w[h], d);
                    else combine<FORM, kGelu>(v[h], w[h], d);
                    if constexpr (FORM == kGatedGrad) second[h].hold(w[h]);
                } else {
                    tmem_wait16(v[h]);
                }
                if (FORM == kWeights && partial) {
                    Row16<float> r;
                    r.hold(v[h]);
                    writer32.stage(r.word, 0);
                    writer32.write(partial + at + c + h * 16, p.k, rows, cols - h * 16);
                } else {
                    Row16<T> r;
                    r.hold(v[h]);
                    writer.stage(r.word, 2 * h);
                }
            }
            if (FORM == kWeights && partial) continue;
            writer.write(out + at + c, p.out_row, rows, cols);
            if constexpr (FORM == kGatedGrad) {
#pragma unroll
                for (int h = 0; h < kChunk / 16; ++h) writer.stage(second[h].word, 2 * h);
                writer.write(static_cast<T*>(p.out[1]) + at + c, p.out_row, rows, cols);
            }
        }
        if (summed) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR && rank != 0) arrive_cluster(tempty + acc * (uint32_t)sizeof(uint64_t));
                else mbar_arrive(&s.tempty[acc]);
            }
            ++done;
        }
    }
}

// With pairs both CTAs allocate TMEM together, meet after the barriers are ready and before they leave; every role
// returns to the end, after a wait that gave up too.
template <int FORM, bool PAIR, typename T>
__global__ void __launch_bounds__(threads_of(FORM), 1) expert_kernel(const __grid_constant__ Params p) {
    using S = Shape<FORM, PAIR>;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)cluster_rank() : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&s.full[i], PAIR ? 2 : 1), mbar_init(&s.empty[i], 1), mbar_init(&s.tail[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&s.tfull[i], 1), mbar_init(&s.tempty[i], kEpiWarps * (PAIR ? 2 : 1));
        s.abort = s.status = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane < 2) prefetch_tmap(&p.a[lane]), prefetch_tmap(&p.b[lane]);
    if (warp == 1) {
        if (PAIR) tmem_alloc_pair(&s.tmem_base, S::kTmemCols), tmem_relinquish_pair();
        else tmem_alloc(&s.tmem_base, S::kTmemCols), tmem_relinquish();
    }
    read_groups(p.offsets, p.groups, p.rows, S::M, s.start, s.tile);
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s.tmem_base;
    if (warp == 0) {
        produce<FORM, PAIR>(p, s, rank);
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) multiply<FORM, PAIR, BF16>(p, s, tmem);
    } else if (warp < 2 + kEpiWarps) {
        write_out<FORM, PAIR, T>(p, s, tmem, rank);
    } else if constexpr (FORM == kWeights) {
        clean_tails<PAIR>(p, s, rank);
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        if (PAIR) tmem_dealloc_pair(tmem, S::kTmemCols);
        else tmem_dealloc(tmem, S::kTmemCols);
    }
}

// ---------------------------------------------------------------- host
namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled find_encode() {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
        return reinterpret_cast<EncodeTiled>(ptr);
    cudaGetLastError();
    return nullptr;
}

// Map of [groups][rows][cols] (groups 0: two dimensions) in boxes of 64 columns (128 bytes) x box_rows, 128-byte swizzle;
// what lies outside is read as zeros.  Blocked (whole boxes of columns): two boxes side by side in one copy.
bool encode(CUtensorMap* m, const Operand& o, int type, int64_t cols, int64_t rows, int64_t groups, int box_rows, bool blocked) {
    static const EncodeTiled enc = find_encode();
    if (!enc) return false;
    const cuuint64_t most = (cuuint64_t)std::max<int64_t>(groups, 1), row = (cuuint64_t)o.row * 2, group = (cuuint64_t)o.group * 2;
    cuuint64_t dims[4] = {(cuuint64_t)cols, (cuuint64_t)rows, most, 1}, strides[3] = {row, group, 0};
    cuuint32_t box[4] = {BK, (cuuint32_t)box_rows, 1, 1};
    const cuuint32_t step[4] = {1, 1, 1, 1};
    if (blocked) {
        dims[0] = BK, dims[2] = (cuuint64_t)cols / BK, dims[3] = most;
        strides[1] = BK * 2, strides[2] = group;
        box[2] = 2;
    }
    return enc(m, type == HB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
               (groups ? 3 : 2) + (blocked ? 1 : 0), const_cast<void*>(o.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FORM, bool PAIR, typename T>
cudaError_t launch(const Params& p, int64_t tiles, cudaStream_t st) {
    const auto fn = expert_kernel<FORM, PAIR, T>;
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    int device = 0, sms = 0;
    if (e == cudaSuccess) e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = PAIR ? 2 : 1;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(PAIR ? sms / 2 * 2 : sms, tiles * (PAIR ? 2 : 1)));
    cfg.blockDim = dim3(threads_of(FORM));
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = PAIR ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, fn, p);
    count_launches(1);
    return e;
}

template <int FORM, bool PAIR>
int run_form(const Job& job, cudaStream_t st) {
    using S = Shape<FORM, PAIR>;
    Params p{};
    p.offsets = job.offsets;
    p.groups = job.groups;
    p.rows = job.rows;
    p.n = job.n;
    p.k = job.k;
    p.segments = FORM == kBack || FORM == kWeights ? job.segments : 1;
    p.activation = job.activation;
    p.dh = job.dh.p;
    p.dh_row = job.dh.row;
    p.out[0] = job.out[0];
    p.out[1] = job.out[1];
    const int width = FORM == kWeights ? job.k : job.n;
    p.out_row = job.out_row;
    p.splits = FORM == kWeights ? job.splits : 1;
    p.partial = job.partial;
    p.col_tiles = (width + S::kCols - 1) / S::kCols;
    p.row_tiles = FORM == kWeights ? (job.n + S::M - 1) / S::M : 0;
    const int64_t most = FORM == kWeights ? (int64_t)p.splits * p.segments * job.groups * p.row_tiles * p.col_tiles
                                          : ((int64_t)job.rows / S::M + job.groups + 1) * p.col_tiles;
    if (most > INT32_MAX) return abi_fail(HB_BAD_ARGUMENT, "expert product: too many tiles");
    p.blocked[0] = FORM == kWeights && job.n % BK == 0;
    p.blocked[1] = (FORM == kWeights || FORM == kBack) && width % BK == 0;
    bool ok = true;
    const int maps = S::kHalves ? 2 : p.segments;
    for (int i = 0; i < maps && ok; ++i) {
        if (FORM == kWeights) {
            ok = encode(&p.a[i], job.a[i], job.type, job.n, job.rows, 0, BK, p.blocked[0]);
            if (i == 0) ok = ok && encode(&p.b[0], job.b[0], job.type, job.k, job.rows, 0, BK, p.blocked[1]);
        } else {
            if (!S::kHalves || i == 0) ok = encode(&p.a[i], job.a[i], job.type, job.k, job.rows, 0, 128, false);
            if (FORM == kBack) ok = ok && encode(&p.b[i], job.b[i], job.type, job.n, job.k, job.groups, BK, p.blocked[1]);
            else ok = ok && encode(&p.b[i], job.b[i], job.type, job.k, job.n, job.groups, S::kHalves && !PAIR ? 64 : 128, false);
        }
    }
    if (!ok) return abi_fail(HB_TENSOR_MAP, "expert product: cuTensorMapEncodeTiled failed");
    if (maps == 1 || FORM == kWeights) p.b[1] = p.b[0];
    if (maps == 1 || S::kHalves) p.a[1] = p.a[0];
    const cudaError_t e = job.type == HB_BF16 ? launch<FORM, PAIR, __nv_bfloat16>(p, most, st) : launch<FORM, PAIR, __half>(p, most, st);
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("expert product: ") + cudaGetErrorString(e));
}

// CTA pairs where their tiles are filled: by an expert's rows (both sides measured above), or by the weight's two sides.
bool use_pairs(const Job& job) {
    return job.form == kWeights ? job.n > 128 && job.k > 128 : job.rows > 128 * (int64_t)job.groups;
}
// kWeights: parts of the rows, where the tiles alone leave most of the device idle and experts have many stages.  Parts
// against none (us): 20000 x 1 x 48 x 142 bf16 25 and 134, 131072 x 1 x 2048 x 1024 422 and 658, 8198 x 8 x 257 x 129 f32
// 35 and 45.  Parts of at least 4 stages instead of 16: 2000 x 1 x 512 x 512 bf16 19 (none: 21), but 3056 x 6 x 376 x 429
// 27 and 21.
constexpr int kSlots = 148, kLeastStages = 16;
int splits_of(const Job& job) {
    const bool f32 = job.type == HB_F32, pair = !f32 && use_pairs(job);
    const int64_t side = f32 ? f32_tile(job) : pair ? 256 : 128;
    const int64_t slots = f32 ? kSlots * (side == 128 ? 2 : 5) : pair ? kSlots / 2 : kSlots;  // resident tiles
    const int64_t tiles = job.segments * (int64_t)job.groups * ((job.n + side - 1) / side) * ((job.k + side - 1) / side);
    const int64_t stages = (job.rows / job.groups + 63) / 64;
    return (int)std::max<int64_t>(1, std::min(slots / tiles, stages / (f32 ? 2 : kLeastStages)));
}
size_t partial_bytes(const Job& job, int splits) {
    return splits > 1 ? (size_t)splits * job.segments * job.groups * job.n * job.k * sizeof(float) : 0;
}

template <int FORM>
int run_pairs(const Job& job, cudaStream_t st) {
    return use_pairs(job) ? run_form<FORM, true>(job, st) : run_form<FORM, false>(job, st);
}

int run(const Job& job, cudaStream_t st) {
    const bool row_form = job.form == kProduct || job.form == kGated;
    // a thread that has not used the device yet has no current context, which encoding a tensor map needs
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaSetDevice(device);
    if (e != cudaSuccess) return abi_fail(HB_CUDA, std::string("expert product: ") + cudaGetErrorString(e));
    if (row_form && is_few(job.type, job.rows, job.groups, job.n, job.k, job.form == kGated ? 2 : 1)) e = few_rows(job, st);
    else if (job.type == HB_F32) e = product_f32(job, st);
    else {
        int rc;
        switch (job.form) {
            case kProduct: rc = run_pairs<kProduct>(job, st); break;
            case kGated: rc = run_pairs<kGated>(job, st); break;
            case kGatedGrad: rc = run_pairs<kGatedGrad>(job, st); break;
            case kBack: rc = run_pairs<kBack>(job, st); break;
            default: rc = run_pairs<kWeights>(job, st);
        }
        if (rc) return rc;
    }
    if (e == cudaSuccess && job.form == kWeights && job.splits > 1) e = join_parts(job, st);
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("expert product: ") + cudaGetErrorString(e));
}

// ---------------------------------------------------------------- checks of the C entries
constexpr int64_t kMostWidth = 1 << 20;
bool fits(const Operand& o, int type, int64_t cols, int64_t rows, bool weights, int64_t groups, bool grid) {
    const uint64_t size = rows::type_bytes(type), unit = grid && type != HB_F32 ? 16 : size;
    if (!o.p || rows::address_bits(o.p) % unit || o.row < 0 || o.row > INT32_MAX) return false;
    if (rows > 1 && ((uint64_t)o.row * size % unit || ((weights || unit == 16) && o.row < cols))) return false;
    if (weights && groups > 1 && (o.group < 0 || o.group >= ((int64_t)1 << 38) || (uint64_t)o.group * size % unit)) return false;
    return true;
}
// Distances that are never stepped over, in the form that a tensor map takes.
Operand tidy(Operand o, int64_t cols, int64_t rows, int64_t groups) {
    if (rows <= 1) o.row = (cols + 7) / 8 * 8;
    if (groups <= 1) o.group = o.row * std::max<int64_t>(rows, 1);
    return o;
}
int check(const hb_expert_shape* s, const int32_t* offsets, const char* what) {
    const std::string at = std::string(what) + ": ";
    if (!s) return abi_fail(HB_BAD_ARGUMENT, at + "null shape");
    if (!rows::valid_type(s->type)) return abi_fail(HB_BAD_ARGUMENT, at + "element type");
    if (s->rows < 0 || s->rows > INT32_MAX - 1024 || s->width < 1 || s->hidden < 1 || s->width > kMostWidth || s->hidden > kMostWidth)
        return abi_fail(HB_BAD_ARGUMENT, at + "rows, width or hidden out of range");
    if (s->experts < 1 || s->experts > kMostGroups || (!offsets && s->experts != 1))
        return abi_fail(HB_BAD_ARGUMENT, at + "1 to 2048 experts, and one without offsets");
    if (rows::address_bits(offsets) % 4) return abi_fail(HB_BAD_ARGUMENT, at + "misaligned offsets");
    if (s->activation != HB_SILU && s->activation != HB_GELU) return abi_fail(HB_BAD_ARGUMENT, at + "activation");
    return HB_OK;
}
Job job_of(const hb_expert_shape* s, const int32_t* offsets, int form, int64_t n, int64_t k) {
    Job j{};
    j.type = s->type;
    j.form = form;
    j.activation = s->activation == HB_GELU ? kGelu : kSilu;
    j.offsets = offsets;
    j.groups = (int)s->experts;
    j.rows = (int)s->rows;
    j.n = (int)n;
    j.k = (int)k;
    j.out_row = n;
    j.segments = j.splits = 1;
    return j;
}
int64_t padded(int64_t width) { return (width + 7) / 8 * 8; }

}  // namespace
}  // namespace experts
}  // namespace hb

using namespace hb;
using namespace hb::experts;

namespace {
constexpr const char* kOperand = "an operand is null, off its grid or has a bad stride";
Operand rows_of(const void* p, int64_t stride) { return {p, stride, 0}; }
Operand weight_of(const hb_expert_weight* w) { return w ? Operand{w->data, w->row_stride, w->expert_stride} : Operand{nullptr, 0, 0}; }
bool aligned_out(const void* p, int type) { return rows::address_bits(p) % rows::type_bytes(type) == 0; }
}  // namespace

extern "C" int hb_expert_any_grid(const hb_expert_shape* s, int weights) {
    return s && (s->type == HB_F32 || is_few(s->type, s->rows, s->experts, s->hidden, s->width, weights));
}

// Up to three operands copied to rows on 16 bytes: a warp a row.
namespace hb {
namespace experts {
struct Copies {
    const uint16_t* from[3];
    uint16_t* to[3];
    int64_t row[3], group[3], to_row[3];
    int64_t rows[3], first[3];  // rows of a group; first row of the operand among all
    int width[3], pairs[3], count;  // pairs: the source's rows lie on 4 bytes
};
__global__ void __launch_bounds__(256) copy_kernel(const __grid_constant__ Copies c, int64_t total) {
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= total) return;
    int i = 0;
    while (i + 1 < c.count && r >= c.first[i + 1]) ++i;
    const int64_t at = r - c.first[i], g = at / c.rows[i];
    const uint16_t* from = c.from[i] + g * c.group[i] + (at - g * c.rows[i]) * c.row[i];
    uint16_t* to = c.to[i] + at * c.to_row[i];
    int k = threadIdx.x & 31;
    if (c.pairs[i]) {
        const int words = c.width[i] >> 1;
#pragma unroll 4
        for (; k < words; k += 32) reinterpret_cast<uint32_t*>(to)[k] = __ldcs(reinterpret_cast<const uint32_t*>(from) + k);
        k = words * 2 + (threadIdx.x & 31);  // an odd width's last
    }
#pragma unroll 4
    for (; k < c.width[i]; k += 32) to[k] = from[k];
}
}  // namespace experts
}  // namespace hb

extern "C" int hb_expert_copy(int64_t count, const void* const* from, const int64_t* groups, const int64_t* rows, const int64_t* width,
                              const int64_t* group_stride, const int64_t* row_stride, void* const* to, const int64_t* to_stride,
                              void* stream) {
    if (count < 0 || count > 3 || (count > 0 && (!from || !groups || !rows || !width || !group_stride || !row_stride || !to || !to_stride)))
        return abi_fail(HB_BAD_ARGUMENT, "hb_expert_copy: at most 3 operands, no null pointer");
    Copies c{};
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (groups[i] < 0 || rows[i] < 0 || width[i] < 1 || width[i] > INT32_MAX || to_stride[i] < width[i] ||
            (groups[i] > 0 && rows[i] > INT64_MAX / 4 / groups[i]))
            return abi_fail(HB_BAD_ARGUMENT, "hb_expert_copy: shape of an operand");
        if (groups[i] * rows[i] == 0) continue;
        if (!from[i] || !to[i] || rows::address_bits(from[i]) % 2 || rows::address_bits(to[i]) % 2)
            return abi_fail(HB_BAD_ARGUMENT, "hb_expert_copy: null or misaligned pointer");
        const int at = c.count++;
        c.from[at] = static_cast<const uint16_t*>(from[i]);
        c.to[at] = static_cast<uint16_t*>(to[i]);
        c.row[at] = row_stride[i];
        c.group[at] = group_stride[i];
        c.to_row[at] = to_stride[i];
        c.rows[at] = rows[i];
        c.width[at] = (int)width[i];
        c.pairs[at] = (rows::address_bits(from[i]) | rows::address_bits(to[i]) |
                       (uint64_t)(row_stride[i] | group_stride[i] | to_stride[i]) * 2) % 4 == 0;
        c.first[at] = total;
        total += groups[i] * rows[i];
    }
    if (total == 0) return HB_OK;
    if ((total + 7) / 8 > INT32_MAX) return abi_fail(HB_BAD_ARGUMENT, "hb_expert_copy: too many rows");
    copy_kernel<<<(unsigned)((total + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(c, total);
    count_launches(1);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("hb_expert_copy: ") + cudaGetErrorString(e));
}

extern "C" int hb_expert_product(const hb_expert_shape* s, const void* x, int64_t x_stride, const int32_t* offsets,
                                 const hb_expert_weight* weight, void* out, void* stream) {
    const char* what = "hb_expert_product";
    if (const int rc = check(s, offsets, what)) return rc;
    if (s->rows == 0) return HB_OK;
    const bool grid = !hb_expert_any_grid(s, 1);
    Job j = job_of(s, offsets, kProduct, s->hidden, s->width);
    j.a[0] = rows_of(x, x_stride);
    j.b[0] = weight_of(weight);
    if (!fits(j.a[0], s->type, s->width, s->rows, false, 1, grid) || !fits(j.b[0], s->type, s->width, s->hidden, true, s->experts, grid) ||
        !out || !aligned_out(out, s->type))
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": " + kOperand);
    j.a[0] = tidy(j.a[0], s->width, s->rows, 1);
    j.b[0] = tidy(j.b[0], s->width, s->hidden, s->experts);
    j.out[0] = out;
    return run(j, static_cast<cudaStream_t>(stream));
}

extern "C" int hb_expert_gated(const hb_expert_shape* s, const void* x, int64_t x_stride, const int32_t* offsets,
                               const hb_expert_weight* gate, const hb_expert_weight* up, void* out, void* stream) {
    const char* what = "hb_expert_gated";
    if (const int rc = check(s, offsets, what)) return rc;
    if (s->rows == 0) return HB_OK;
    const bool grid = !hb_expert_any_grid(s, 2);
    Job j = job_of(s, offsets, kGated, s->hidden, s->width);
    j.a[0] = rows_of(x, x_stride);
    j.b[0] = weight_of(gate);
    j.b[1] = weight_of(up);
    if (!fits(j.a[0], s->type, s->width, s->rows, false, 1, grid) || !fits(j.b[0], s->type, s->width, s->hidden, true, s->experts, grid) ||
        !fits(j.b[1], s->type, s->width, s->hidden, true, s->experts, grid) || !out || !aligned_out(out, s->type))
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": " + kOperand);
    j.a[0] = tidy(j.a[0], s->width, s->rows, 1);
    for (Operand& b : j.b) b = tidy(b, s->width, s->hidden, s->experts);
    j.out[0] = out;
    return run(j, static_cast<cudaStream_t>(stream));
}

namespace {
int bad_workspace(const void* ws, size_t bytes, size_t need, const char* what) {
    if (need == 0) return HB_OK;
    if (!ws || rows::address_bits(ws) % 256)
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": the workspace must be 256-byte aligned");
    return bytes < need ? abi_fail(HB_WORKSPACE, std::string(what) + ": workspace smaller than its query says") : HB_OK;
}
// The gradients of weights without rows.
int zero_weights(const hb_expert_shape* s, void* w, cudaStream_t st, const char* what) {
    if (!w) return HB_OK;
    const cudaError_t e = cudaMemsetAsync(w, 0, (size_t)s->experts * s->hidden * s->width * rows::type_bytes(s->type), st);
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
}
// dW of one or two products over the same x.
Job weights_job(const hb_expert_shape* s, const int32_t* offsets, int segments) {
    Job j = job_of(s, offsets, kWeights, s->hidden, s->width);
    j.out_row = s->width;
    j.segments = segments;
    j.splits = splits_of(j);
    return j;
}
bool valid(const hb_expert_shape* s) {
    return s && rows::valid_type(s->type) && s->rows >= 0 && s->rows <= INT32_MAX - 1024 && s->hidden >= 1 && s->width >= 1 &&
           s->hidden <= kMostWidth && s->width <= kMostWidth && s->experts >= 1 && s->experts <= kMostGroups;
}
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t held_bytes(const hb_expert_shape* s) { return round256((size_t)s->rows * padded(s->hidden) * rows::type_bytes(s->type)); }
}  // namespace

extern "C" size_t hb_expert_product_grad_workspace(const hb_expert_shape* s) {
    if (!valid(s)) return 0;
    const Job j = weights_job(s, nullptr, 1);
    return partial_bytes(j, j.splits);
}

extern "C" int hb_expert_product_grad(const hb_expert_shape* s, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                      const int32_t* offsets, const hb_expert_weight* weight, void* dx, void* dweight,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "hb_expert_product_grad";
    if (const int rc = check(s, offsets, what)) return rc;
    const auto st = static_cast<cudaStream_t>(stream);
    const Operand dyo = rows_of(dy, dy_stride), xo = rows_of(x, x_stride), w = weight_of(weight);
    if ((s->rows > 0 && (!fits(dyo, s->type, s->hidden, s->rows, false, 1, true) ||
                         (dweight && !fits(xo, s->type, s->width, s->rows, false, 1, true)))) ||
        (dx && !fits(w, s->type, s->width, s->hidden, true, s->experts, true)) || !aligned_out(dx, s->type) || !aligned_out(dweight, s->type))
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": " + kOperand);
    if (s->rows == 0) return zero_weights(s, dweight, st, what);
    if (dweight)
        if (const int rc = bad_workspace(workspace, workspace_bytes, hb_expert_product_grad_workspace(s), what)) return rc;
    if (dx) {
        Job j = job_of(s, offsets, kBack, s->width, s->hidden);
        j.a[0] = tidy(dyo, s->hidden, s->rows, 1);
        j.b[0] = tidy(w, s->width, s->hidden, s->experts);
        j.out[0] = dx;
        if (const int rc = run(j, st)) return rc;
    }
    if (!dweight) return HB_OK;
    Job j = weights_job(s, offsets, 1);
    j.a[0] = tidy(dyo, s->hidden, s->rows, 1);
    j.b[0] = tidy(xo, s->width, s->rows, 1);
    j.out[0] = dweight;
    j.partial = static_cast<float*>(workspace);
    return run(j, st);
}

extern "C" size_t hb_expert_gated_grad_workspace(const hb_expert_shape* s) {
    if (!valid(s)) return 0;
    size_t most = 0;  // one gradient alone may be cut into more parts than both
    for (int segments : {1, 2}) {
        const Job j = weights_job(s, nullptr, segments);
        most = std::max(most, partial_bytes(j, j.splits));
    }
    return 2 * held_bytes(s) + most;
}

extern "C" int hb_expert_gated_grad(const hb_expert_shape* s, const void* dh, int64_t dh_stride, const void* x, int64_t x_stride,
                                    const int32_t* offsets, const hb_expert_weight* gate, const hb_expert_weight* up, void* dx,
                                    void* dgate, void* dup, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "hb_expert_gated_grad";
    if (const int rc = check(s, offsets, what)) return rc;
    const auto st = static_cast<cudaStream_t>(stream);
    const Operand dho = rows_of(dh, dh_stride), xo = rows_of(x, x_stride), g = weight_of(gate), u = weight_of(up);
    if ((s->rows > 0 && (!fits(dho, s->type, s->hidden, s->rows, false, 1, false) || !fits(xo, s->type, s->width, s->rows, false, 1, true))) ||
        !fits(g, s->type, s->width, s->hidden, true, s->experts, true) || !fits(u, s->type, s->width, s->hidden, true, s->experts, true) ||
        !aligned_out(dx, s->type) || !aligned_out(dgate, s->type) || !aligned_out(dup, s->type))
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": " + kOperand);
    if (s->rows == 0) {
        if (const int rc = zero_weights(s, dgate, st, what)) return rc;
        return zero_weights(s, dup, st, what);
    }
    if (const int rc = bad_workspace(workspace, workspace_bytes, hb_expert_gated_grad_workspace(s), what)) return rc;
    const int64_t held = padded(s->hidden);
    char* const ws = static_cast<char*>(workspace);
    void* const part[2] = {ws, ws + held_bytes(s)};
    Job j = job_of(s, offsets, kGatedGrad, s->hidden, s->width);
    j.a[0] = tidy(xo, s->width, s->rows, 1);
    j.b[0] = tidy(g, s->width, s->hidden, s->experts);
    j.b[1] = tidy(u, s->width, s->hidden, s->experts);
    j.dh = dho;
    j.out[0] = part[0];
    j.out[1] = part[1];
    j.out_row = held;
    if (const int rc = run(j, st)) return rc;
    if (dx) {
        Job back = job_of(s, offsets, kBack, s->width, s->hidden);
        back.a[0] = {part[0], held, 0};
        back.a[1] = {part[1], held, 0};
        back.b[0] = j.b[0];
        back.b[1] = j.b[1];
        back.segments = 2;
        back.out[0] = dx;
        if (const int rc = run(back, st)) return rc;
    }
    if (!dgate && !dup) return HB_OK;
    Job w = weights_job(s, offsets, (dgate ? 1 : 0) + (dup ? 1 : 0));
    for (int i = 0, at = 0; i < 2; ++i) {
        if (!(i ? dup : dgate)) continue;
        w.a[at] = {part[i], held, 0};
        w.out[at++] = i ? dup : dgate;
    }
    w.b[0] = j.a[0];
    w.partial = reinterpret_cast<float*>(ws + 2 * held_bytes(s));
    return run(w, st);
}
