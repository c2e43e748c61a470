// Stable counting sort of entries by expert (or by row of a table).
//
// Least significant digit first, digits of up to 11 bits, so one pass for up to
// 2047 bins and two for up to 4 million.  A pass counts each tile's digits, scans
// the counts over the tiles of a digit (a warp a digit), and places the entries:
// a warp ranks 32 entries at a time with a match over its lanes on top of its own
// shared-memory counters, so equal digits keep their order and nothing depends on
// the order of atomics.  Up to 4096 entries sort in one block with the entries in
// shared memory: one launch, which is what counts for single tokens.
#include <string>

#include "../../include/hello_b200.h"
#include "index_sort.cuh"
#include "internal.h"

namespace hb {
namespace isort {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kSmallRounds = 8, kSmallMost = kThreads * kSmallRounds;
constexpr int kMaxDigitBits = 11;

// The keys of a pass: the caller's index (first pass) or the keys of the pass before.
struct Source {
    const void* data;
    int kind;  // 4: int32 index, 8: int64 index, 0: uint32 keys
    uint32_t bins;
    __device__ __forceinline__ uint32_t key(int64_t i) const {
        if (kind == 0) return static_cast<const uint32_t*>(data)[i];
        const int64_t v = kind == 8 ? static_cast<const int64_t*>(data)[i] : (int64_t)static_cast<const int32_t*>(data)[i];
        return v >= 0 && v < (int64_t)bins ? (uint32_t)v : bins;
    }
};

// Rank of every lane's digit among the equal digits its warp has seen, in order.
__device__ __forceinline__ uint32_t warp_rank(uint16_t* counts, uint32_t digit, bool valid, uint32_t none) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t same = __match_any_sync(0xffffffffu, valid ? digit : none);
    const uint32_t before = valid ? counts[digit] : 0;
    __syncwarp();
    if (valid && (same >> lane) == 1u) counts[digit] = (uint16_t)(before + __popc(same));
    __syncwarp();
    return before + __popc(same & ((1u << lane) - 1u));
}

// counts[warp][digit] -> digits before this warp's in the block; total[digit] the block's.
__device__ __forceinline__ void scan_warps(uint16_t* counts, uint32_t* total, int digits) {
    for (int d = threadIdx.x; d < digits; d += kThreads) {
        uint32_t sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t c = counts[w * digits + d];
            counts[w * digits + d] = (uint16_t)sum;
            sum += c;
        }
        total[d] = sum;
    }
}

// Exclusive scan of v[0..digits) in place by the whole block.
__device__ __forceinline__ void block_scan(uint32_t* v, int digits) {
    __shared__ uint32_t sums[kWarps];
    const int per = (digits + kThreads - 1) / kThreads;
    const int lo = min(digits, (int)threadIdx.x * per), hi = min(digits, lo + per);
    uint32_t mine = 0;
    for (int d = lo; d < hi; ++d) mine += v[d];
    uint32_t incl = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, incl, s);
        if ((threadIdx.x & 31) >= s) incl += o;
    }
    if ((threadIdx.x & 31) == 31) sums[threadIdx.x >> 5] = incl;
    __syncthreads();
    uint32_t base = incl - mine;
    for (int w = 0; w < (int)(threadIdx.x >> 5); ++w) base += sums[w];
    for (int d = lo; d < hi; ++d) {
        const uint32_t c = v[d];
        v[d] = base;
        base += c;
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads) sort_small(Source src, int n, int passes, int digit_bits, int digits,
                                                       int32_t* __restrict__ order, int32_t* __restrict__ position,
                                                       uint32_t* __restrict__ keys_out, int32_t* __restrict__ offsets) {
    extern __shared__ uint32_t smem[];
    uint32_t* key_at = smem;                              // kSmallMost
    uint16_t* val_at = reinterpret_cast<uint16_t*>(key_at + (passes > 1 ? kSmallMost : 0));
    uint32_t* total = smem + (passes > 1 ? kSmallMost + kSmallMost / 2 : 0);  // digits
    uint16_t* counts = reinterpret_cast<uint16_t*>(total + digits);           // kWarps x digits
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rounds = (n + kThreads - 1) / kThreads;
    const int first = warp * 32 * rounds + lane;
    uint32_t key[kSmallRounds], val[kSmallRounds], rank[kSmallRounds];
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
        const int i = first + r * 32;
        if (r < rounds && i < n) key[r] = src.key(i);
        val[r] = i;
    }
    const uint32_t mask = (1u << digit_bits) - 1u;
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * digit_bits;
        for (int i = threadIdx.x; i < kWarps * digits; i += kThreads) counts[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSmallRounds; ++r)
            if (r < rounds)
                rank[r] = warp_rank(counts + warp * digits, (key[r] >> shift) & mask, first + r * 32 < n, digits);
        __syncthreads();
        scan_warps(counts, total, digits);
        __syncthreads();
        block_scan(total, digits);
        const bool last = pass + 1 == passes;
#pragma unroll
        for (int r = 0; r < kSmallRounds; ++r) {
            if (r < rounds && first + r * 32 < n) {
                const uint32_t d = (key[r] >> shift) & mask;
                const uint32_t p = total[d] + counts[warp * digits + d] + rank[r];
                if (last) {
                    if (order) order[p] = (int32_t)val[r];
                    if (position) position[val[r]] = (int32_t)p;
                    if (keys_out) keys_out[p] = key[r];
                } else {
                    key_at[p] = key[r];
                    val_at[p] = (uint16_t)val[r];
                }
            }
        }
        if (!last) {
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kSmallRounds; ++r) {
                const int i = first + r * 32;
                if (r < rounds && i < n) {
                    key[r] = key_at[i];
                    val[r] = val_at[i];
                }
            }
        }
    }
    if (offsets && passes == 1)
        for (int d = threadIdx.x; d < digits; d += kThreads) offsets[d] = (int32_t)total[d];
}

template <int ROUNDS>
__global__ void __launch_bounds__(kThreads) tile_counts(Source src, int64_t n, int shift, uint32_t mask, int digits,
                                                        int tiles, uint32_t* __restrict__ counts) {
    extern __shared__ uint32_t smem[];
    for (int d = threadIdx.x; d < digits; d += kThreads) smem[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * (kThreads * ROUNDS);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = base + r * kThreads + threadIdx.x;
        if (i < n) atomicAdd(&smem[(src.key(i) >> shift) & mask], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kThreads) counts[(int64_t)d * tiles + blockIdx.x] = smem[d];
}

// A warp a digit: its counts become exclusive sums over the tiles, its total goes to totals.
__global__ void __launch_bounds__(256) scan_tiles(uint32_t* __restrict__ counts, int tiles, int digits,
                                                  uint32_t* __restrict__ totals) {
    const int d = (blockIdx.x * 256 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    if (d >= digits) return;
    uint32_t* row = counts + (int64_t)d * tiles;
    uint32_t run = 0;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        const int t = t0 + lane;
        const uint32_t c = t < tiles ? row[t] : 0;
        uint32_t incl = c;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const uint32_t o = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += o;
        }
        if (t < tiles) row[t] = run + incl - c;
        run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) totals[d] = run;
}

template <int ROUNDS>
__global__ void __launch_bounds__(kThreads) tile_place(Source src, const int32_t* __restrict__ vals, int64_t n, int shift,
                                                       uint32_t mask, int digits, int tiles,
                                                       const uint32_t* __restrict__ counts,
                                                       const uint32_t* __restrict__ totals, int32_t* __restrict__ order,
                                                       int32_t* __restrict__ position, uint32_t* __restrict__ keys_out,
                                                       int32_t* __restrict__ offsets) {
    extern __shared__ uint32_t smem[];
    uint32_t* base = smem;                                            // digits
    uint32_t* total = base + digits;                                  // digits
    uint16_t* mine = reinterpret_cast<uint16_t*>(total + digits);     // kWarps x digits
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * (kThreads * ROUNDS) + warp * (32 * ROUNDS) + lane;
    uint32_t key[ROUNDS], rank[ROUNDS];
    int32_t val[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = first + r * 32;
        key[r] = i < n ? src.key(i) : 0;
        val[r] = i < n ? (vals ? vals[i] : (int32_t)i) : 0;
    }
    for (int d = threadIdx.x; d < digits; d += kThreads) base[d] = totals[d];
    for (int i = threadIdx.x; i < kWarps * digits; i += kThreads) mine[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        rank[r] = warp_rank(mine + warp * digits, (key[r] >> shift) & mask, first + r * 32 < n, digits);
    block_scan(base, digits);
    if (offsets && blockIdx.x == 0)
        for (int d = threadIdx.x; d < digits; d += kThreads) offsets[d] = (int32_t)base[d];
    scan_warps(mine, total, digits);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        if (first + r * 32 >= n) continue;
        const uint32_t d = (key[r] >> shift) & mask;
        const uint32_t p = base[d] + counts[(int64_t)d * tiles + blockIdx.x] + mine[warp * digits + d] + rank[r];
        if (order) order[p] = val[r];
        if (position) position[val[r]] = (int32_t)p;
        if (keys_out) keys_out[p] = key[r];
    }
}

// offsets[b] = first place whose key is not below b.
__global__ void __launch_bounds__(256) find_offsets(const uint32_t* __restrict__ keys, int64_t n, int64_t bins,
                                                    int32_t* __restrict__ offsets) {
    const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (b > bins) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < (uint32_t)b) lo = mid + 1;
        else hi = mid;
    }
    offsets[b] = (int32_t)lo;
}

struct Plan {
    int passes, digit_bits, digits, rounds, tiles;
};

// One pass over bins + 1 digits when they fit, else equal digits of at most 11 bits.  Tiles of 1024
// entries keep all SMs busy up to half a million entries, tiles of 4096 keep the counts short above.
inline Plan plan_of(int64_t n, int64_t bins) {
    Plan p{};
    int bits = 1;
    while (bits < 32 && (bins >> bits) != 0) ++bits;
    p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.digit_bits = (bits + p.passes - 1) / p.passes;
    p.digits = p.passes == 1 ? (int)(bins + 1) : 1 << p.digit_bits;
    p.rounds = n > (1 << 19) ? 8 : 2;
    const int64_t tile = (int64_t)kThreads * p.rounds;
    p.tiles = (int)((n + tile - 1) / tile);
    return p;
}

// counts and totals of a pass, the keys and entries between passes, and the last
// pass's keys (searched for the offsets when the caller takes no keys).
struct Layout {
    uint32_t *counts, *totals, *keys[2], *sorted;
    int32_t* vals[2];
    size_t bytes;
};
inline Layout layout(void* ws, int64_t n, const Plan& p) {
    Layout l{};
    char* base = static_cast<char*>(ws);
    auto take = [&](size_t bytes) {
        char* r = base + l.bytes;
        l.bytes += (bytes + 255) / 256 * 256;
        return r;
    };
    if (n > kSmallMost) {
        l.counts = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t) * (size_t)p.digits * p.tiles));
        l.totals = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t) * p.digits));
        for (int i = 0; i < 2 && i + 1 < p.passes; ++i) {
            l.keys[i] = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t) * n));
            l.vals[i] = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * n));
        }
    }
    if (p.passes > 1) l.sorted = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t) * n));
    return l;
}

inline size_t small_smem(const Plan& p) {
    return (p.passes > 1 ? (size_t)kSmallMost * 6 : 0) + (size_t)p.digits * (4 + 2 * kWarps);
}
inline size_t place_smem(const Plan& p) { return (size_t)p.digits * (8 + 2 * kWarps); }

// Dynamic shared memory above 48 KB has to be allowed once per kernel.
template <typename K>
inline cudaError_t allow(K* kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return cudaSuccess;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <int ROUNDS>
cudaError_t sort_tiles(const Source& input, int64_t n, const Plan& p, const Layout& l, int32_t* order, int32_t* position,
                       uint32_t* keys, int32_t* offsets, cudaStream_t st) {
    cudaError_t e = allow(tile_place<ROUNDS>, place_smem(p));
    if (e != cudaSuccess) return e;
    const uint32_t mask = (1u << p.digit_bits) - 1u;
    Source src = input;
    const int32_t* vals = nullptr;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.digit_bits;
        const bool last = pass + 1 == p.passes;
        uint32_t* to_keys = last ? keys : l.keys[pass & 1];
        int32_t* to_vals = last ? order : l.vals[pass & 1];
        tile_counts<ROUNDS><<<p.tiles, kThreads, sizeof(uint32_t) * p.digits, st>>>(src, n, shift, mask, p.digits,
                                                                                    p.tiles, l.counts);
        scan_tiles<<<(p.digits + 7) / 8, 256, 0, st>>>(l.counts, p.tiles, p.digits, l.totals);
        tile_place<ROUNDS><<<p.tiles, kThreads, place_smem(p), st>>>(
            src, vals, n, shift, mask, p.digits, p.tiles, l.counts, l.totals, to_vals, last ? position : nullptr, to_keys,
            last && p.passes == 1 ? offsets : nullptr);
        count_launches(3);
        src.data = to_keys;
        src.kind = 0;
        vals = to_vals;
    }
    return cudaGetLastError();
}

}  // namespace isort

size_t index_sort_bytes(int64_t n, int64_t bins) {
    if (n <= 0) return 0;
    return isort::layout(nullptr, n, isort::plan_of(n, bins)).bytes;
}

int index_sort(const void* index, int index_bytes, int64_t n, int64_t bins, int32_t* order, int32_t* position,
               uint32_t* keys, int32_t* offsets, void* ws, size_t ws_bytes, cudaStream_t st) {
    using namespace isort;
    cudaError_t e = cudaSuccess;
    if (n == 0) {
        if (offsets) e = cudaMemsetAsync(offsets, 0, sizeof(int32_t) * (bins + 1), st);
        return e == cudaSuccess ? HB_OK : abi_fail(HB_CUDA, std::string("index sort: ") + cudaGetErrorString(e));
    }
    const Plan p = plan_of(n, bins);
    const Layout l = layout(ws, n, p);
    if (l.bytes > ws_bytes || (l.bytes > 0 && !ws))
        return abi_fail(HB_WORKSPACE, "workspace too small for the index sort");
    const Source src{index, index_bytes, (uint32_t)bins};
    if (!keys && p.passes > 1 && offsets) keys = l.sorted;
    if (n <= kSmallMost) {
        e = allow(sort_small, small_smem(p));
        if (e == cudaSuccess) {
            sort_small<<<1, kThreads, small_smem(p), st>>>(src, (int)n, p.passes, p.digit_bits, p.digits, order, position,
                                                           keys, offsets);
            count_launches(1);
            e = cudaGetLastError();
        }
    } else {
        e = p.rounds == 8 ? sort_tiles<8>(src, n, p, l, order, position, keys, offsets, st)
                          : sort_tiles<2>(src, n, p, l, order, position, keys, offsets, st);
    }
    if (e == cudaSuccess && offsets && p.passes > 1) {
        find_offsets<<<(unsigned)((bins + 256) / 256), 256, 0, st>>>(keys, n, bins, offsets);
        count_launches(1);
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("index sort: ") + cudaGetErrorString(e));
}

}  // namespace hb
