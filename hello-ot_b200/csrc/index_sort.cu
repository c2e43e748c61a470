// Stable counting sort of entries by expert (or by row of a table).
//
// Least significant digit first, digits of up to 11 bits, so one pass for up to
// 2047 bins and two for up to 4 million.  A pass counts digits block by block, and
// places the entries: a warp ranks 32 entries at a time by ballots over its lanes
// on top of its own shared-memory counters, so equal digits keep their order and
// nothing depends on the order of atomics.
//
// Such a sort moves little (a megabyte at 131072 entries), so its time is launches,
// barriers and the single sector a cycle at which an SM scatters 4-byte stores.
//   up to 2048 entries   one launch of independent blocks: each ranks its 64 entries
//                        against all keys by comparing, n^2 comparisons in all, which
//                        at this size are cheaper than any barrier, and as many
//                        offsets; no passes, whatever the number of bins
//   up to 32768          one launch of one cluster of up to 16 blocks: the entries
//                        stay in the blocks' shared memory over all passes, the
//                        blocks read each other's counts and write each other's
//                        entries there, and the hardware's cluster barrier stands
//                        between the steps
//   up to 524288         tiles over all SMs, a launch for the first pass's counts
//                        and one a pass: a block adds up the counts of all tiles
//                        itself, and counts the next pass's digits as it places; the
//                        launches overlap (the first pass ranks while it is counted)
//   above                tiles of 4096 and three launches a pass, the counts scanned
//                        over the tiles by a launch of their own
//
// Measured on a B200 (us): 2 entries 1.8, 3111 by 37 experts 5.1, 131072 by 64 7.6, 262144
// by 1024 14.5, 524288 by 128 12.9; 131072 ids by 65536 rows in two passes 20.  What is left
// is latency: a launch, a barrier or an L2 access for every step of a pass.
#include <string>

#include <cooperative_groups.h>

#include "../../include/hello_b200.h"
#include "index_sort.cuh"
#include "internal.h"

namespace hb {
namespace isort {

constexpr int kThreads = 1024, kWarps = kThreads / 32;     // a tile's block
constexpr int kBlock = 1024, kBlockWarps = kBlock / 32;     // a cluster's block
constexpr int kRounds = 2;                                  // entries a thread of a cluster
constexpr int kRankMost = 2048, kRankThreads = 512;         // sort by comparing
constexpr int kRankSlices = 8, kRankQueries = kRankThreads / kRankSlices;
// Most bins whose offsets it finds; above, they are searched in the sorted pairs.  Found / searched (us): 1000 entries by
// 4000 bins 3.5 / 6.6, 2000 by 4000 4.7 / 8.1, by 16000 7.0 / 8.2, by 32000 12.0 / 8.2.
constexpr int64_t kRankBins = 4096;
constexpr int kMostClusters = 16;
constexpr int64_t kClusterMost = (int64_t)kMostClusters * kBlock * kRounds;
constexpr int kMaxDigitBits = 11;
constexpr int kMostTiles = 128;                             // that every block adds up itself

// What a pass sorts: the caller's index (first pass), or the (key, entry) pairs of the pass before.
struct Source {
    const void* data;
    int kind;  // 4: int32 index, 8: int64 index, 0: pairs
    uint32_t bins;
    __device__ __forceinline__ uint2 entry(int64_t i) const {
        if (kind == 0) return static_cast<const uint2*>(data)[i];
        const int64_t v = kind == 8 ? static_cast<const int64_t*>(data)[i] : (int64_t)static_cast<const int32_t*>(data)[i];
        return make_uint2(v >= 0 && v < (int64_t)bins ? (uint32_t)v : bins, (uint32_t)i);
    }
};

// Places of the entries, and the offsets, each a count of the keys below: of key k at entry i the keys <= k before
// i and those < k after it, of offset b the keys < b.  64 queries a block, 8 threads a query, each over an eighth of
// the keys in shared memory, where a warp reads the same 16 bytes in all its lanes.
__global__ void __launch_bounds__(kRankThreads) sort_rank(Source src, int n, int entry_blocks, int32_t* __restrict__ order,
                                                          int32_t* __restrict__ position, uint2* __restrict__ pairs,
                                                          int32_t* __restrict__ offsets, int bins,
                                                          uint32_t* __restrict__ zero, int64_t zeros) {
    __shared__ __align__(16) uint32_t keys[kRankMost];
    __shared__ uint32_t parts[kRankSlices][kRankQueries];
    allow_next();
    for (int64_t i = (int64_t)blockIdx.x * kRankThreads + threadIdx.x; i < zeros; i += (int64_t)gridDim.x * kRankThreads)
        zero[i] = 0;
    const int slice_keys = (n + kRankSlices * 4 - 1) / (kRankSlices * 4) * 4;  // whole vectors
    uint32_t own[kRankMost / kRankThreads];  // all loads before the first store
#pragma unroll
    for (int r = 0; r < kRankMost / kRankThreads; ++r) {
        const int i = r * kRankThreads + threadIdx.x;
        own[r] = i < n ? src.entry(i).x : 0xffffffffu;
    }
#pragma unroll
    for (int r = 0; r < kRankMost / kRankThreads; ++r) {
        const int i = r * kRankThreads + threadIdx.x;
        if (i < slice_keys * kRankSlices) keys[i] = own[r];
    }
    __syncthreads();
    const int query = threadIdx.x % kRankQueries, slice = threadIdx.x / kRankQueries;
    const bool entries = (int)blockIdx.x < entry_blocks;
    const int first = entries ? blockIdx.x * kRankQueries : 0;  // of the block's entries
    const int i = first + query, b = ((int)blockIdx.x - entry_blocks) * kRankQueries + query;
    const uint32_t key = entries ? (i < n ? keys[i] : 0) : (uint32_t)b;
    uint32_t count = 0;
    auto below = [&](int from, int to, uint32_t limit) {  // whole vectors
#pragma unroll 4
        for (int j = from; j < to; j += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(keys + j);
            count += (v.x < limit) + (v.y < limit) + (v.z < limit) + (v.w < limit);
        }
    };
    const int lo = slice * slice_keys, hi = lo + slice_keys;
    if (entries) {
        below(lo, min(hi, first), key + 1);
        for (int j = max(lo, first); j < min(hi, first + kRankQueries); ++j) count += keys[j] < key + (j < i);
        below(max(lo, first + kRankQueries), hi, key);
    } else {
        below(lo, hi, key);
    }
    parts[slice][query] = count;
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int s = 1; s < kRankSlices; ++s) count += parts[s][query];
    if (!entries) {
        if (b <= bins) offsets[b] = (int32_t)count;
    } else if (i < n) {
        if (order) order[count] = i;
        if (position) position[i] = (int32_t)count;
        if (pairs) pairs[count] = make_uint2(key, (uint32_t)i);
    }
}

// The lanes whose digit equals this lane's, from a ballot a bit of it.
__device__ __forceinline__ uint32_t equal_lanes(uint32_t digit, bool valid, int bits) {
    uint32_t same = __ballot_sync(0xffffffffu, valid);
#pragma unroll 4
    for (int b = 0; b < bits; ++b) {
        const uint32_t set = __ballot_sync(0xffffffffu, (digit >> b) & 1u);
        same &= (digit >> b) & 1u ? set : ~set;
    }
    return same;
}
// Ranks of a thread's digits among the equal ones that its warp has seen, in order.  left: entries from this
// lane's first to the last.
template <int ROUNDS, typename D>
__device__ __forceinline__ void warp_ranks(uint16_t* counts, D&& digit, int rounds, int64_t left, int bits,
                                           uint32_t (&rank)[ROUNDS]) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (r < rounds) rank[r] = equal_lanes(digit(r), r * 32 < left, bits);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        if (r >= rounds) break;
        const uint32_t same = rank[r], d = digit(r);
        const bool valid = r * 32 < left;
        const uint32_t before = valid ? counts[d] : 0;
        __syncwarp();
        if (valid && (same >> lane) == 1u) counts[d] = (uint16_t)(before + __popc(same));
        __syncwarp();
        rank[r] = before + __popc(same & ((1u << lane) - 1u));
    }
}

// counts[warp][digit] -> digits before this warp's in the block; total[digit] the block's.
template <int WARPS>
__device__ __forceinline__ void scan_warps(uint16_t* counts, uint32_t* total, int digits) {
    for (int d = threadIdx.x; d < digits; d += WARPS * 32) {
        constexpr int B = 8;  // loads before stores
        uint32_t sum = 0;
#pragma unroll
        for (int w0 = 0; w0 < WARPS; w0 += B) {
            uint32_t c[B];
#pragma unroll
            for (int w = 0; w < B; ++w) c[w] = counts[(w0 + w) * digits + d];
#pragma unroll
            for (int w = 0; w < B; ++w) {
                counts[(w0 + w) * digits + d] = (uint16_t)sum;
                sum += c[w];
            }
        }
        total[d] = sum;
    }
}

// Exclusive scan of v[0..digits) in place by the whole block.
template <int WARPS>
__device__ __forceinline__ void block_scan(uint32_t* v, int digits) {
    __shared__ uint32_t sums[WARPS];
    const int per = (digits + WARPS * 32 - 1) / (WARPS * 32);
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
    // every warp adds up the warps before it: lane w has warp w's sum
    uint32_t base = (threadIdx.x & 31) < min((int)(threadIdx.x >> 5), WARPS) ? sums[threadIdx.x & 31] : 0;
    base = __reduce_add_sync(0xffffffffu, base) + incl - mine;
    for (int d = lo; d < hi; ++d) {
        const uint32_t c = v[d];
        v[d] = base;
        base += c;
    }
    __syncthreads();
}

// All of a sort in one cluster.  Block b holds entries b * rounds * 1024 and on; a thread of warp w its
// entries w * rounds * 32 + r * 32 + lane, so the order of (block, warp, round, lane) is the entries'.
__global__ void __launch_bounds__(kBlock, 1) sort_cluster(Source src, int n, int rounds, int passes, int digit_bits,
                                                          int digits, int32_t* __restrict__ order,
                                                          int32_t* __restrict__ position, uint2* __restrict__ pairs,
                                                          int32_t* __restrict__ offsets, uint32_t* __restrict__ zero,
                                                          int64_t zeros) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint32_t smem[];
    allow_next();
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
    const int mine = rounds * kBlock;                      // entries a block
    uint32_t* total = smem;                                // digits: this block's counts, read by the others
    uint32_t* base = total + digits;                       // digits: first place of this block's
    uint32_t* before = base + digits;                      // digits: those of the blocks before
    uint2* entry_at = reinterpret_cast<uint2*>(smem + (3 * digits + 1) / 2 * 2);  // (key, entry) between passes
    uint16_t* counts = reinterpret_cast<uint16_t*>(entry_at + (passes > 1 ? mine : 0));  // kBlockWarps x digits
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int within = warp * 32 * rounds + lane;
    const int first = me * mine + within;
    for (int64_t i = (int64_t)me * kBlock + threadIdx.x; i < zeros; i += blocks * kBlock) zero[i] = 0;
    uint2 entry[kRounds];  // (key, entry)
    uint32_t rank[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
        if (r < rounds && first + r * 32 < n) entry[r] = src.entry(first + r * 32);
        else entry[r] = make_uint2(0, 0);
    const uint32_t mask = (1u << digit_bits) - 1u;
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * digit_bits;
        const bool last = pass + 1 == passes;
        for (int i = threadIdx.x; i < kBlockWarps * digits / 2; i += kBlock) reinterpret_cast<uint32_t*>(counts)[i] = 0;
        __syncthreads();
        auto digit = [&](int r) { return (entry[r].x >> shift) & mask; };
        warp_ranks(counts + warp * digits, digit, rounds, n - first, digit_bits, rank);
        __syncthreads();
        scan_warps<kBlockWarps>(counts, total, digits);
        cluster.sync();
        for (int d = threadIdx.x; d < digits; d += kBlock) {
            uint32_t all = 0, lower = 0;
#pragma unroll
            for (int b = 0; b < kMostClusters; ++b) {
                const uint32_t c = b < blocks ? *cluster.map_shared_rank(total + d, b) : 0;
                if (b < me) lower += c;
                all += c;
            }
            base[d] = all;
            before[d] = lower;
        }
        __syncthreads();
        block_scan<kBlockWarps>(base, digits);
        if (offsets && passes == 1 && me == 0)
            for (int d = threadIdx.x; d < digits; d += kBlock) offsets[d] = (int32_t)base[d];
        // all counts are read: a block may leave, or count again
        if (last) cluster.sync();
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            if (r < rounds && first + r * 32 < n) {
                const uint32_t d = digit(r);
                const uint32_t p = base[d] + before[d] + counts[warp * digits + d] + rank[r];
                if (last) {
                    if (order) order[p] = (int32_t)entry[r].y;
                    if (position) position[entry[r].y] = (int32_t)p;
                    if (pairs) pairs[p] = entry[r];
                } else {
                    const uint32_t to = p / (uint32_t)mine, at = p - to * (uint32_t)mine;
                    *cluster.map_shared_rank(entry_at + at, to) = entry[r];
                }
            }
        }
        if (!last) {
            cluster.sync();
#pragma unroll
            for (int r = 0; r < kRounds; ++r)
                if (r < rounds && first + r * 32 < n) entry[r] = entry_at[within + r * 32];
        }
    }
}

// Words of a tile's packed counts: 16 bits a digit, in whole 16-byte vectors.
__host__ __device__ inline int words_of(int digits) { return (digits + 7) / 8 * 4; }

// A tile's digits: counts[digit][tile] for scan_tiles (SCANNED), else packed, counts[tile][words_of].  Clears
// `next` and `zero` too.
template <int ROUNDS, bool SCANNED>
__global__ void __launch_bounds__(kThreads) tile_counts(Source src, int64_t n, int shift, uint32_t mask, int digits,
                                                        int tiles, uint32_t* __restrict__ counts,
                                                        uint32_t* __restrict__ next, int64_t nexts,
                                                        uint32_t* __restrict__ zero, int64_t zeros) {
    extern __shared__ uint32_t smem[];
    allow_next();
    const int64_t thread = (int64_t)blockIdx.x * kThreads + threadIdx.x, threads = (int64_t)tiles * kThreads;
    for (int64_t i = thread; i < nexts; i += threads) next[i] = 0;
    for (int64_t i = thread; i < zeros; i += threads) zero[i] = 0;
    const int words = SCANNED ? digits : words_of(digits);
    for (int d = threadIdx.x; d < words; d += kThreads) smem[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * (kThreads * ROUNDS);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t i = base + r * kThreads + threadIdx.x;
        if (i < n) {
            const uint32_t d = (src.entry(i).x >> shift) & mask;
            atomicAdd(&smem[SCANNED ? d : d / 2], SCANNED ? 1u : 1u << (d % 2 * 16));
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < words; d += kThreads)
        counts[SCANNED ? (int64_t)d * tiles + blockIdx.x : (int64_t)blockIdx.x * words + d] = smem[d];
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

// Places a tile's entries.  SCANNED: counts and totals as scan_tiles leaves them; else the tiles' packed counts,
// and the digits of the next pass are counted into `next` (cleared before), tile by tile of where entries go.
// FIRST: the first pass, whose keys are the caller's: the block ranks them while the counts are still being made.
// counts and totals are written while this kernel may already run, so they are not declared unaliased: the compiler
// could read them before after_last(), or through the read-only path.
template <int ROUNDS, bool SCANNED, bool FIRST>
__global__ void __launch_bounds__(kThreads) tile_place(Source src, int64_t n, int shift, uint32_t mask, int digits,
                                                       int tiles, const uint32_t* counts, const uint32_t* totals,
                                                       uint32_t* __restrict__ next,
                                                       int next_shift, int32_t* __restrict__ order,
                                                       int32_t* __restrict__ position, uint2* __restrict__ pairs,
                                                       int32_t* __restrict__ offsets) {
    extern __shared__ uint32_t smem[];
    uint32_t* base = smem;                                            // digits: of all entries
    uint32_t* before = base + digits;                                 // digits: of the tiles before
    uint32_t* total = before + digits;                                // digits
    uint16_t* mine = reinterpret_cast<uint16_t*>(total + digits);     // kWarps x digits
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * (kThreads * ROUNDS) + warp * (32 * ROUNDS) + lane;
    uint2 entry[ROUNDS];  // (key, entry)
    uint32_t rank[ROUNDS];
    auto digit = [&](int r) { return (entry[r].x >> shift) & mask; };
    allow_next();
    for (int d = threadIdx.x; d < digits; d += kThreads) base[d] = before[d] = 0;
    for (int i = threadIdx.x; i < kWarps * digits / 2; i += kThreads) reinterpret_cast<uint32_t*>(mine)[i] = 0;
    if (!FIRST) after_last();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        entry[r] = make_uint2(0, 0);
        if (first + r * 32 < n) entry[r] = src.entry(first + r * 32);
    }
    __syncthreads();
    warp_ranks(mine + warp * digits, digit, ROUNDS, n - first, __popc(mask), rank);
    __syncthreads();
    scan_warps<kWarps>(mine, total, digits);
    if (FIRST) after_last();
    const int words = words_of(digits);
    if (SCANNED) {
        for (int d = threadIdx.x; d < digits; d += kThreads) {
            base[d] = totals[d];
            before[d] = counts[(int64_t)d * tiles + blockIdx.x];
        }
    } else {  // a vector of 8 digits a thread, as many threads a vector as there are, each every slices-th tile
        const int vectors = words / 4, slices = kThreads / vectors;
        const int v = threadIdx.x % vectors, slice = threadIdx.x / vectors;
        if (slice < slices) {
            uint32_t all[8] = {}, lower[8] = {};
#pragma unroll 4
            for (int t = slice; t < tiles; t += slices) {
                const uint4 c = reinterpret_cast<const uint4*>(counts + (int64_t)t * words)[v];
                const uint32_t w[4] = {c.x, c.y, c.z, c.w};
                const uint32_t own = t < (int)blockIdx.x ? ~0u : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    all[2 * i] += w[i] & 0xffffu, all[2 * i + 1] += w[i] >> 16;
                    lower[2 * i] += w[i] & 0xffffu & own, lower[2 * i + 1] += w[i] >> 16 & own;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (v * 8 + i < digits) {
                    atomicAdd(&base[v * 8 + i], all[i]);
                    atomicAdd(&before[v * 8 + i], lower[i]);
                }
        }
    }
    __syncthreads();
    block_scan<kWarps>(base, digits);
    if (offsets && blockIdx.x == 0)
        for (int d = threadIdx.x; d < digits; d += kThreads) offsets[d] = (int32_t)base[d];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        if (first + r * 32 >= n) continue;
        const uint32_t d = digit(r), e = FIRST ? (uint32_t)(first + r * 32) : entry[r].y;
        const uint32_t p = base[d] + before[d] + mine[warp * digits + d] + rank[r];
        if (order) order[p] = (int32_t)e;
        if (position) position[e] = (int32_t)p;
        if (pairs) pairs[p] = make_uint2(entry[r].x, e);
        if (next) {
            const uint32_t q = (entry[r].x >> next_shift) & mask;
            atomicAdd(&next[(int64_t)(p / (kThreads * ROUNDS)) * words + q / 2], 1u << (q % 2 * 16));
        }
    }
}

// offsets[b] = first place whose key is not below b.
__global__ void __launch_bounds__(256) find_offsets(const uint2* pairs, int64_t n, int64_t bins,
                                                    int32_t* __restrict__ offsets) {
    const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
    after_last();
    if (b > bins) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (pairs[mid].x < (uint32_t)b) lo = mid + 1;
        else hi = mid;
    }
    offsets[b] = (int32_t)lo;
}

struct Plan {
    int passes, digit_bits, digits, rounds, tiles;
    int cluster;  // blocks of the one-launch sort, 0: tiles
    bool rank;    // by comparing
};

// One pass over bins + 1 digits when they fit, else equal digits of at most 11 bits.
// A cluster has a block for every 1024 entries up to 16; tiles have 1024, 2048 or 4096
// entries, the least that makes at most 128 tiles, so that a block adds up their counts in a few loads a thread.
inline Plan plan_of(int64_t n, int64_t bins) {
    Plan p{};
    p.rank = n <= kRankMost;
    int bits = 1;
    while (bits < 32 && (bins >> bits) != 0) ++bits;
    p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.digit_bits = (bits + p.passes - 1) / p.passes;
    p.digits = p.passes == 1 ? (int)(bins + 1) : 1 << p.digit_bits;
    if (n <= kClusterMost) {
        p.cluster = 1;
        while (p.cluster < kMostClusters && (int64_t)p.cluster * kBlock < n) p.cluster <<= 1;
        p.rounds = (int)((n + p.cluster * kBlock - 1) / (p.cluster * kBlock));
        return p;
    }
    p.rounds = 1;
    while (p.rounds < 4 && (int64_t)p.rounds * kThreads * kMostTiles < n) p.rounds <<= 1;
    const int64_t tile = (int64_t)kThreads * p.rounds;
    p.tiles = (int)((n + tile - 1) / tile);
    return p;
}
inline bool scanned(const Plan& p) { return p.tiles > kMostTiles; }

// Counts (of a pass, or of each) and totals, the pairs between passes, and the sorted pairs (searched for the
// offsets when the caller takes none).
struct Layout {
    uint32_t *counts, *totals;
    uint2 *pairs[2], *sorted;
    size_t bytes;
};
inline Layout layout(void* ws, int64_t n, int64_t bins, const Plan& p) {
    Layout l{};
    char* base = static_cast<char*>(ws);
    auto take = [&](size_t bytes) {
        char* r = base + l.bytes;
        l.bytes += (bytes + 255) / 256 * 256;
        return r;
    };
    if (!p.cluster) {
        l.counts = reinterpret_cast<uint32_t*>(
            take(sizeof(uint32_t) * p.tiles * (scanned(p) ? (size_t)p.digits : (size_t)words_of(p.digits) * p.passes)));
        l.totals = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t) * p.digits));
        for (int i = 0; i < 2 && i + 1 < p.passes; ++i) l.pairs[i] = reinterpret_cast<uint2*>(take(sizeof(uint2) * n));
    }
    if (p.rank ? bins > kRankBins : p.passes > 1) l.sorted = reinterpret_cast<uint2*>(take(sizeof(uint2) * n));
    return l;
}

constexpr size_t cluster_smem(int digits, int passes, int rounds) {
    return (size_t)(3 * digits + 1) / 2 * 8 + (passes > 1 ? (size_t)rounds * kBlock * 8 : 0) +
           (size_t)digits * 2 * kBlockWarps;
}
constexpr size_t place_smem(int digits) { return (size_t)digits * (12 + 2 * kWarps); }

// Dynamic shared memory above 48 KB has to be allowed for the kernel, a setting that the process's calls share: always
// the most that any plan takes (plan_of: at most 2^kMaxDigitBits digits), so that no thread's call lowers another's.
constexpr size_t kClusterSmem = cluster_smem(1 << kMaxDigitBits, 2, kRounds), kPlaceSmem = place_smem(1 << kMaxDigitBits);
static_assert(kClusterSmem <= 227 * 1024 && kPlaceSmem <= 227 * 1024, "shared memory of a block");
template <typename K>
inline cudaError_t allow(K* kernel, size_t bytes, size_t most) {
    if (bytes <= 48 * 1024) return cudaSuccess;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
}

cudaError_t sort_one_launch(const Source& src, int n, const Plan& p, int32_t* order, int32_t* position, uint2* pairs,
                            int32_t* offsets, uint32_t* zero, int64_t zeros, cudaStream_t st) {
    const size_t smem = cluster_smem(p.digits, p.passes, p.rounds);
    cudaError_t e = allow(sort_cluster, smem, kClusterSmem);
    if (e == cudaSuccess && p.cluster > 8)
        e = cudaFuncSetAttribute(sort_cluster, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(p.cluster);
    config.blockDim = dim3(kBlock);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    config.attrs = &attr;
    config.numAttrs = 1;
    count_launches(1);
    return cudaLaunchKernelEx(&config, sort_cluster, src, n, p.rounds, p.passes, p.digit_bits, p.digits, order, position,
                              pairs, offsets, zero, zeros);
}

template <int ROUNDS, bool SCANNED>
cudaError_t sort_tiles(const Source& input, int64_t n, const Plan& p, const Layout& l, int32_t* order, int32_t* position,
                       uint2* pairs, int32_t* offsets, uint32_t* zero, int64_t zeros, cudaStream_t st) {
    const size_t smem = place_smem(p.digits);
    cudaError_t e = allow(tile_place<ROUNDS, SCANNED, true>, smem, kPlaceSmem);
    if (e == cudaSuccess) e = allow(tile_place<ROUNDS, SCANNED, false>, smem, kPlaceSmem);
    if (e != cudaSuccess) return e;
    const uint32_t mask = (1u << p.digit_bits) - 1u;
    const int64_t counted = (int64_t)words_of(p.digits) * p.tiles;  // words of a pass (SCANNED has one area)
    Source src = input;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.digit_bits;
        const bool last = pass + 1 == p.passes;
        uint2* to = last ? pairs : l.pairs[pass & 1];
        uint32_t* counts = l.counts + (SCANNED ? 0 : pass * counted);
        if (SCANNED || pass == 0) {
            const size_t counted_smem = sizeof(uint32_t) * (SCANNED ? p.digits : words_of(p.digits));
            tile_counts<ROUNDS, SCANNED><<<p.tiles, kThreads, counted_smem, st>>>(
                src, n, shift, mask, p.digits, p.tiles, counts, l.counts + counted,
                SCANNED ? 0 : counted * (p.passes - 1), zero, pass == 0 ? zeros : 0);
            count_launches(1);
        }
        if (SCANNED) {
            scan_tiles<<<(p.digits + 7) / 8, 256, 0, st>>>(counts, p.tiles, p.digits, l.totals);
            count_launches(1);
        }
        const auto place = pass == 0 ? tile_place<ROUNDS, SCANNED, true> : tile_place<ROUNDS, SCANNED, false>;
        e = launch_next(place, p.tiles, kThreads, smem, st, src, n, shift, mask, p.digits, p.tiles, counts,
                        l.totals, SCANNED || last ? nullptr : counts + counted, shift + p.digit_bits,
                        last ? order : nullptr, last ? position : nullptr, to,
                        last && p.passes == 1 ? offsets : nullptr);
        if (e != cudaSuccess) return e;
        count_launches(1);
        src.data = to;
        src.kind = 0;
    }
    return cudaGetLastError();
}

}  // namespace isort

size_t index_sort_bytes(int64_t n, int64_t bins) {
    if (n <= 0) return 0;
    return isort::layout(nullptr, n, bins, isort::plan_of(n, bins)).bytes;
}

int index_sort(const void* index, int index_bytes, int64_t n, int64_t bins, int32_t* order, int32_t* position,
               uint2* pairs, int32_t* offsets, void* ws, size_t ws_bytes, cudaStream_t st, uint32_t* zero,
               int64_t zeros) {
    using namespace isort;
    cudaError_t e = cudaSuccess;
    if (n == 0) {
        if (offsets) e = cudaMemsetAsync(offsets, 0, sizeof(int32_t) * (bins + 1), st);
        return e == cudaSuccess ? HB_OK : abi_fail(HB_CUDA, std::string("index sort: ") + cudaGetErrorString(e));
    }
    const Plan p = plan_of(n, bins);
    const Layout l = layout(ws, n, bins, p);
    if ((uintptr_t)ws % 256 || (uintptr_t)index % index_bytes)
        return abi_fail(HB_BAD_ARGUMENT, "index sort: misaligned index, or a workspace that is not 256-byte aligned");
    if (l.bytes > ws_bytes || (l.bytes > 0 && !ws))
        return abi_fail(HB_WORKSPACE, "workspace too small for the index sort");
    const Source src{index, index_bytes, (uint32_t)bins};
    const bool search = offsets && (p.rank ? bins > kRankBins : p.passes > 1);  // offsets by searching the sorted pairs
    if (!pairs && search) pairs = l.sorted;
    if (p.rank) {
        const int blocks = (int)((n + kRankQueries - 1) / kRankQueries);
        const int more = offsets && !search ? (int)(bins / kRankQueries + 1) : 0;
        sort_rank<<<blocks + more, kRankThreads, 0, st>>>(src, (int)n, blocks, order, position, pairs, offsets,
                                                          (int)bins, zero, zeros);
        count_launches(1);
        e = cudaGetLastError();
    } else if (p.cluster) {
        e = sort_one_launch(src, (int)n, p, order, position, pairs, offsets, zero, zeros, st);
    } else {
        auto sort = scanned(p) ? sort_tiles<4, true>
                    : p.rounds == 4 ? sort_tiles<4, false>
                    : p.rounds == 2 ? sort_tiles<2, false>
                                    : sort_tiles<1, false>;
        e = sort(src, n, p, l, order, position, pairs, offsets, zero, zeros, st);
    }
    if (e == cudaSuccess && search) {
        e = launch_next(find_offsets, dim3((unsigned)((bins + 256) / 256)), 256, 0, st, pairs, n, bins, offsets);
        count_launches(1);
    }
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("index sort: ") + cudaGetErrorString(e));
}

}  // namespace hb
