// Rows of a table by index, scaled, and the table's gradient.
//
//   lookup   y[i]  = scale * W[id_i]              (0 for an id outside the table)
//   gradient dW[v] = scale * sum over id_i = v of dy[i],   dense
//
// The lookup is a gather of whole rows: HBM-bound, a group of threads a row.
//
// The gradient sorts the tokens by row (index_sort.cu), so a row's tokens lie
// together and each dy row is read once, each dW row written once.  Rows differ
// wildly in how often they occur, so the work is cut by sorted places, not by
// rows: a group of threads sums a chunk of places in fp32 registers and writes the
// rows that begin and end inside it.  A row that crosses chunks leaves one fp32
// partial a chunk; the group that leaves the last of 16 chunks' (a counter says so,
// nobody waits) adds those up in order, and the last of these groups their sums, so
// a row that holds most of the batch is joined by many, and the result does not
// depend on the launch.
// Blocks behind the chunks write the zeros of the rows that no token names.
//
// Measured on a B200: 32768 rows of 2048 bf16 looked up in 37 us (187 MB, 5.1 TB/s); the
// gradient of 131072 tokens into 65536 x 2048 bf16 157 us, 134 of them here (806 MB, 6.0
// TB/s) and the rest the sort; 1000 tokens into 5003 x 129 f32 11 us, which is the chain of
// dependent accesses (places, rows, counter, join), not bytes.
#include <string>

#include "index_sort.cuh"
#include "internal.h"
#include "rows.cuh"

namespace hb {
namespace embedding {

using rows::Vec;

__device__ __forceinline__ int64_t load_id(const void* ids, int bytes, int64_t i) {
    return bytes == 8 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// N values of TO at an address aligned to min(16, N * sizeof(TO)).
template <typename TO, int N>
struct Values {
    static constexpr int kBytes = N * (int)sizeof(TO), kPiece = kBytes < 16 ? kBytes : 16, kPieces = kBytes / kPiece;
    using V = Vec<TO, kPiece>;
    static __device__ __forceinline__ void load(const TO* p, float (&f)[N]) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            V v;
            v.raw = *reinterpret_cast<const typename V::Raw*>(p + j * V::N);
#pragma unroll
            for (int i = 0; i < V::N; ++i) f[j * V::N + i] = rows::to_float(v.v[i]);
        }
    }
    // what other blocks have written in this launch
    static __device__ __forceinline__ void load_l2(const TO* p, float (&f)[N]) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            V v;
            v.raw = __ldcg(reinterpret_cast<const typename V::Raw*>(p + j * V::N));
#pragma unroll
            for (int i = 0; i < V::N; ++i) f[j * V::N + i] = rows::to_float(v.v[i]);
        }
    }
    static __device__ __forceinline__ void store(TO* p, const float (&f)[N]) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            V v;
#pragma unroll
            for (int i = 0; i < V::N; ++i) v.v[i] = rows::from_float<TO>(f[j * V::N + i]);
            v.store(p + j * V::N);
        }
    }
};

// A group of threads serves M rows, U column steps at a time: M * U vectors a thread in flight.
template <typename T, int VB, int M, int U>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ table, int64_t stride, int64_t rows_,
                                                     int64_t width, const void* __restrict__ ids, int id_bytes, int64_t n,
                                                     float scale, T* __restrict__ out) {
    using V = Vec<T, VB>;
    const int64_t first = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * M;
    const int64_t step = (int64_t)blockDim.x * V::N;
    int64_t id[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        id[m] = first + m < n ? load_id(ids, id_bytes, first + m) : -1;
        if (id[m] >= rows_) id[m] = -1;
    }
    for (int64_t c = threadIdx.x * V::N; c < width; c += step * U) {
        V v[M][U];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (id[m] >= 0 && c + u * step < width) v[m][u].load(table + id[m] * stride + c + u * step);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (first + m >= n || c + u * step >= width) break;
                V r;
#pragma unroll
                for (int j = 0; j < V::N; ++j)
                    r.v[j] = rows::from_float<T>(id[m] >= 0 ? scale * rows::to_float(v[m][u].v[j]) : 0.0f);
                r.store_once(out + (first + m) * width + c + u * step);
            }
    }
}

template <typename T, typename TO>
struct Grad {
    const T* dy;
    int64_t dy_stride, n, rows, width;
    float scale;
    const uint2* pairs;      // (row, token) of each sorted place; row `rows` for an id outside the table
    int chunk;               // places a group
    int64_t chunks;
    int tiles;               // column tiles
    float* partial;          // [chunks][2][width]: the row that a chunk continues, the row that it leaves open
    uint32_t* arrived;       // [chunks][3][tiles], zero: a block's partials of a row that it continues, of one that
                             // begins in it, and the sums there are of a row's blocks
    TO* out;
    int accumulate;
    int64_t sum_blocks;
    int rows_per_warp;
};

// A row is written by one group alone, so adding to what is there needs no atomics.  Atomic additions would not wait for
// the old values (92503 tokens added into 105992 x 368 f32 75 us against 99, x 369 97 against 142), but round the sum
// before they add it and, on fp32 in global memory, may flush subnormal values to zero.
template <typename T, typename TO, int N>
__device__ __forceinline__ void write_row(const Grad<T, TO>& g, uint32_t key, int64_t c, const float (&sum)[N]) {
    TO* to = g.out + (int64_t)key * g.width + c;
    float r[N];
    if (g.accumulate) {
        Values<TO, N>::load(to, r);
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = fmaf(g.scale, sum[i], r[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = g.scale * sum[i];
    }
    Values<TO, N>::store(to, r);
}

// The far chunk of a row `key` that crosses chunks: the first one of a row that chunk c continues (down), or the
// last one of a row that chunk c leaves open.  Doubling steps, then halving ones.
template <typename G>
__device__ __forceinline__ int64_t far_chunk(const G& g, uint32_t key, int64_t c, bool down) {
    const int64_t way = down ? -1 : 1;
    int64_t x = c + way, step = 1;
    auto holds = [&](int64_t chunk) {  // its last place, or its first
        return chunk >= 0 && chunk < g.chunks && g.pairs[down ? (chunk + 1) * g.chunk - 1 : chunk * g.chunk].x == key;
    };
    while (holds(x + way * step)) x += way * step, step <<= 1;
    for (; step; step >>= 1)
        if (holds(x + way * step)) x += way * step;
    return x;
}

// All threads of a group (a part of a warp, or whole warps).
__device__ __forceinline__ unsigned group_lanes() {
    const int n = blockDim.x;
    return n >= 32 ? 0xffffffffu : ((1u << n) - 1u) << ((threadIdx.y * n) & 31);
}
__device__ __forceinline__ void group_sync() {
    if (blockDim.x <= 32) __syncwarp(group_lanes());
    else asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(blockDim.x) : "memory");
}

// sum of `count` partials at part + i * step, in order
template <int N>
__device__ __forceinline__ void add_partials(const float* part, int64_t step, int count, float (&sum)[N]) {
    constexpr int U = N > 4 ? 4 : 8;
    for (int q = 0; q < count; q += U) {
        float v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q + u < count) Values<float, N>::load_l2(part + (q + u) * step, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q + u < count) {
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += v[u][i];
            }
    }
}

// Partial 1 of a row's first chunk holds what the row begins with, partial 0 of each later chunk what continues it.
// Chunks go by blocks of kJoin: whoever leaves the last partial of a block adds them up, in the place of the
// block's first one, and whoever leaves the last block's sum adds those.
constexpr int kJoin = 16;
struct Join {
    int32_t first, last, complete;  // chunks of a row; whether this group left its block's last partial
};
// How many of a row's partials a chunk's block has beside one, and their counter.
template <typename T, typename TO>
__device__ __forceinline__ uint32_t* block_counter(const Grad<T, TO>& g, int64_t first, int64_t last, int64_t chunk, int tile,
                                                   uint32_t* others) {
    const int64_t from = max(first, chunk / kJoin * kJoin), to = min(last, chunk / kJoin * kJoin + kJoin - 1);
    *others = (uint32_t)(to - from);
    return g.arrived + (from * 3 + (from == first)) * g.tiles + tile;
}
// Called by a group that left the last partial of chunk `chunk`'s block of the row.
template <typename T, typename TO, int N>
__device__ void join_row(const Grad<T, TO>& g, uint32_t key, int64_t first, int64_t last, int64_t chunk, int tile, int64_t c,
                         bool mine, int32_t* complete) {
    const int64_t from = max(first, chunk / kJoin * kJoin), to = min(last, chunk / kJoin * kJoin + kJoin - 1);
    const bool whole = first / kJoin == last / kJoin;
    float* place = g.partial + (from * 2 + (from == first)) * g.width + c;
    float sum[N];
    if (mine) {
        Values<float, N>::load_l2(place, sum);
        add_partials<N>(g.partial + (from + 1) * 2 * g.width + c, 2 * g.width, (int)(to - from), sum);
        if (whole) write_row<T, TO, N>(g, key, c, sum);
        else Values<float, N>::store(place, sum);
    }
    if (whole) return;
    __threadfence();
    group_sync();
    if (threadIdx.x == 0) {
        *complete = atomicAdd(g.arrived + (first * 3 + 2) * g.tiles + tile, 1u) == (uint32_t)(last / kJoin - first / kJoin);
        __threadfence();
    }
    group_sync();
    if (!*complete || !mine) return;
    Values<float, N>::load_l2(g.partial + (first * 2 + 1) * g.width + c, sum);
    const int64_t next = (first / kJoin + 1) * kJoin;
    add_partials<N>(g.partial + next * 2 * g.width + c, 2 * kJoin * g.width, (int)(last / kJoin - first / kJoin), sum);
    write_row<T, TO, N>(g, key, c, sum);
}

__device__ __forceinline__ void add_pair(float& a, float& b, float x, float y) {
    asm("{\n\t.reg .b64 s, v;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tadd.rn.f32x2 s, s, v;\n\t"
        "mov.b64 {%0, %1}, s;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(x), "f"(y));
}
template <typename T, int VB>
__device__ __forceinline__ void add_vector(float (&sum)[Vec<T, VB>::N], const Vec<T, VB>& v) {
    constexpr int N = Vec<T, VB>::N;
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) add_pair(sum[i], sum[i + 1], rows::to_float(v.v[i]), rows::to_float(v.v[i + 1]));
    if (N % 2) sum[N - 1] += rows::to_float(v.v[N - 1]);
}

// The rows and tokens of 8 consecutive places; the array is padded to whole groups of 8.  Plain loads: the sort may
// still be writing them when this kernel starts (after_last), which rules out the read-only path.
__device__ __forceinline__ void load8(const uint2* pairs, uint32_t (&row)[8], uint32_t (&token)[8]) {
    const uint4* p = reinterpret_cast<const uint4*>(pairs);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint4 v = p[i];
        row[2 * i] = v.x, token[2 * i] = v.y, row[2 * i + 1] = v.z, token[2 * i + 1] = v.w;
    }
}

// Sums a chunk.  Each thread has its own ring of 8 vectors in shared memory, one a sorted place, filled ahead by
// asynchronous copies: 8 rows are in flight while the sums hold few registers, and no thread waits for another.
// Vectors of 4 and 2 bytes are loaded 8 rows ahead into registers instead: they fit there, and the ring's
// instructions a row weigh more the fewer bytes a row has (92503 tokens into 105992 x 369 f32 98 us against 102,
// 40000 into 30000 x 1002 f16 60 against 65; vectors of 8 bytes 51.5 in the ring against 53.7).  The loop goes by 8
// places (chunks are multiples of 8), whose rows and tokens come in whole vectors, since its instructions are the
// next bound after the bytes.
template <typename T, typename TO, int VB>
__device__ __forceinline__ void sum_chunk(const Grad<T, TO>& g, int64_t block) {
    using V = Vec<T, VB>;
    constexpr int N = V::N, D = 8;
    __shared__ Join joins[64][2];  // a group: of the row that its chunk continues, of the row that it leaves open
    __shared__ __align__(16) typename V::Raw ring[VB >= 8 ? D * 256 : 1];
    const int tile = (int)(block % g.tiles);
    const int64_t c = ((int64_t)tile * blockDim.x + threadIdx.x) * N;
    const int64_t chunk = block / g.tiles * blockDim.y + threadIdx.y;
    if (chunk >= g.chunks) return;  // the whole group
    const bool mine = c < g.width;
    const uint32_t none = (uint32_t)g.rows;
    const int64_t p0 = chunk * g.chunk;
    const int count = (int)min((int64_t)g.chunk, g.n - p0);
    const uint32_t first_key = g.pairs[p0].x;
    if (first_key >= none) return;
    typename V::Raw* slots = ring + threadIdx.y * blockDim.x + threadIdx.x;
    const int step = blockDim.x * blockDim.y;
    const char* column = reinterpret_cast<const char*>(g.dy + (mine ? c : 0));
    const uint32_t stride = (uint32_t)(g.dy_stride * (int64_t)sizeof(T));  // bytes, below 2^32
    auto fetch = [&](int j, uint32_t token, bool there) {  // into slot j
        const char* p = column + (uint64_t)token * stride;
        if constexpr (VB >= 8) {
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(slots + j * step));
            if (there) {
                if constexpr (VB == 16)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(p) : "memory");
                else
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(p) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
    uint32_t keys[D], tokens[D], after[D];
    load8(g.pairs + p0, after, tokens);
#pragma unroll
    for (int j = 0; j < D; ++j) fetch(j, tokens[j], mine && j < count);
    // The rows that cross the chunk's ends, and their far chunks: a thread for each search, while the rows come.
    const int64_t p1 = p0 + count;
    const uint32_t last_key = g.pairs[p1 - 1].x;
    const bool continues = p0 > 0 && g.pairs[p0 - 1].x == first_key;
    const bool open = last_key < none && p1 < g.n && g.pairs[p1].x == last_key;
    const bool through = continues && open && first_key == last_key;
    int64_t far = chunk;
    if (threadIdx.x == 0 ? continues : threadIdx.x == 1 ? through : threadIdx.x == 2 && open && !through)
        far = far_chunk(g, threadIdx.x < 2 ? first_key : last_key, chunk, threadIdx.x == 0);
    uint32_t key = first_key;
    bool head = continues;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    auto flush = [&]() {
        if (mine) {
            if (head) Values<float, N>::store(g.partial + (chunk * 2) * g.width + c, sum);
            else write_row<T, TO, N>(g, key, c, sum);
        }
    };
    // short vectors: 8 rows ahead in registers
    typename V::Raw ahead[VB >= 8 ? 1 : D], raw[VB >= 8 ? 1 : D];
    auto load_ahead = [&](int i) {
#pragma unroll
        for (int j = 0; j < D; ++j)
            if (mine && i + j < count)
                ahead[j] = __ldcs(reinterpret_cast<const typename V::Raw*>(column + (uint64_t)tokens[j] * stride));
    };
    if constexpr (VB < 8) load_ahead(0);
    for (int i = 0; i < count; i += D) {
        const bool more = i + D < count;
#pragma unroll
        for (int j = 0; j < D; ++j) keys[j] = i + j < count ? after[j] : none;
        if (more) load8(g.pairs + p0 + i + D, after, tokens);
        if constexpr (VB < 8) {
#pragma unroll
            for (int j = 0; j < D; ++j) raw[j] = ahead[j];
            load_ahead(i + D);
        }
#pragma unroll
        for (int j = 0; j < D; ++j) {
            if (keys[j] != key) {
                flush();
#pragma unroll
                for (int q = 0; q < N; ++q) sum[q] = 0.0f;
                key = keys[j];
                head = false;
                if (key >= none) break;
            }
            V v;
            if constexpr (VB >= 8) {
                asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
                v.raw = slots[j * step];
            } else {
                v.raw = raw[j];
            }
            add_vector<T, VB>(sum, v);
            fetch(j, tokens[j], mine && more && i + D + j < count);
        }
        if (key >= none) break;
    }
    if constexpr (VB >= 8) asm volatile("cp.async.wait_all;" ::: "memory");
    if (key < none) {
        if (!head && open) {
            if (mine) Values<float, N>::store(g.partial + (chunk * 2 + 1) * g.width + c, sum);
        } else {
            flush();
        }
    }
    const bool starts = open && !through;
    if (!continues && !starts) return;
    // this group's partials are out: count them in, and join the rows whose last one that was
    __threadfence();
    group_sync();
    Join* join = joins[threadIdx.y];
    if (threadIdx.x < 32) {
        const unsigned lanes = blockDim.x < 32 ? group_lanes() : 0xffffffffu;
        const int base = blockDim.x < 32 ? (threadIdx.y * blockDim.x) & 31 : 0;
        const int64_t last = __shfl_sync(lanes, far, base + 1);  // of the row that goes on to this chunk
        const bool second = threadIdx.x == 2;
        if (threadIdx.x == 0 ? continues : second && starts) {
            const int64_t from = second ? chunk : far, to = second ? far : last;
            uint32_t others;
            uint32_t* counter = block_counter(g, from, to, chunk, tile, &others);
            join[second] = {(int32_t)from, (int32_t)to, atomicAdd(counter, 1u) == others};
            __threadfence();
        }
    }
    group_sync();
    if (continues && join[0].complete)
        join_row<T, TO, N>(g, first_key, join[0].first, join[0].last, chunk, tile, c, mine, &join[0].complete);
    if (starts && join[1].complete)
        join_row<T, TO, N>(g, last_key, join[1].first, join[1].last, chunk, tile, c, mine, &join[1].complete);
}

// Zeros of the rows that no sorted place holds: a lane searches a row, then the warp writes.  The search is in
// shared memory where the places fit there: its steps wait for one another, and from L2 they take most of the
// time of a small call.
constexpr int kStaged = 2048;
template <typename T, typename TO>
__device__ __forceinline__ void zero_rows(const Grad<T, TO>& g, int64_t block) {
    __shared__ uint32_t staged[kStaged];
    const int threads = blockDim.x * blockDim.y, t = threadIdx.y * blockDim.x + threadIdx.x, lane = t & 31;
    const int64_t first = (block * (threads >> 5) + (t >> 5)) * g.rows_per_warp;
    const int64_t row = first + lane;
    const bool small = g.n <= kStaged;
    if (small) {
#pragma unroll 4
        for (int i = t; i < g.n; i += threads) staged[i] = g.pairs[i].x;
        __syncthreads();
    }
    bool empty = lane < g.rows_per_warp && row < g.rows;
    if (empty) {
        int64_t lo = 0, hi = g.n;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if ((small ? staged[mid] : g.pairs[mid].x) < (uint32_t)row) lo = mid + 1;
            else hi = mid;
        }
        empty = lo >= g.n || (small ? staged[lo] : g.pairs[lo].x) != (uint32_t)row;
    }
    for (unsigned left = __ballot_sync(0xffffffffu, empty); left;) {  // by runs of empty rows
        const int from = __ffs(left) - 1, run = __ffs(~(left >> from)) - 1, rows_ = run < 0 ? 32 : run;
        left &= ~((rows_ == 32 ? ~0u : (1u << rows_) - 1u) << from);
        TO* to = g.out + (first + from) * g.width;
        const int64_t elements = rows_ * g.width;
        // single elements up to the first 16-byte boundary, whole vectors, the rest
        const int64_t lead = min(elements, (int64_t)((16 - (reinterpret_cast<uintptr_t>(to) & 15)) & 15) / (int)sizeof(TO));
        const int64_t whole = (elements - lead) * (int)sizeof(TO) / 16;
        const int64_t done = lead + whole * (16 / (int)sizeof(TO));
        if (lane < lead) to[lane] = rows::from_float<TO>(0.0f);
        for (int64_t i = lane; i < whole; i += 32) reinterpret_cast<uint4*>(to + lead)[i] = make_uint4(0, 0, 0, 0);
        if (done + lane < elements) to[done + lane] = rows::from_float<TO>(0.0f);
    }
}

template <typename T, typename TO, int VB>
__global__ void __launch_bounds__(256, 3) grad_kernel(const Grad<T, TO> g) {
    after_last();
    if ((int64_t)blockIdx.x < g.sum_blocks) sum_chunk<T, TO, VB>(g, blockIdx.x);
    else zero_rows(g, blockIdx.x - g.sum_blocks);
}

// Threads a row: a power of two from 4 up to 32 vectors, else whole warps, at most 256 a column tile.  Up to
// 32768 tokens a warp at least: groups that share a warp take their turns wherever their rows end differently.  A warp
// against less (us, bf16): 2000 into 1000 x 32 12.3 / 14.7, 32768 into 5000 x 64 24.1 / 23.2, 131072 into 100000 x 64
// 41.7 / 35.9.
struct Shape {
    int group, groups, tiles;
};
inline Shape shape_of(int64_t n, int64_t vectors) {
    Shape s{};
    s.tiles = (int)((vectors + 255) / 256);
    if (vectors <= 32) {
        s.group = n <= 32768 ? 32 : 4;
        while (s.group < vectors) s.group <<= 1;
    } else {
        s.group = (int)(((vectors + s.tiles - 1) / s.tiles + 31) / 32 * 32);
    }
    s.groups = 256 / s.group;
    return s;
}

// Places a chunk, a multiple of 8 as sum_chunk needs.  A chunk costs some microseconds of its own (its first
// loads, its join), so up to 128 while that leaves 16 warps of work an SM; at least 16.  Measured with chunks of
// 16 / 32 / 64 / 128: 131072 x 2048 bf16 212 / 173 / 162 / 156 us, 20000 x 2048 f16 37 / 32 / 28 / 32 us,
// 1000 x 129 f32 11 / 13 / 16 / 25 us.
inline int chunk_of(int64_t n, const Shape& s) {
    const int64_t c = n * s.tiles * s.group / 32 / (148 * 16);
    return (int)(c < 16 ? 16 : c > 128 ? 128 : c / 8 * 8);
}

struct Layout {
    uint2* pairs;
    float* partial;
    uint32_t* arrived;
    int64_t arrivals;
    void* sort;
    size_t sort_bytes, bytes;
};
// The chunk and the column tiles depend on the vector size, which a workspace query does not give: the
// partials are sized for the fewest vectors a row can have (16 bytes of a 16-bit type), which makes the
// shortest chunk, the counters for that chunk and the most tiles (an element a vector).
inline Layout layout(void* ws, int64_t n, int64_t rows_, int64_t width) {
    Layout l{};
    char* base = static_cast<char*>(ws);
    auto take = [&](size_t bytes) {
        char* r = base + l.bytes;
        l.bytes += (bytes + 255) / 256 * 256;
        return r;
    };
    l.pairs = reinterpret_cast<uint2*>(take(sizeof(uint2) * n));
    l.sort_bytes = index_sort_bytes(n, rows_);
    l.sort = take(l.sort_bytes);
    const int chunk = chunk_of(n, shape_of(n, (width + 7) / 8));
    const int64_t chunks = (n + chunk - 1) / chunk;
    l.partial = reinterpret_cast<float*>(take(sizeof(float) * 2 * width * chunks));
    l.arrivals = chunks * 3 * shape_of(n, width).tiles;
    l.arrived = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t) * l.arrivals));
    return l;
}

template <typename T, typename TO, int VB>
cudaError_t run_grad(Grad<T, TO> g, cudaStream_t st) {
    const Shape s = shape_of(g.n, g.width * (int64_t)sizeof(T) / VB);
    const dim3 block(s.group, s.groups);
    g.tiles = s.tiles;
    g.chunk = chunk_of(g.n, s);
    g.chunks = (g.n + g.chunk - 1) / g.chunk;
    g.sum_blocks = (g.chunks + s.groups - 1) / s.groups * s.tiles;
    int64_t zero_blocks = 0;
    if (!g.accumulate) {  // at most 32 rows a warp, fewer to have 16 warps an SM
        const int64_t per = g.rows / (148 * 16);
        g.rows_per_warp = (int)(per < 1 ? 1 : per > 32 ? 32 : per);
        const int warps = s.group * s.groups / 32;
        zero_blocks = (g.rows + (int64_t)g.rows_per_warp * warps - 1) / ((int64_t)g.rows_per_warp * warps);
    }
    count_launches(1);
    return launch_next(grad_kernel<T, TO, VB>, dim3((unsigned)(g.sum_blocks + zero_blocks)), block, 0, st, g);
}

}  // namespace embedding
}  // namespace hb

using namespace hb;
using namespace hb::embedding;

extern "C" int hb_embedding_lookup(int type, const void* table, int64_t table_stride, int64_t rows_, int64_t width,
                                   const void* ids, int id_bytes, int64_t n, double scale, void* out, void* stream) {
    if (!rows::valid_type(type) || (id_bytes != 4 && id_bytes != 8))
        return abi_fail(HB_BAD_ARGUMENT, "embedding lookup: unknown type");
    if (rows_ < 0 || width < 0 || n < 0 || n > INT32_MAX || width > INT32_MAX)
        return abi_fail(HB_BAD_ARGUMENT, "embedding lookup: sizes out of range");
    if (n == 0 || width == 0) return HB_OK;
    if ((rows_ > 0 && !table) || !ids || !out) return abi_fail(HB_BAD_ARGUMENT, "embedding lookup: null pointer");
    const int size = rows::type_bytes(type);
    if ((rows::address_bits(table) | rows::address_bits(out)) % size || rows::address_bits(ids) % id_bytes)
        return abi_fail(HB_BAD_ARGUMENT, "embedding lookup: misaligned pointer");
    const int vb = rows::vector_bytes(rows::address_bits(table) | rows::address_bits(out) |
                                      (uint64_t)(table_stride * size) | (uint64_t)(width * size), type);
    // few rows: a thread a vector, so that every load starts at once.  Enough rows for 16 blocks an SM: 4
    // vectors in flight a thread, of 4 rows, or of one where a row has more than 128.  One vector against 4 (us, rows of
    // 2048 bf16): 5 rows 1.8 / 2.5, 1000 2.8 / 2.7, 2400 4.9 / 4.0, 8000 12.4 / 7.5.  Four of 4 rows against one: 32768
    // rows of 64 vectors 8.0 / 10.9, of 128 20.8 / 19.9, of 256 45.0 / 41.1; 97839 of 335 vectors 83 / 58.
    const int64_t vectors = width * size / vb;
    const bool many = n * (vectors < 256 ? vectors : 256) >= (int64_t)148 * 16 * 256, wide = many && vectors > 128;
    const int group = (int)(wide ? 32 : vectors < 256 ? vectors : 256), groups = 256 / group;
    const int64_t per = groups * (many && !wide ? 4 : 1);
    const unsigned blocks = (unsigned)((n + per - 1) / per);
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        constexpr int VB = decltype(b)::value;
        const auto kernel = wide ? lookup_kernel<T, VB, 1, 4> : many ? lookup_kernel<T, VB, 4, 1> : lookup_kernel<T, VB, 1, 1>;
        kernel<<<blocks, dim3(group, groups), 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(table), table_stride, rows_, width, ids, id_bytes, n, (float)scale,
            static_cast<T*>(out));
    });
    count_launches(1);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("embedding lookup: ") + cudaGetErrorString(e));
}

extern "C" size_t hb_embedding_grad_workspace(int64_t n, int64_t rows_, int64_t width) {
    if (n < 0 || n > INT32_MAX || rows_ < 1 || rows_ >= INT32_MAX || width < 0 || width > INT32_MAX) return 0;
    return layout(nullptr, n, rows_, width).bytes;
}

extern "C" int hb_embedding_grad(int type, const void* dy, int64_t dy_stride, const void* ids, int id_bytes, int64_t n,
                                 int64_t rows_, int64_t width, double scale, int out_type, void* out, int accumulate,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    if (!rows::valid_type(type) || (out_type != type && out_type != HB_F32) || (id_bytes != 4 && id_bytes != 8))
        return abi_fail(HB_BAD_ARGUMENT, "embedding gradient: the gradient has dy's type or is fp32, ids are 32 or 64 bits");
    if (rows_ < 1 || rows_ >= INT32_MAX || width < 0 || width > INT32_MAX || n < 0 || n > INT32_MAX)
        return abi_fail(HB_BAD_ARGUMENT, "embedding gradient: sizes out of range");
    if (dy_stride < 0 || dy_stride > UINT32_MAX / rows::type_bytes(type))
        return abi_fail(HB_BAD_ARGUMENT, "embedding gradient: rows of dy must start less than 2^32 bytes apart");
    if (width == 0) return HB_OK;
    if (!out || (n > 0 && (!dy || !ids || !workspace))) return abi_fail(HB_BAD_ARGUMENT, "embedding gradient: null pointer");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int size = rows::type_bytes(type), out_size = rows::type_bytes(out_type);
    cudaError_t e = cudaSuccess;
    if (n == 0) {
        if (!accumulate) e = cudaMemsetAsync(out, 0, (size_t)rows_ * width * out_size, st);
        return e == cudaSuccess ? HB_OK : abi_fail(HB_CUDA, std::string("embedding gradient: ") + cudaGetErrorString(e));
    }
    if (rows::address_bits(workspace) % 256 || rows::address_bits(dy) % size || rows::address_bits(out) % out_size ||
        rows::address_bits(ids) % id_bytes)
        return abi_fail(HB_BAD_ARGUMENT, "embedding gradient: misaligned pointer, or a workspace that is not 256-byte aligned");
    const Layout l = layout(workspace, n, rows_, width);
    if (workspace_bytes < l.bytes)
        return abi_fail(HB_WORKSPACE, "workspace smaller than hb_embedding_grad_workspace()");
    const int rc = index_sort(ids, id_bytes, n, rows_, nullptr, nullptr, l.pairs, nullptr, l.sort, l.sort_bytes, st,
                              l.arrived, l.arrivals);
    if (rc) return rc;
    int vb = rows::vector_bytes(rows::address_bits(dy) | (uint64_t)(dy_stride * size) | (uint64_t)(width * size), type);
    while (vb > size) {
        const int need = vb / size * out_size < 16 ? vb / size * out_size : 16;
        if (rows::address_bits(out) % need == 0) break;
        vb >>= 1;
    }
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        constexpr int VB = decltype(b)::value;
        auto run = [&](auto o) {
            using TO = decltype(o);
            Grad<T, TO> g{};
            g.dy = static_cast<const T*>(dy);
            g.dy_stride = dy_stride;
            g.n = n;
            g.rows = rows_;
            g.width = width;
            g.scale = (float)scale;
            g.pairs = l.pairs;
            g.partial = l.partial;
            g.arrived = l.arrived;
            g.out = static_cast<TO*>(out);
            g.accumulate = accumulate;
            e = run_grad<T, TO, VB>(g, st);
        };
        if (out_type == HB_F32) run(float{});
        else run(T{});
    });
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("embedding gradient: ") + cudaGetErrorString(e));
}
