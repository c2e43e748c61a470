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
// partial a chunk, and a second launch adds them in chunk order.  No atomics: the
// result does not depend on the launch.  Blocks behind the chunks write the zeros
// of the rows that no token names.
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

template <typename T, int VB>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ table, int64_t stride, int64_t rows_,
                                                     int64_t width, const void* __restrict__ ids, int id_bytes, int64_t n,
                                                     float scale, T* __restrict__ out) {
    using V = Vec<T, VB>;
    constexpr int U = 4;
    const int g = blockDim.x;
    const int64_t i = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (i >= n) return;
    const int64_t id = load_id(ids, id_bytes, i);
    const bool there = id >= 0 && id < rows_;
    const T* row = table + (there ? id : 0) * stride;
    T* to = out + i * width;
    for (int64_t c0 = threadIdx.x * V::N; c0 < width; c0 += (int64_t)g * V::N * U) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * g * V::N < width && there) v[u].load(row + c0 + u * g * V::N);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t c = c0 + u * g * V::N;
            if (c < width) {
#pragma unroll
                for (int j = 0; j < V::N; ++j)
                    v[u].v[j] = rows::from_float<T>(there ? scale * rows::to_float(v[u].v[j]) : 0.0f);
                v[u].store(to + c);
            }
        }
    }
}

template <typename T, typename TO>
struct Grad {
    const T* dy;
    int64_t dy_stride, n, rows, width;
    float scale;
    const int32_t* order;    // token of each sorted place
    const uint32_t* keys;    // row of each sorted place; `rows` for an id outside the table
    int chunk;               // places a group
    int64_t chunks;
    int tiles;               // column tiles
    float* partial;          // [chunks][2][width]: the row that a chunk continues, the row that it leaves open
    TO* out;
    int accumulate;
    int64_t sum_blocks;
    int rows_per_warp;
};

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

template <typename T, typename TO, int VB>
__device__ __forceinline__ void sum_chunk(const Grad<T, TO>& g, int64_t block) {
    using V = Vec<T, VB>;
    constexpr int N = V::N, U = 8;
    const int tile = (int)(block % g.tiles);
    const int64_t c = ((int64_t)tile * blockDim.x + threadIdx.x) * N;
    const int64_t chunk = block / g.tiles * blockDim.y + threadIdx.y;
    if (chunk >= g.chunks || c >= g.width) return;
    const int64_t p0 = chunk * g.chunk, p1 = min(g.n, p0 + g.chunk);
    uint32_t key = g.keys[p0];
    bool head = p0 > 0 && g.keys[p0 - 1] == key;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    for (int64_t p = p0; p < p1; p += U) {
        V v[U];
        uint32_t k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = p + u < p1 ? g.keys[p + u] : (uint32_t)g.rows;
            if (k[u] < (uint32_t)g.rows) v[u].load_once(g.dy + (int64_t)g.order[p + u] * g.dy_stride + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p + u >= p1) break;
            if (k[u] != key) {
                if (head) Values<float, N>::store(g.partial + (chunk * 2) * g.width + c, sum);
                else write_row<T, TO, N>(g, key, c, sum);
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] = 0.0f;
                key = k[u];
                head = false;
            }
            if (key < (uint32_t)g.rows) {
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += rows::to_float(v[u].v[i]);
            }
        }
    }
    if (key >= (uint32_t)g.rows) return;
    const bool open = p1 < g.n && g.keys[p1] == key;
    if (head) Values<float, N>::store(g.partial + (chunk * 2) * g.width + c, sum);
    else if (open) Values<float, N>::store(g.partial + (chunk * 2 + 1) * g.width + c, sum);
    else write_row<T, TO, N>(g, key, c, sum);
}

// Zeros of the rows that no sorted place holds: a lane searches a row, then the warp writes.
template <typename T, typename TO>
__device__ __forceinline__ void zero_rows(const Grad<T, TO>& g, int64_t block) {
    const int t = threadIdx.y * blockDim.x + threadIdx.x, lane = t & 31;
    const int warps = (blockDim.x * blockDim.y) >> 5;
    if ((t >> 5) >= warps) return;
    const int64_t first = (block * warps + (t >> 5)) * g.rows_per_warp;
    const int64_t row = first + lane;
    bool empty = lane < g.rows_per_warp && row < g.rows;
    if (empty) {
        int64_t lo = 0, hi = g.n;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (g.keys[mid] < (uint32_t)row) lo = mid + 1;
            else hi = mid;
        }
        empty = lo >= g.n || g.keys[lo] != (uint32_t)row;
    }
    for (unsigned left = __ballot_sync(0xffffffffu, empty); left; left &= left - 1) {
        TO* to = g.out + (first + __ffs(left) - 1) * g.width;
        // bytes up to the first 16-byte boundary, whole vectors, the rest
        const int64_t lead = min(g.width, (int64_t)((16 - (reinterpret_cast<uintptr_t>(to) & 15)) & 15) / (int)sizeof(TO));
        const int64_t whole = (g.width - lead) * (int)sizeof(TO) / 16;
        const int64_t done = lead + whole * (16 / (int)sizeof(TO));
        if (lane < lead) to[lane] = rows::from_float<TO>(0.0f);
        for (int64_t i = lane; i < whole; i += 32) reinterpret_cast<uint4*>(to + lead)[i] = make_uint4(0, 0, 0, 0);
        if (done + lane < g.width) to[done + lane] = rows::from_float<TO>(0.0f);
    }
}

template <typename T, typename TO, int VB>
__global__ void __launch_bounds__(256) grad_kernel(const Grad<T, TO> g) {
    if ((int64_t)blockIdx.x < g.sum_blocks) sum_chunk<T, TO, VB>(g, blockIdx.x);
    else zero_rows(g, blockIdx.x - g.sum_blocks);
}

// The rows that cross chunks: the group of the chunk that a row begins in adds its partials in chunk order.
template <typename T, typename TO, int VB>
__global__ void __launch_bounds__(256) join_kernel(const Grad<T, TO> g) {
    constexpr int N = Vec<T, VB>::N, U = 4;
    const int tile = (int)(blockIdx.x % g.tiles);
    const int64_t c = ((int64_t)tile * blockDim.x + threadIdx.x) * N;
    const int64_t chunk = (int64_t)(blockIdx.x / g.tiles) * blockDim.y + threadIdx.y;
    if (chunk + 1 >= g.chunks || c >= g.width) return;
    const int64_t p0 = chunk * g.chunk, p1 = p0 + g.chunk;
    const uint32_t key = g.keys[p1 - 1];
    if (key >= (uint32_t)g.rows || g.keys[p1] != key || (p0 > 0 && g.keys[p0 - 1] == key)) return;
    int64_t lo = p1, hi = g.n;  // first place above the row's
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (g.keys[mid] <= key) lo = mid + 1;
        else hi = mid;
    }
    const int64_t last = (lo - 1) / g.chunk;
    float sum[N];
    Values<float, N>::load(g.partial + (chunk * 2 + 1) * g.width + c, sum);
    for (int64_t q = chunk + 1; q <= last; q += U) {
        float v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q + u <= last) Values<float, N>::load(g.partial + ((q + u) * 2) * g.width + c, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q + u <= last) {
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += v[u][i];
            }
    }
    write_row<T, TO, N>(g, key, c, sum);
}

// Threads a row: a power of two up to 32 vectors, else whole warps, at most 256 a column tile.
struct Shape {
    int group, groups, tiles;
};
inline Shape shape_of(int64_t vectors) {
    Shape s{};
    s.tiles = (int)((vectors + 255) / 256);
    if (vectors <= 32) {
        s.group = 1;
        while (s.group < vectors) s.group <<= 1;
    } else {
        s.group = (int)(((vectors + s.tiles - 1) / s.tiles + 31) / 32 * 32);
    }
    s.groups = 256 / s.group;
    return s;
}

// Places a chunk: 64 when there are plenty, fewer (at least 8) to have 64 warps of work an SM.
inline int chunk_of(int64_t n, const Shape& s) {
    const int64_t warps = n * s.tiles * s.group / 32;
    const int64_t c = warps / (148 * 64);
    return (int)(c < 8 ? 8 : c > 64 ? 64 : c);
}

struct Layout {
    uint32_t* keys;
    int32_t* order;
    float* partial;
    void* sort;
    size_t sort_bytes, bytes;
};
// The chunk depends on the vector size, which a workspace query does not give: the partials are sized
// for the fewest vectors a row can have (16 bytes of a 16-bit type), which makes the shortest chunk.
inline Layout layout(void* ws, int64_t n, int64_t rows_, int64_t width) {
    Layout l{};
    char* base = static_cast<char*>(ws);
    auto take = [&](size_t bytes) {
        char* r = base + l.bytes;
        l.bytes += (bytes + 255) / 256 * 256;
        return r;
    };
    l.keys = reinterpret_cast<uint32_t*>(take(sizeof(uint32_t) * n));
    l.order = reinterpret_cast<int32_t*>(take(sizeof(int32_t) * n));
    l.sort_bytes = index_sort_bytes(n, rows_);
    l.sort = take(l.sort_bytes);
    const int chunk = chunk_of(n, shape_of((width + 7) / 8));
    l.partial = reinterpret_cast<float*>(take(sizeof(float) * 2 * width * ((n + chunk - 1) / chunk)));
    return l;
}

template <typename T, typename TO, int VB>
cudaError_t run_grad(Grad<T, TO> g, cudaStream_t st) {
    const Shape s = shape_of(g.width * (int64_t)sizeof(T) / VB);
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
    grad_kernel<T, TO, VB><<<(unsigned)(g.sum_blocks + zero_blocks), block, 0, st>>>(g);
    count_launches(1);
    if (g.chunks > 1) {
        join_kernel<T, TO, VB><<<(unsigned)g.sum_blocks, block, 0, st>>>(g);
        count_launches(1);
    }
    return cudaGetLastError();
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
    const int vb = rows::vector_bytes(rows::address_bits(table) | rows::address_bits(out) |
                                      (uint64_t)(table_stride * size) | (uint64_t)(width * size), type);
    // a warp a row; a block when the rows are too few to fill the SMs with warps
    const int64_t vectors = width * size / vb;
    Shape s = shape_of(vectors < 32 ? vectors : 32);
    if (n < 148 * 8 && vectors > 32) s = shape_of(256);
    const unsigned blocks = (unsigned)((n + s.groups - 1) / s.groups);
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        lookup_kernel<T, decltype(b)::value><<<blocks, dim3(s.group, s.groups), 0, static_cast<cudaStream_t>(stream)>>>(
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
    if (width == 0) return HB_OK;
    if (!out || (n > 0 && (!dy || !ids || !workspace))) return abi_fail(HB_BAD_ARGUMENT, "embedding gradient: null pointer");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int size = rows::type_bytes(type), out_size = rows::type_bytes(out_type);
    cudaError_t e = cudaSuccess;
    if (n == 0) {
        if (!accumulate) e = cudaMemsetAsync(out, 0, (size_t)rows_ * width * out_size, st);
        return e == cudaSuccess ? HB_OK : abi_fail(HB_CUDA, std::string("embedding gradient: ") + cudaGetErrorString(e));
    }
    const Layout l = layout(workspace, n, rows_, width);
    if (workspace_bytes < l.bytes)
        return abi_fail(HB_WORKSPACE, "workspace smaller than hb_embedding_grad_workspace()");
    const int rc = index_sort(ids, id_bytes, n, rows_, l.order, nullptr, l.keys, nullptr, l.sort, l.sort_bytes, st);
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
            g.order = l.order;
            g.keys = l.keys;
            g.partial = l.partial;
            g.out = static_cast<TO*>(out);
            g.accumulate = accumulate;
            e = run_grad<T, TO, VB>(g, st);
        };
        if (out_type == HB_F32) run(float{});
        else run(T{});
    });
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string("embedding gradient: ") + cudaGetErrorString(e));
}
