// Rows sorted by expert and back: the moves around the experts of a routed layer,
// and their gradients.
//
// Entry e = t * slots + k of an assignment sends token t to expert index[t, k];
// position[e] is its place among the entries sorted by expert, and the first
// `kept` places have an expert.
//   dispatch       xs[p] = x[t]                         (0 for p >= kept)
//   combine        y[t]  = sum_k w[t, k] z[position[t, k]]   over places < kept
//   combine grad   dz[p] = w[t, k] dy[t] (0 for p >= kept),  dw[t, k] = <dy[t], z[p]>
//   dispatch grad  dx[t] = combine of dxs without weights
//
// Every kernel goes by token: a group of threads holds the columns of a token, so
// x, dy and y cross HBM once and each sorted row once, which is all they have to.
// Bound by HBM, so what counts is loads in flight: each thread has 4 vectors of 8 or
// 16 bytes under way, or 16 and more shorter ones, of one row or of 4.  Sums are fp32
// and run over k in order (no atomics): the result does not depend on the launch.
//
// Measured on a B200, us and TB/s of the bytes above: 32768 tokens x 4 of 2048 bf16
// dispatch 110 (6.1), combine 110 (6.1), its gradient 194 (6.2); 65536 x 8: 389 (6.2), 380
// (6.4), 710 (6.4).  262144 x 1 of 128 f32: 43, 43, 64.  Rows off the 16-byte grid stay at
// 60 % of that (30000 x 2 of 1001 bf16: 42, 46, 79): 2-byte loads hold too few bytes in
// flight, and shifting aligned words together costs more registers than it saves.
#include <string>

#include "index_sort.cuh"
#include "internal.h"
#include "rows.cuh"

namespace hb {
namespace routing {

using rows::Vec;

struct Moves {
    int64_t tokens, entries, width;
    int slots;
    const int32_t* position;
    const int32_t* kept;  // device
};

__device__ __forceinline__ uint32_t kept_entries(const Moves& m) {
    return (uint32_t)min((int64_t)max(*m.kept, 0), m.entries);
}

// Column steps of a narrow row: short vectors (rows off the 16-byte grid) take four to hold as many bytes in
// flight as one long vector.
constexpr int steps_of(int vb) { return vb >= 8 ? 1 : 4; }

// A group serves M tokens, U column steps at a time: 4 vectors a thread in flight, 16 of 4 bytes, 32 of 2.  Wide
// rows: one token; narrow ones, of at most steps_of(VB) vectors a thread: 4.
template <typename T, int VB, int G, bool NARROW>
__global__ void __launch_bounds__(256) dispatch_kernel(Moves m, const T* __restrict__ x, int64_t x_stride,
                                                       T* __restrict__ out) {
    using V = Vec<T, VB>;
    constexpr int M = NARROW ? 4 : 1, U = NARROW ? steps_of(VB) : VB >= 8 ? 4 : VB == 4 ? 16 : 32;
    const int64_t token = ((int64_t)blockIdx.x * (256 / G) + threadIdx.x / G) * M;
    if (token >= m.tokens) return;
    const uint32_t kept = kept_entries(m);
    for (int64_t c0 = (threadIdx.x % G) * V::N; c0 < m.width; c0 += G * V::N * U) {
        V v[M][U];
#pragma unroll
        for (int t = 0; t < M; ++t)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (token + t < m.tokens && c0 + u * G * V::N < m.width)
                    v[t][u].load_once(x + (token + t) * x_stride + c0 + u * G * V::N);
        for (int k = 0; k < m.slots; ++k) {
            uint32_t p[M];
#pragma unroll
            for (int t = 0; t < M; ++t)
                p[t] = token + t < m.tokens ? (uint32_t)m.position[(token + t) * m.slots + k] : ~0u;
#pragma unroll
            for (int t = 0; t < M; ++t) {
                if (p[t] >= (uint64_t)m.entries) continue;
                T* to = out + (int64_t)p[t] * m.width + c0;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (c0 + u * G * V::N >= m.width) break;
                    if (p[t] >= kept) {
                        V w;
                        w.zero();
                        w.store(to + u * G * V::N);
                    } else {
                        v[t][u].store_once(to + u * G * V::N);
                    }
                }
            }
        }
    }
}

// Weights of the entries e0..e0+B-1 (the last entry's beyond it); 1 without weights.
template <int B>
__device__ __forceinline__ void load_weights(const Moves& m, const void* weights, int type, int64_t e0, float (&w)[B]) {
#pragma unroll
    for (int b = 0; b < B; ++b) w[b] = 1.0f;
    if (!weights) return;
    if (type == HB_F32) {
#pragma unroll
        for (int b = 0; b < B; ++b) w[b] = static_cast<const float*>(weights)[min(e0 + b, m.entries - 1)];
    } else {
#pragma unroll
        for (int b = 0; b < B; ++b) w[b] = rows::load_weight(weights, type, min(e0 + b, m.entries - 1));
    }
}

// SLOTS 1, 2, 4: a group serves 4, 2, 1 tokens, 4 sorted rows in flight; 0: any number of slots, 4 at a time.
template <typename T, int VB, int G, int SLOTS>
__global__ void __launch_bounds__(256) combine_kernel(Moves m, const T* __restrict__ z, int64_t z_stride,
                                                      const void* __restrict__ weights, int weight_type,
                                                      T* __restrict__ out) {
    using V = Vec<T, VB>;
    constexpr int B = 4, M = SLOTS ? B / SLOTS : 1, S = B / M;  // rows, tokens, rows of a token in flight
    constexpr int U = VB >= 8 ? 1 : VB == 4 ? 4 : 8;            // column steps in flight
    const int64_t token = ((int64_t)blockIdx.x * (256 / G) + threadIdx.x / G) * M;
    if (token >= m.tokens) return;
    const int slots = SLOTS ? SLOTS : m.slots;
    const int64_t e0 = token * slots, e1 = min(m.entries, e0 + (SLOTS ? B : slots));
    uint32_t p[B];
    float w[B];
    // places first, then weights, then rows: loads that wait for one another only where they must
    auto places = [&](int64_t e) {
#pragma unroll
        for (int b = 0; b < B; ++b) p[b] = (uint32_t)m.position[min(e + b, e1 - 1)];
        load_weights(m, weights, weight_type, e, w);
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (e + b >= e1) p[b] = ~0u;
    };
    if (SLOTS) places(e0);
    const uint32_t kept = kept_entries(m);
    for (int64_t c0 = (threadIdx.x % G) * V::N; c0 < m.width; c0 += G * V::N * U) {
        V v[U][B];
        auto load = [&]() {
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const T* row = z + (int64_t)p[b] * z_stride + c0;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (p[b] < kept && c0 + u * G * V::N < m.width) v[u][b].load_once(row + u * G * V::N);
            }
        };
        auto add = [&](int b, int u, float (&sum)[V::N]) {
            if (p[b] < kept) {
#pragma unroll
                for (int i = 0; i < V::N; ++i) sum[i] = fmaf(w[b], rows::to_float(v[u][b].v[i]), sum[i]);
            }
        };
        auto store = [&](int64_t t, int u, const float (&sum)[V::N]) {
            if (t >= m.tokens || c0 + u * G * V::N >= m.width) return;
            V r;
#pragma unroll
            for (int i = 0; i < V::N; ++i) r.v[i] = rows::from_float<T>(sum[i]);
            r.store_once(out + t * m.width + c0 + u * G * V::N);
        };
        if (SLOTS) {  // all rows of the tokens at once; one token's sum at a time
            load();
#pragma unroll
            for (int t = 0; t < M; ++t)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float sum[V::N] = {};
#pragma unroll
                    for (int k = 0; k < S; ++k) add(t * S + k, u, sum);
                    store(token + t, u, sum);
                }
        } else {
            float sum[U][V::N] = {};
            for (int64_t e = e0; e < e1; e += B) {
                places(e);
                load();
#pragma unroll
                for (int b = 0; b < B; ++b)
#pragma unroll
                    for (int u = 0; u < U; ++u) add(b, u, sum[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) store(token, u, sum[u]);
        }
    }
}

// Sums of B values a thread over the group; every thread has them.
template <int G, int B>
__device__ __forceinline__ void group_sum(float (&v)[B]) {
    constexpr int W = G < 32 ? G : 32;
    const unsigned lanes = G < 32 ? ((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G) : 0xffffffffu;
#pragma unroll
    for (int s = W / 2; s > 0; s >>= 1)
#pragma unroll
        for (int b = 0; b < B; ++b) v[b] += __shfl_xor_sync(lanes, v[b], s);
    if (G == 256) {
        __shared__ float part[B][8];
        __syncthreads();
#pragma unroll
        for (int b = 0; b < B; ++b)
            if ((threadIdx.x & 31) == 0) part[b][threadIdx.x >> 5] = v[b];
        __syncthreads();
#pragma unroll
        for (int b = 0; b < B; ++b) {
            v[b] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[b] += part[b][i];
        }
    }
}

// Wide rows: a group goes through a token's entries, 4 vectors a thread (8 of 4 bytes, 16 of 2) of z and of dy,
// which is in L1 after the first entry.  ways: groups a token, 1, or one an entry when tokens are few.
template <typename T, int VB, int G>
__global__ void __launch_bounds__(256) combine_grad_kernel(Moves m, int ways, const T* __restrict__ dy, int64_t dy_stride,
                                                           const T* __restrict__ z, int64_t z_stride,
                                                           const void* __restrict__ weights, int weight_type,
                                                           T* __restrict__ dz, void* __restrict__ dw) {
    using V = Vec<T, VB>;
    constexpr int U = VB >= 8 ? 4 : VB == 4 ? 8 : 16;
    const int64_t group = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int64_t token = ways == 1 ? group : group / ways;
    if (token >= m.tokens) return;  // G = 256: the whole block or none of it
    const uint32_t kept = kept_entries(m);
    const T* grow = dy + token * dy_stride;
    const int first = ways == 1 ? 0 : (int)(group % ways), last = ways == 1 ? m.slots : first + 1;
    for (int k = first; k < last; ++k) {
        const int64_t e = token * m.slots + k;
        const uint32_t p = (uint32_t)m.position[e];
        const bool there = p < kept;
        const float w = weights && there ? rows::load_weight(weights, weight_type, e) : 1.0f;
        const T* zrow = z + (int64_t)p * z_stride;
        T* to = dz + (int64_t)p * m.width;
        float dot[1] = {0.0f};
        if (there) {
            for (int64_t c0 = (threadIdx.x % G) * V::N; c0 < m.width; c0 += G * V::N * U) {
                V g[U], a[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t c = c0 + u * G * V::N;
                    if (c < m.width) {
                        if (dw) a[u].load_once(zrow + c);
                        g[u].load(grow + c);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t c = c0 + u * G * V::N;
                    if (c < m.width) {
                        V r;
#pragma unroll
                        for (int i = 0; i < V::N; ++i) {
                            const float gv = rows::to_float(g[u].v[i]);
                            if (dw) dot[0] = fmaf(gv, rows::to_float(a[u].v[i]), dot[0]);
                            r.v[i] = rows::from_float<T>(w * gv);
                        }
                        if (VB >= 8) r.store_once(to + c);
                        else r.store(to + c);  // sectors of short ones are written in two parts: kept until whole
                    }
                }
            }
        } else if (p < (uint64_t)m.entries) {
            V r;
            r.zero();
            for (int64_t c = (threadIdx.x % G) * V::N; c < m.width; c += G * V::N) r.store(to + c);
        }
        if (dw) {
            group_sum<G>(dot);
            if (threadIdx.x % G == 0) rows::store_weight(dw, weight_type, e, dot[0]);
        }
    }
}

// Narrow rows, of at most steps_of(VB) vectors a thread: a group serves 4 entries that follow each other.
template <typename T, int VB, int G>
__global__ void __launch_bounds__(256) combine_grad_narrow(Moves m, const T* __restrict__ dy, int64_t dy_stride,
                                                           const T* __restrict__ z, int64_t z_stride,
                                                           const void* __restrict__ weights, int weight_type,
                                                           T* __restrict__ dz, void* __restrict__ dw) {
    using V = Vec<T, VB>;
    constexpr int B = 4, U = steps_of(VB);
    const int64_t e0 = ((int64_t)blockIdx.x * (256 / G) + threadIdx.x / G) * B;
    if (e0 >= m.entries) return;
    const int64_t c = (threadIdx.x % G) * V::N;
    uint32_t p[B];
    float w[B], dot[B];
    V g[B][U], a[B][U];
#pragma unroll
    for (int b = 0; b < B; ++b) p[b] = (uint32_t)m.position[min(e0 + b, m.entries - 1)];
    load_weights(m, weights, weight_type, e0, w);
    const uint32_t kept = kept_entries(m);
#pragma unroll
    for (int b = 0; b < B; ++b) {
        if (e0 + b >= m.entries) p[b] = ~0u;
        const T* zrow = z + (int64_t)p[b] * z_stride;
        const T* grow = dy + (int64_t)((uint32_t)(e0 + b) / (uint32_t)m.slots) * dy_stride;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (p[b] < kept && c + u * G * V::N < m.width) {
                if (dw) a[b][u].load_once(zrow + c + u * G * V::N);
                g[b][u].load(grow + c + u * G * V::N);
            }
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
        dot[b] = 0.0f;
        if (p[b] >= (uint64_t)m.entries) continue;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c + u * G * V::N >= m.width) break;
            V r;
            if (p[b] < kept) {
#pragma unroll
                for (int i = 0; i < V::N; ++i) {
                    const float gv = rows::to_float(g[b][u].v[i]);
                    if (dw) dot[b] = fmaf(gv, rows::to_float(a[b][u].v[i]), dot[b]);
                    r.v[i] = rows::from_float<T>(w[b] * gv);
                }
            } else {
                r.zero();
            }
            r.store(dz + (int64_t)p[b] * m.width + c + u * G * V::N);
        }
    }
    if (!dw) return;
    group_sum<G>(dot);
    if (threadIdx.x % G == 0) {
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (e0 + b < m.entries) rows::store_weight(dw, weight_type, e0 + b, dot[b]);
    }
}

// Threads a group: 8 for rows that they hold in their column steps, else a warp; a block when the groups are
// too few to fill the SMs with warps and a row has more than a warp's vectors.
// A warp against 8 threads (us): 262144 x 1 entries of 64 bf16 dispatch 16.3 / 8.1, combine 27.5 / 8.8, gradient
// 46 / 14.6; 2000 x 2 the same.  Warps against blocks (us, rows of 2048 bf16): combine of 64 x 2 entries 5.2 / 2.3,
// 1000 x 8 10.6 / 6.3; dispatch of 1180 x 2 3.4 / 3.3, 4000 x 2 7.6 / 7.2; the gradient, by an entry, of 300 x 2
// 3.7 / 4.0, 600 x 2 4.5 / 5.6, 2000 x 2 6.0 / 13.
inline int group_of(int64_t groups, int64_t vectors, int vb) {
    if (vectors <= 8 * steps_of(vb)) return 8;
    if (groups < 148 * 8 && vectors > 32) return 256;
    return 32;
}
// Tokens a group of combine_kernel.
inline int tokens_of(int64_t slots) { return slots == 1 ? 4 : slots == 2 ? 2 : 1; }
template <typename F>
inline void for_group(int g, F&& f) {
    if (g == 8) f(rows::Bytes<8>{});
    else if (g == 32) f(rows::Bytes<32>{});
    else f(rows::Bytes<256>{});
}
inline unsigned blocks_of(int64_t groups, int g) { return (unsigned)((groups + 256 / g - 1) / (256 / g)); }

// Shapes and pointers that every move checks; HB_OK or the failure.
int check(const char* what, int type, int64_t tokens, int64_t slots, int64_t width, const void* position,
          const void* kept) {
    if (!rows::valid_type(type)) return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": unknown element type");
    if (tokens < 0 || slots < 1 || width < 0 || tokens > INT32_MAX / slots || width > INT32_MAX)
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": sizes out of range");
    if (tokens > 0 && width > 0 && (!position || !kept))
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": null pointer");
    if ((rows::address_bits(position) | rows::address_bits(kept)) % sizeof(int32_t))
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": misaligned pointer");
    return HB_OK;
}
inline bool misaligned(const void* weights, int type) { return rows::address_bits(weights) % rows::type_bytes(type) != 0; }
int launched(const char* what) {
    count_launches(1);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? HB_OK : abi_fail(HB_LAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace routing
}  // namespace hb

using namespace hb;
using namespace hb::routing;

extern "C" size_t hb_index_sort_workspace(int64_t entries, int64_t bins) {
    if (entries < 0 || entries > INT32_MAX || bins < 1 || bins >= INT32_MAX) return 0;
    return index_sort_bytes(entries, bins);
}

extern "C" int hb_index_sort(const void* index, int index_bytes, int64_t entries, int64_t bins, int32_t* order,
                             int32_t* position, int32_t* offsets, void* workspace, size_t workspace_bytes,
                             void* stream) {
    if (entries < 0 || entries > INT32_MAX || bins < 1 || bins >= INT32_MAX || (index_bytes != 4 && index_bytes != 8))
        return abi_fail(HB_BAD_ARGUMENT, "index sort: sizes out of range");
    if (!offsets || (entries > 0 && (!index || !order || !position)))
        return abi_fail(HB_BAD_ARGUMENT, "index sort: null pointer");
    if ((rows::address_bits(order) | rows::address_bits(position) | rows::address_bits(offsets)) % sizeof(int32_t))
        return abi_fail(HB_BAD_ARGUMENT, "index sort: misaligned pointer");
    return index_sort(index, index_bytes, entries, bins, order, position, nullptr, offsets, workspace, workspace_bytes,
                      static_cast<cudaStream_t>(stream));
}

extern "C" int hb_route_dispatch(int type, const void* x, int64_t x_stride, int64_t tokens, int64_t slots, int64_t width,
                                 const int32_t* position, const int32_t* kept, void* sorted, void* stream) {
    const int rc = check("route dispatch", type, tokens, slots, width, position, kept);
    if (rc) return rc;
    if (tokens == 0 || width == 0) return HB_OK;
    if (!x || !sorted) return abi_fail(HB_BAD_ARGUMENT, "route dispatch: null pointer");
    const int size = rows::type_bytes(type);
    const Moves m{tokens, tokens * slots, width, (int)slots, position, kept};
    if ((rows::address_bits(x) | rows::address_bits(sorted)) % size)
        return abi_fail(HB_BAD_ARGUMENT, "route dispatch: misaligned pointer");
    const int vb = rows::vector_bytes(rows::address_bits(x) | rows::address_bits(sorted) | (uint64_t)(x_stride * size) |
                                      (uint64_t)(width * size), type);
    const int64_t vectors = width * size / vb;
    const int g = group_of(tokens, vectors, vb);
    const auto st = static_cast<cudaStream_t>(stream);
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        for_group(g, [&](auto gg) {
            constexpr int G = decltype(gg)::value, VB = decltype(b)::value;
            if constexpr (G < 256) {
                if (vectors <= G * steps_of(VB)) {
                    dispatch_kernel<T, VB, G, true><<<blocks_of((tokens + 3) / 4, G), 256, 0, st>>>(
                        m, static_cast<const T*>(x), x_stride, static_cast<T*>(sorted));
                    return;
                }
            }
            if constexpr (G > 8)  // 8 threads are for narrow rows
                dispatch_kernel<T, VB, G, false><<<blocks_of(tokens, G), 256, 0, st>>>(
                    m, static_cast<const T*>(x), x_stride, static_cast<T*>(sorted));
        });
    });
    return launched("route dispatch");
}

extern "C" int hb_route_combine(int type, const void* z, int64_t z_stride, int64_t tokens, int64_t slots, int64_t width,
                                const int32_t* position, const int32_t* kept, const void* weights, int weight_type,
                                void* out, void* stream) {
    const int rc = check("route combine", type, tokens, slots, width, position, kept);
    if (rc) return rc;
    if (weights && !rows::valid_type(weight_type)) return abi_fail(HB_BAD_ARGUMENT, "route combine: unknown weight type");
    if (tokens == 0 || width == 0) return HB_OK;
    if (!z || !out) return abi_fail(HB_BAD_ARGUMENT, "route combine: null pointer");
    const int size = rows::type_bytes(type);
    const Moves m{tokens, tokens * slots, width, (int)slots, position, kept};
    if ((rows::address_bits(z) | rows::address_bits(out)) % size || (weights && misaligned(weights, weight_type)))
        return abi_fail(HB_BAD_ARGUMENT, "route combine: misaligned pointer");
    const int vb = rows::vector_bytes(rows::address_bits(z) | rows::address_bits(out) | (uint64_t)(z_stride * size) |
                                      (uint64_t)(width * size), type);
    const int64_t groups = (tokens + tokens_of(slots) - 1) / tokens_of(slots);
    const int g = group_of(groups, width * size / vb, vb);
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        for_group(g, [&](auto gg) {
            constexpr int G = decltype(gg)::value, VB = decltype(b)::value;
            auto launch = [&](auto s) {
                combine_kernel<T, VB, G, decltype(s)::value>
                    <<<blocks_of(groups, G), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                        m, static_cast<const T*>(z), z_stride, weights, weight_type, static_cast<T*>(out));
            };
            if (slots == 1) launch(rows::Bytes<1>{});
            else if (slots == 2) launch(rows::Bytes<2>{});
            else if (slots == 4) launch(rows::Bytes<4>{});
            else launch(rows::Bytes<0>{});
        });
    });
    return launched("route combine");
}

extern "C" int hb_route_combine_grad(int type, const void* dy, int64_t dy_stride, const void* z, int64_t z_stride,
                                     int64_t tokens, int64_t slots, int64_t width, const int32_t* position,
                                     const int32_t* kept, const void* weights, int weight_type, void* dz, void* dweights,
                                     void* stream) {
    const int rc = check("route combine gradient", type, tokens, slots, width, position, kept);
    if (rc) return rc;
    if ((weights || dweights) && !rows::valid_type(weight_type))
        return abi_fail(HB_BAD_ARGUMENT, "route combine gradient: unknown weight type");
    if (tokens == 0) return HB_OK;
    if (!position || !kept || (width > 0 && (!dy || !dz || (dweights && !z))))
        return abi_fail(HB_BAD_ARGUMENT, "route combine gradient: null pointer");
    if (width == 0 && !dweights) return HB_OK;
    const int size = rows::type_bytes(type);
    const Moves m{tokens, tokens * slots, width, (int)slots, position, kept};
    uint64_t bits = rows::address_bits(dy) | rows::address_bits(dz) | (uint64_t)(dy_stride * size) | (uint64_t)(width * size);
    if (dweights) bits |= rows::address_bits(z) | (uint64_t)(z_stride * size);
    if (bits % size || (weights && misaligned(weights, weight_type)) || (dweights && misaligned(dweights, weight_type)))
        return abi_fail(HB_BAD_ARGUMENT, "route combine gradient: misaligned pointer");
    const int vb = rows::vector_bytes(bits, type);
    const int64_t vectors = width * size / vb;
    // Too few tokens to fill the SMs with a warp each: a group an entry.  A group a token against an entry (us, bf16): 457 x
    // 8 x 145 17.9 / 4.6, 2000 x 8 x 2048 26.7 / 20.2, 4000 x 8 x 2048 48.7 / 43.0; 8000 x 8 x 2048 88.8 / 88.9.
    const int ways = tokens < 148 * 32 ? (int)slots : 1;
    const int g = group_of(tokens * ways, vectors, vb);
    const auto st = static_cast<cudaStream_t>(stream);
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        for_group(g, [&](auto gg) {
            constexpr int G = decltype(gg)::value, VB = decltype(b)::value;
            if constexpr (G < 256) {
                if (vectors <= G * steps_of(VB)) {
                    combine_grad_narrow<T, VB, G><<<blocks_of((m.entries + 3) / 4, G), 256, 0, st>>>(
                        m, static_cast<const T*>(dy), dy_stride, static_cast<const T*>(z), z_stride, weights, weight_type,
                        static_cast<T*>(dz), dweights);
                    return;
                }
            }
            if constexpr (G > 8)
                combine_grad_kernel<T, VB, G><<<blocks_of(tokens * ways, G), 256, 0, st>>>(
                    m, ways, static_cast<const T*>(dy), dy_stride, static_cast<const T*>(z), z_stride, weights, weight_type,
                    static_cast<T*>(dz), dweights);
        });
    });
    return launched("route combine gradient");
}
