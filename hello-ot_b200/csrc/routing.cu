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
// Every kernel goes by token: a group of threads holds the columns of one token,
// so x, dy and y cross HBM once and each sorted row once, which is all they have
// to.  Bound by HBM.  Sums are fp32 and run over k in order (no atomics): the
// result does not depend on the launch.
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

template <typename T, int VB, int G>
__global__ void __launch_bounds__(256) dispatch_kernel(Moves m, const T* __restrict__ x, int64_t x_stride,
                                                       T* __restrict__ out) {
    using V = Vec<T, VB>;
    constexpr int U = 4;
    const int64_t token = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (token >= m.tokens) return;
    const uint32_t kept = kept_entries(m);
    const T* row = x + token * x_stride;
    const int32_t* place = m.position + token * m.slots;
    for (int64_t c0 = (threadIdx.x % G) * V::N; c0 < m.width; c0 += G * V::N * U) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * G * V::N < m.width) v[u].load(row + c0 + u * G * V::N);
        for (int k = 0; k < m.slots; ++k) {
            const uint32_t p = (uint32_t)place[k];
            if (p >= (uint64_t)m.entries) continue;
            T* to = out + (int64_t)p * m.width;
            V w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = c0 + u * G * V::N;
                if (c < m.width) {
                    if (p >= kept) {
                        w[u].zero();
                        w[u].store(to + c);
                    } else {
                        v[u].store(to + c);
                    }
                }
            }
        }
    }
}

template <typename T, int VB, int G>
__global__ void __launch_bounds__(256) combine_kernel(Moves m, const T* __restrict__ z, int64_t z_stride,
                                                      const void* __restrict__ weights, int weight_type,
                                                      T* __restrict__ out) {
    using V = Vec<T, VB>;
    constexpr int B = 4;  // rows in flight
    const int64_t token = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (token >= m.tokens) return;
    const uint32_t kept = kept_entries(m);
    for (int64_t c = (threadIdx.x % G) * V::N; c < m.width; c += G * V::N) {
        float sum[V::N];
#pragma unroll
        for (int i = 0; i < V::N; ++i) sum[i] = 0.0f;
        for (int k0 = 0; k0 < m.slots; k0 += B) {
            V v[B];
            float w[B];
            bool there[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int64_t e = token * m.slots + k0 + b;
                there[b] = false;
                if (k0 + b < m.slots) {
                    const uint32_t p = (uint32_t)m.position[e];
                    there[b] = p < kept;
                    if (there[b]) {
                        v[b].load_once(z + (int64_t)p * z_stride + c);
                        w[b] = weights ? rows::load_weight(weights, weight_type, e) : 1.0f;
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (there[b]) {
#pragma unroll
                    for (int i = 0; i < V::N; ++i) sum[i] = fmaf(w[b], rows::to_float(v[b].v[i]), sum[i]);
                }
        }
        V r;
#pragma unroll
        for (int i = 0; i < V::N; ++i) r.v[i] = rows::from_float<T>(sum[i]);
        r.store(out + token * m.width + c);
    }
}

template <typename T, int VB, int G>
__global__ void __launch_bounds__(256) combine_grad_kernel(Moves m, const T* __restrict__ dy, int64_t dy_stride,
                                                           const T* __restrict__ z, int64_t z_stride,
                                                           const void* __restrict__ weights, int weight_type,
                                                           T* __restrict__ dz, void* __restrict__ dw) {
    using V = Vec<T, VB>;
    constexpr int U = 4;
    __shared__ float part[8];
    const int64_t token = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (token >= m.tokens) return;  // G = 256: the whole block or none of it
    const uint32_t kept = kept_entries(m);
    const T* grow = dy + token * dy_stride;
    for (int k = 0; k < m.slots; ++k) {
        const int64_t e = token * m.slots + k;
        const uint32_t p = (uint32_t)m.position[e];
        const bool there = p < kept;
        const float w = weights && there ? rows::load_weight(weights, weight_type, e) : 1.0f;
        const T* zrow = z + (int64_t)p * z_stride;
        T* to = dz + (int64_t)p * m.width;
        float dot = 0.0f;
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
                            if (dw) dot = fmaf(gv, rows::to_float(a[u].v[i]), dot);
                            r.v[i] = rows::from_float<T>(w * gv);
                        }
                        r.store(to + c);
                    }
                }
            }
        } else if (p < (uint64_t)m.entries) {
            V r;
            r.zero();
            for (int64_t c = (threadIdx.x % G) * V::N; c < m.width; c += G * V::N) r.store(to + c);
        }
        if (dw) {
            constexpr int W = G < 32 ? G : 32;
            const unsigned lanes = G < 32 ? ((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G) : 0xffffffffu;
#pragma unroll
            for (int s = W / 2; s > 0; s >>= 1) dot += __shfl_xor_sync(lanes, dot, s);
            if (G == 256) {
                if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
                __syncthreads();
                dot = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) dot += part[i];
                __syncthreads();
            }
            if (threadIdx.x % G == 0) rows::store_weight(dw, weight_type, e, dot);
        }
    }
}

// Threads a token: 8 for rows of up to 8 vectors, else a warp; a block when the tokens are too few to
// fill the SMs with warps and a row has more than a warp's vectors.
inline int group_of(int64_t tokens, int64_t vectors) {
    if (vectors <= 8) return 8;
    if (tokens < 148 * 8 && vectors > 32) return 256;
    return 32;
}
template <typename F>
inline void for_group(int g, F&& f) {
    if (g == 8) f(rows::Bytes<8>{});
    else if (g == 32) f(rows::Bytes<32>{});
    else f(rows::Bytes<256>{});
}
inline unsigned blocks_of(int64_t tokens, int g) { return (unsigned)((tokens + 256 / g - 1) / (256 / g)); }

// Shapes and pointers that every move checks; HB_OK or the failure.
int check(const char* what, int type, int64_t tokens, int64_t slots, int64_t width, const void* position,
          const void* kept) {
    if (!rows::valid_type(type)) return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": unknown element type");
    if (tokens < 0 || slots < 1 || width < 0 || tokens > INT32_MAX / slots || width > INT32_MAX)
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": sizes out of range");
    if (tokens > 0 && width > 0 && (!position || !kept))
        return abi_fail(HB_BAD_ARGUMENT, std::string(what) + ": null pointer");
    return HB_OK;
}
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
    const int vb = rows::vector_bytes(rows::address_bits(x) | rows::address_bits(sorted) | (uint64_t)(x_stride * size) |
                                      (uint64_t)(width * size), type);
    const int g = group_of(tokens, width * size / vb);
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        for_group(g, [&](auto gg) {
            constexpr int G = decltype(gg)::value;
            dispatch_kernel<T, decltype(b)::value, G><<<blocks_of(tokens, G), 256, 0, static_cast<cudaStream_t>(stream)>>>(
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
    const int vb = rows::vector_bytes(rows::address_bits(z) | rows::address_bits(out) | (uint64_t)(z_stride * size) |
                                      (uint64_t)(width * size), type);
    const int g = group_of(tokens, width * size / vb);
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        for_group(g, [&](auto gg) {
            constexpr int G = decltype(gg)::value;
            combine_kernel<T, decltype(b)::value, G><<<blocks_of(tokens, G), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                m, static_cast<const T*>(z), z_stride, weights, weight_type, static_cast<T*>(out));
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
    const int vb = rows::vector_bytes(bits, type);
    const int g = group_of(tokens, width * size / vb);
    rows::for_type(type, vb, [&](auto t, auto b) {
        using T = decltype(t);
        for_group(g, [&](auto gg) {
            constexpr int G = decltype(gg)::value;
            combine_grad_kernel<T, decltype(b)::value, G>
                <<<blocks_of(tokens, G), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                    m, static_cast<const T*>(dy), dy_stride, static_cast<const T*>(z), z_stride, weights, weight_type,
                    static_cast<T*>(dz), dweights);
        });
    });
    return launched("route combine gradient");
}
