// Rows of 32- and 16-bit floating types as vectors of 2 to 16 bytes: what the
// routing, lookup and clipping kernels load and store.  Arithmetic is always
// fp32; a value is rounded once, when it is stored.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/hello_b200.h"

namespace hb {
namespace rows {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

template <int BYTES> struct Bits;
template <> struct Bits<16> { using type = uint4; };
template <> struct Bits<8> { using type = uint2; };
template <> struct Bits<4> { using type = uint32_t; };
template <> struct Bits<2> { using type = uint16_t; };
template <> struct Bits<1> { using type = uint8_t; };  // 8-bit codes alone

// BYTES of T at an address aligned to BYTES.
template <typename T, int BYTES>
struct Vec {
    static constexpr int N = BYTES / (int)sizeof(T);
    using Raw = typename Bits<BYTES>::type;
    union {
        Raw raw;
        T v[N];
    };
    __device__ __forceinline__ Vec() {}
    __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const Raw*>(p)); }
    __device__ __forceinline__ void load_once(const T* p) { raw = __ldcs(reinterpret_cast<const Raw*>(p)); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
    // first to leave L2: rows that nothing of this kernel reads again, so that those it does read stay
    __device__ __forceinline__ void store_once(T* p) const { __stcs(reinterpret_cast<Raw*>(p), raw); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = from_float<T>(0.0f);
    }
};

// A weight of any of the three types.
__device__ __forceinline__ float load_weight(const void* w, int type, int64_t i) {
    if (type == HB_F32) return static_cast<const float*>(w)[i];
    if (type == HB_F16) return __half2float(static_cast<const __half*>(w)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}
__device__ __forceinline__ void store_weight(void* w, int type, int64_t i, float v) {
    if (type == HB_F32) static_cast<float*>(w)[i] = v;
    else if (type == HB_F16) static_cast<__half*>(w)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(v);
}

inline bool valid_type(int t) { return t == HB_F32 || t == HB_F16 || t == HB_BF16; }
inline int type_bytes(int t) { return t == HB_F32 ? 4 : 2; }

// Widest vector (16, 8, 4 or 2 bytes) that every row of every given array
// allows: base addresses and row strides in bytes or-ed together.
inline int vector_bytes(uint64_t bits, int type) {
    for (int b = 16; b > type_bytes(type); b >>= 1)
        if (bits % (uint64_t)b == 0) return b;
    return type_bytes(type);
}
inline uint64_t address_bits(const void* p) { return (uint64_t)(uintptr_t)p; }

// Calls f with a value of the element type and the vector size as an integral constant.
template <int B> struct Bytes { static constexpr int value = B; };
template <typename F>
inline void for_type(int type, int vb, F&& f) {
    if (type == HB_F32) {
        if (vb == 16) f(float{}, Bytes<16>{});
        else if (vb == 8) f(float{}, Bytes<8>{});
        else f(float{}, Bytes<4>{});
    } else if (type == HB_F16) {
        if (vb == 16) f(__half{}, Bytes<16>{});
        else if (vb == 8) f(__half{}, Bytes<8>{});
        else if (vb == 4) f(__half{}, Bytes<4>{});
        else f(__half{}, Bytes<2>{});
    } else {
        if (vb == 16) f(__nv_bfloat16{}, Bytes<16>{});
        else if (vb == 8) f(__nv_bfloat16{}, Bytes<8>{});
        else if (vb == 4) f(__nv_bfloat16{}, Bytes<4>{});
        else f(__nv_bfloat16{}, Bytes<2>{});
    }
}

}  // namespace rows
}  // namespace hb
