// Stable sort of entries by a small integer key (index_sort.cu).
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace hb {

// Launches in a row whose later ones start while the earlier ones end (programmatic dependent launch).  A kernel
// lets the next one of the row start with allow_next(), and calls after_last() before it reads what earlier ones
// of the row wrote, or writes what they read; after_last() returns when the kernel before has ended and its
// writes are there, and that one waited for its own.  The first kernel of a row is launched plainly, so
// before after_last() everything older than the row is done.  What a row's earlier kernels write is read by plain loads
// from pointers without __restrict__: it is not constant for the whole of a later kernel.
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
inline cudaError_t launch_next(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = st;
    config.attrs = &attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

// Entries i = 0..n-1 with key index[i] when 0 <= index[i] < bins and key `bins`
// otherwise, sorted by key, equal keys in entry order.  Any output may be null:
// order (n, entry of each place), position (n, place of each entry), pairs (n,
// (key, entry) of each place), offsets (bins + 1, first place of a key not below it; offsets[bins] is
// the number of entries with a valid index).  `zeros` words at `zero` are set to 0 on the
// way (n > 0).  The last kernel calls allow_next().  Returns 0, or an HB_* code.
size_t index_sort_bytes(int64_t n, int64_t bins);
int index_sort(const void* index, int index_bytes, int64_t n, int64_t bins, int32_t* order, int32_t* position,
               uint2* pairs, int32_t* offsets, void* ws, size_t ws_bytes, cudaStream_t st,
               uint32_t* zero = nullptr, int64_t zeros = 0);

}  // namespace hb
