// Stable sort of entries by a small integer key (index_sort.cu).
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace hb {

// Entries i = 0..n-1 with key index[i] when 0 <= index[i] < bins and key `bins`
// otherwise, sorted by key, equal keys in entry order.  Any output may be null:
// order (n, entry of each place), position (n, place of each entry), keys (n,
// sorted), offsets (bins + 1, first place of a key not below it; offsets[bins] is
// the number of entries with a valid index).  `zeros` words at `zero` are set to 0 on the
// way (n > 0).  Returns 0, or an HB_* code.
size_t index_sort_bytes(int64_t n, int64_t bins);
int index_sort(const void* index, int index_bytes, int64_t n, int64_t bins, int32_t* order, int32_t* position,
               uint32_t* keys, int32_t* offsets, void* ws, size_t ws_bytes, cudaStream_t st,
               uint32_t* zero = nullptr, int64_t zeros = 0);

}  // namespace hb
