// How a cache's rows lie in memory (CacheParams).  A row is one position of one head: its channels, padded to a multiple of 64,
// as f16 or as whole numbers + 128 (the low byte of 1024 + 128 + q in f16, whence two instructions make f16 of two of them).
//
// The 16-byte chunks of a row are written in an order that depends on the position, so that 16 rows copied to shared memory as
// they lie are read without bank conflicts both as the matrix instructions read keys (8 positions x 64 bytes) and as they
// read values (4 positions, 4 apart or so, x 32 bytes): kernels/cache_attention.cu.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cuda_runtime.h>

#include "../kernels.h"

namespace kn {

constexpr uint32_t kCacheZeros = 0x80808080u;   // four channels that are 0

// chunk j of position t lies where chunk j ^ cache_swizzle(.) would
__host__ __device__ __forceinline__ int cache_swizzle(int row_bytes, int t) {
    return row_bytes % 128 == 0 ? (((t >> 2) & 3) << 1) ^ ((t & 1) << 2) : ((t >> 3) & 1) << 1;
}
__host__ __device__ __forceinline__ int64_t cache_row(const CacheParams& c, int part, int64_t seq, int64_t head, int64_t t) {
    return part * c.part_rows + (seq * c.heads + head) * c.padded + t;
}

}  // namespace kn
