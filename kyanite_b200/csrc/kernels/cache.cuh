// How a cache lies in memory (CacheParams).  A row is one position of one head: its channels, padded to a multiple of 64, as f16
// or as whole numbers + 128 (the low byte of 1024 + 128 + q in f16, whence two instructions make f16 of two of them).  Keys, values
// and scales of 16 positions lie together, so that one bulk copy brings all that is needed of them.
//
// The 16-byte chunks of a row are written in an order that depends on the position, so that a tile copied to shared memory as
// it lies is read without bank conflicts both as the matrix instructions read keys (8 positions x 64 bytes) and as they
// read values (4 positions, 4 apart or so, x 32 bytes): kernels/cache_attention.cu.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../kernels.h"

namespace kn {

constexpr uint32_t kCacheZeros = 0x80808080u;   // four channels that are 0

// chunk j of position t lies where chunk j ^ cache_swizzle(.) would
__host__ __device__ __forceinline__ int cache_swizzle(int row_bytes, int t) {
    return row_bytes % 128 == 0 ? (((t >> 2) & 3) << 1) ^ ((t & 1) << 2) : ((t >> 3) & 1) << 1;
}
// The first byte of the tile that position t is in: keys, values, then, of an i8 cache, the keys' scales and the values'
__host__ __device__ __forceinline__ uint8_t* cache_tile(const CacheParams& c, int64_t head /* of all sequences */, int t) {
    return c.base + (head * c.tiles + (t >> 4)) * c.tile_bytes;
}

}  // namespace kn
