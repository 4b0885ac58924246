// A decoder's cache: writing the keys and values of new tokens into it, and reading all of it back as numbers.
//
//   scale = max_d |x_d| / 127,   q_d = round(x_d / scale)  (half to even),   read back as q_d * scale
//
// per position and head, in f32 with IEEE divisions, so that any other program gets the same q and scale.  A row that holds an
// infinity or a NaN reads back as NaN throughout (its scale is NaN).
//
// Both are bound by memory: 8 channels a thread, so that a row's loads and stores are 16 bytes wide, and several rows a thread
// in flight.
#include "cache.cuh"
#include "launch.cuh"

namespace kn {

int64_t cache_bytes(const CacheParams& c) { return (int64_t)c.seqs * c.heads * c.tiles * c.tile_bytes; }

CacheParams cache_params(int64_t seqs, int64_t heads, int64_t capacity, int64_t dim, DType dtype) {
    CacheParams c{};
    c.half = dtype == DType::F16;
    c.seqs = (int32_t)seqs, c.heads = (int32_t)heads, c.capacity = (int32_t)capacity, c.dim = (int32_t)dim;
    c.tiles = (int32_t)((capacity + kCacheTile - 1) / kCacheTile);
    c.row_bytes = (int32_t)((dim + 63) / 64 * 64) * (c.half ? 2 : 1);
    c.tile_bytes = 2 * kCacheTile * c.row_bytes + (c.half ? 0 : 2 * kCacheTile * 4);
    return c;
}

int cache_clear_async(const CacheParams& c, cudaStream_t stream) {
    const size_t rows = 2 * kCacheTile * (size_t)c.row_bytes, bytes = (size_t)cache_bytes(c);
    cudaError_t e = cudaMemsetAsync(c.base, c.half ? 0 : (int)(kCacheZeros & 0xff), bytes, stream);
    if (e == cudaSuccess && !c.half) e = cudaMemset2DAsync(c.base + rows, (size_t)c.tile_bytes, 0, (size_t)c.tile_bytes - rows, bytes / c.tile_bytes, stream);
    return (int)e;
}

namespace {

// What a thread holds of a row: channels d .. d + 7
struct Eight {
    float x[8];
};

template <typename T, bool VEC>
__device__ __forceinline__ Eight load_eight(const T* row, int64_t stride, int d, int dim) {
    Eight e;
    if constexpr (VEC && sizeof(T) == 2) {
        const uint4 raw = d < dim ? *(const uint4*)(row + d) : make_uint4(0, 0, 0, 0);
        const __half2* h = (const __half2*)&raw;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            e.x[2 * i] = f.x, e.x[2 * i + 1] = f.y;
        }
    } else if constexpr (VEC) {
        const float4 zero = make_float4(0, 0, 0, 0);
        const float4 a = d < dim ? *(const float4*)(row + d) : zero, b = d < dim ? *(const float4*)(row + d + 4) : zero;
        e.x[0] = a.x, e.x[1] = a.y, e.x[2] = a.z, e.x[3] = a.w, e.x[4] = b.x, e.x[5] = b.y, e.x[6] = b.z, e.x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) e.x[i] = d + i < dim ? (float)row[(d + i) * stride] : 0.f;
    }
    return e;
}

// THREADS threads a row (8 channels each).  VEC: rows whose channels are contiguous, 16-byte aligned and a multiple of 8
template <typename T, bool VEC, int THREADS>
__global__ void __launch_bounds__(256) cache_write_kernel(const __grid_constant__ CacheWriteParams p) {
    pdl_enter();
    const CacheParams& c = p.cache;
    const int d = (threadIdx.x % THREADS) * 8;
    const int64_t per_part = (int64_t)c.seqs * p.tokens * c.heads;
    const int64_t rows = 2 * per_part, step = (int64_t)gridDim.x * (256 / THREADS);
    // (all threads of a row go round as often as each other: they exchange the maximum)
    for (int64_t r = (int64_t)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS; r - threadIdx.x / THREADS < rows; r += step) {
        const bool live = r < rows;
        const int64_t at = live ? r : rows - 1;
        const int part = at >= per_part;
        const int64_t token = (at - part * per_part) / c.heads;
        const int h = (int)((at - part * per_part) - token * c.heads);
        const int64_t s = token / p.tokens;
        const int t = (int)(token - s * p.tokens);
        const int64_t position = (int64_t)p.start[s] + t;
        const bool keep = live && position >= 0 && position < c.capacity && (p.count == nullptr || t < p.count[s]);
        const T* row = (const T*)p.in[part] + s * p.strides[part][0] + t * p.strides[part][1] + h * p.strides[part][2];
        const Eight e = load_eight<T, VEC>(row, p.strides[part][3], d, c.dim);
        const int64_t head = s * c.heads + h;
        uint8_t* out = cache_row(c, part, head, keep ? (int)position : 0);
        if (c.half) {
            __half2 q[4];
#pragma unroll
            for (int i = 0; i < 4; i++) q[i] = __floats2half2_rn(e.x[2 * i], e.x[2 * i + 1]);
            if (keep && d < c.dim) *(uint4*)(out + (((d >> 3) ^ cache_swizzle(c.row_bytes, (int)position)) << 4)) = *(uint4*)q;
            continue;
        }
        float most = 0.f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            most = fmaxf(most, fabsf(e.x[i]));
            nan = nan || e.x[i] != e.x[i];
        }
        if (nan) most = __int_as_float(0x7f800000);
#pragma unroll
        for (int o = THREADS / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float scale = most < __int_as_float(0x7f800000) ? __fdiv_rn(most, 127.f) : __int_as_float(0x7fc00000);
        uint32_t q[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // (a scale of few bits, of numbers next to nothing, may give more than 127)
            const float y = scale > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(e.x[i], scale)), -127.f), 127.f) : 0.f;
            q[i >> 2] |= (uint32_t)((int)y + 128) << (8 * (i & 3));
        }
        if (keep && d < c.dim) *(uint2*)(out + (((d >> 4) ^ cache_swizzle(c.row_bytes, (int)position)) << 4) + (d & 8)) = make_uint2(q[0], q[1]);
        if (keep && d == 0) *cache_scale(c, part, head, (int)position) = scale;
    }
}

template <typename T, bool VEC, int THREADS>
__global__ void __launch_bounds__(256) cache_read_kernel(const __grid_constant__ CacheReadParams p) {
    pdl_enter();
    const CacheParams& c = p.cache;
    constexpr int kRows = 256 / THREADS, kEach = 4;
    const int d = (threadIdx.x % THREADS) * 8;
    if (d >= c.dim) return;
    const int t0 = blockIdx.x * kRows * kEach + threadIdx.x / THREADS;
    const int64_t heads = (int64_t)c.seqs * c.heads;
    for (int64_t both = blockIdx.y; both < 2 * heads; both += gridDim.y) {   // part and head
        const int part = both >= heads;
        const int64_t head = both - part * heads;
        uint4 raw[kEach];
        float scale[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int t = t0 + i * kRows;
            const int from = min(t, c.capacity - 1), x = cache_swizzle(c.row_bytes, from);
            const uint8_t* in = cache_row(c, part, head, from);
            if (c.half) {
                raw[i] = *(const uint4*)(in + (((d >> 3) ^ x) << 4));
            } else {
                *(uint2*)&raw[i] = *(const uint2*)(in + (((d >> 4) ^ x) << 4) + (d & 8));
                scale[i] = *cache_scale(c, part, head, from);
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int t = t0 + i * kRows;
            if (t >= c.capacity) break;
            float x[8];
            if (c.half) {
                const __half* h = (const __half*)&raw[i];
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = __half2float(h[k]);
            } else {
                const uint8_t* q = (const uint8_t*)&raw[i];
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = (float)((int)q[k] - 128) * scale[i];
            }
            T* out = (T*)p.out + (both * c.capacity + t) * c.dim + d;
            if constexpr (VEC && sizeof(T) == 2) {
                __half2 y[4];
#pragma unroll
                for (int k = 0; k < 4; k++) y[k] = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
                *(uint4*)out = *(uint4*)y;
            } else if constexpr (VEC) {
                *(float4*)out = make_float4(x[0], x[1], x[2], x[3]);
                *(float4*)(out + 4) = make_float4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (d + k < c.dim) out[k] = (T)x[k];
            }
        }
    }
}

template <typename T, bool VEC>
void write_threads(const CacheWriteParams& p, cudaStream_t stream) {
    const int threads = p.cache.dim <= 64 ? 8 : p.cache.dim <= 128 ? 16 : 32;
    const int64_t rows = 2ll * p.cache.seqs * p.tokens * p.cache.heads, per_block = 256 / threads;
    const dim3 grid((unsigned)std::min<int64_t>((rows + per_block - 1) / per_block, 148 * 16));
    if (threads == 8) launch_pdl(cache_write_kernel<T, VEC, 8>, grid, dim3(256), 0, stream, p);
    if (threads == 16) launch_pdl(cache_write_kernel<T, VEC, 16>, grid, dim3(256), 0, stream, p);
    if (threads == 32) launch_pdl(cache_write_kernel<T, VEC, 32>, grid, dim3(256), 0, stream, p);
}

template <typename T, bool VEC>
void read_threads(const CacheReadParams& p, cudaStream_t stream) {
    const int threads = p.cache.dim <= 64 ? 8 : p.cache.dim <= 128 ? 16 : 32;
    const int per_block = 4 * 256 / threads;
    const dim3 grid((unsigned)((p.cache.capacity + per_block - 1) / per_block), (unsigned)std::min<int64_t>(2ll * p.cache.seqs * p.cache.heads, 65535));
    if (threads == 8) launch_pdl(cache_read_kernel<T, VEC, 8>, grid, dim3(256), 0, stream, p);
    if (threads == 16) launch_pdl(cache_read_kernel<T, VEC, 16>, grid, dim3(256), 0, stream, p);
    if (threads == 32) launch_pdl(cache_read_kernel<T, VEC, 32>, grid, dim3(256), 0, stream, p);
}

}  // namespace

int launch_cache_write(const CacheWriteParams& p, cudaStream_t stream) {
    const int unit = p.half ? 8 : 4;   // elements of 16 bytes
    bool vec = p.cache.dim % 8 == 0;
    for (int k = 0; k < 2; k++) {
        vec = vec && p.strides[k][3] == 1 && (uintptr_t)p.in[k] % 16 == 0;
        for (int i = 0; i < 3; i++) vec = vec && p.strides[k][i] % unit == 0;
    }
    if (p.half) vec ? write_threads<__half, true>(p, stream) : write_threads<__half, false>(p, stream);
    else vec ? write_threads<float, true>(p, stream) : write_threads<float, false>(p, stream);
    return (int)cudaGetLastError();
}

int launch_cache_read(const CacheReadParams& p, cudaStream_t stream) {
    const bool vec = p.cache.dim % 8 == 0 && (uintptr_t)p.out % 16 == 0;
    if (p.half) vec ? read_threads<__half, true>(p, stream) : read_threads<__half, false>(p, stream);
    else vec ? read_threads<float, true>(p, stream) : read_threads<float, false>(p, stream);
    return (int)cudaGetLastError();
}

}  // namespace kn
