// A decoder's cache: writing the keys and values of new tokens into it, and reading all of it back as numbers.
//
//   scale = max_d |x_d| * (1/127),   q_d = round(x_d / scale)  (half to even),   read back as q_d * scale
//
// per position and head, in f32 with each operation and the constant rounded to nearest, so that any other program gets the same q and scale.
// (Not max / 127: what divides by a number that it knows beforehand multiplies, as tensor programs do, and one step of the scale moves the
// numbers next to a half.)  A row that holds an
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

// Four numbers + 128 in a word: round(x / scale), of the quotient that IEEE division gives.  With r = 1 / scale rounded to nearest, y = x r
// and y + r (x - y scale), both in one rounding, is that quotient (Markstein 1990; scales next to either end of the range, and the one
// mantissa of all ones, for which r may be off, divide).  Adding 1.5 x 2^23 rounds it half to even and leaves it in the low byte.
__device__ __forceinline__ uint32_t low_bytes(const float (&y)[4]) {
    uint32_t b[4];
#pragma unroll
    for (int k = 0; k < 4; k++) b[k] = __float_as_uint(__fadd_rn(y[k], 12582912.f + 128.f));
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t four_of(const float* x, float scale, float r) {
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        y[k] = x[k] * r;
        y[k] = fmaf(fmaf(-y[k], scale, x[k]), r, y[k]);
    }
    return low_bytes(y);
}
// Rows for which that does not hold: the scale and eight numbers.  (A scale of few bits, of numbers next to nothing, may give more than 127)
__device__ __noinline__ uint2 divided(const float* x, float most, float* scale) {
    *scale = most < __int_as_float(0x7f800000) ? __fmul_rn(most, 1.f / 127.f) : __int_as_float(0x7fc00000);
    float y[8];
#pragma unroll 1
    for (int k = 0; k < 8; k++) y[k] = *scale > 0.f ? fminf(fmaxf(__fdiv_rn(x[k], *scale), -127.f), 127.f) : 0.f;
    const float lo[4] = {y[0], y[1], y[2], y[3]}, hi[4] = {y[4], y[5], y[6], y[7]};
    return make_uint2(low_bytes(lo), low_bytes(hi));
}

// THREADS threads a row (8 channels each), kEach rows a thread with their loads in flight together.  VEC: rows whose channels are
// contiguous, 16-byte aligned and a multiple of 8.  A block takes positions of one head (and writes whole tiles), of few tokens heads of one
// position (and reads what lies together).  7 prompts of up to 1500 tokens, 32 heads of 128 channels, f32 into i8 (270 MB): bound by
// instructions while every row found its place by divisions and every number was divided (149 us); now 64 us.  Along the positions from
// 16 tokens on (step alone, 32 heads of 128 channels, f16 into i8, along the positions / across the heads): 7 prompts of up to 1500 tokens 78.6 /
// 94.8 us, 16 sequences x 64 9.6 / 10.6, 16 x 16 5.6 / 4.4, 32 x 4 7.7 / 4.2, 32 x 1 8.6 / 3.0.
template <typename T, bool VEC, int THREADS>
__global__ void __launch_bounds__(256) cache_write_kernel(const __grid_constant__ CacheWriteParams p) {
    pdl_enter();
    constexpr int kRows = 256 / THREADS, kEach = 4;
    const CacheParams& c = p.cache;
    const int d = (threadIdx.x % THREADS) * 8;
    const bool along = p.tokens >= 16;   // along the positions
    const int inner = along ? p.tokens : c.heads, outer = along ? c.heads : p.tokens;
    const int first = blockIdx.x * (kRows * kEach) + threadIdx.x / THREADS;
    for (int y = blockIdx.y; y < 2 * c.seqs * outer; y += gridDim.y) {
        const int part = y >= c.seqs * outer, rest = y - part * c.seqs * outer, s = rest / outer, fixed = rest - s * outer;
        const int64_t start = p.start[s];
        const int count = p.count != nullptr ? p.count[s] : p.tokens;
        const T* in = (const T*)p.in[part] + s * p.strides[part][0] + fixed * p.strides[part][along ? 2 : 1];
        const int64_t stride = p.strides[part][along ? 1 : 2], head_bytes = (int64_t)c.tiles * c.tile_bytes;
        uint8_t* const tiles = c.base + ((int64_t)s * c.heads + (along ? fixed : 0)) * head_bytes;
        Eight e[kEach];
        int position[kEach];   // -1: not written
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int r = first + i * kRows, t = along ? r : fixed;
            const int64_t at = start + t;
            position[i] = r < inner && t < count && at >= 0 && at < c.capacity ? (int)at : -1;
            e[i] = position[i] >= 0 ? load_eight<T, VEC>(in + r * stride, p.strides[part][3], d, c.dim) : Eight{};
        }
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            if (!__any_sync(0xffffffffu, position[i] >= 0)) continue;
            const int t = max(position[i], 0), x = cache_swizzle(c.row_bytes, t);
            uint8_t* const tile = tiles + (along ? 0 : (first + i * kRows) * head_bytes) + (int64_t)(t >> 4) * c.tile_bytes;
            uint8_t* const out = tile + (part * kCacheTile + (t & 15)) * c.row_bytes;
            const bool keep = position[i] >= 0 && d < c.dim;
            if (c.half) {
                __half2 q[4];
#pragma unroll
                for (int k = 0; k < 4; k++) q[k] = __floats2half2_rn(e[i].x[2 * k], e[i].x[2 * k + 1]);
                if (keep) *(uint4*)(out + (((d >> 3) ^ x) << 4)) = *(uint4*)q;
                continue;
            }
            uint32_t most = 0;   // the largest magnitude as bits, a NaN above all others
#pragma unroll
            for (int k = 0; k < 8; k++) most = max(most, __float_as_uint(e[i].x[k]) & 0x7fffffffu);
#pragma unroll
            for (int o = THREADS / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float top = __uint_as_float(most);
            float scale = __fmul_rn(top, 1.f / 127.f);
            uint2 q;
            if (!(top > 1e-28f && top < 1e30f) || (__float_as_uint(scale) & 0x7fffffu) == 0x7fffffu) {
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; k++) y[k] = e[i].x[k];
                q = divided(y, top, &scale);
            } else {
                const float inverse = __frcp_rn(scale);
                q = make_uint2(four_of(e[i].x, scale, inverse), four_of(e[i].x + 4, scale, inverse));
            }
            if (keep) *(uint2*)(out + (((d >> 4) ^ x) << 4) + (d & 8)) = q;
            if (keep && d == 0) ((float*)(tile + 2 * kCacheTile * c.row_bytes))[part * kCacheTile + (t & 15)] = scale;
        }
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
        const uint8_t* const tiles = c.base + head * ((int64_t)c.tiles * c.tile_bytes);
        T* const rows = (T*)p.out + both * c.capacity * c.dim + d;
        uint4 raw[kEach];
        float scale[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int t = min(t0 + i * kRows, c.capacity - 1), x = cache_swizzle(c.row_bytes, t);
            const uint8_t* const tile = tiles + (int64_t)(t >> 4) * c.tile_bytes;
            const uint8_t* const in = tile + (part * kCacheTile + (t & 15)) * c.row_bytes;
            if (c.half) {
                raw[i] = *(const uint4*)(in + (((d >> 3) ^ x) << 4));
            } else {
                *(uint2*)&raw[i] = *(const uint2*)(in + (((d >> 4) ^ x) << 4) + (d & 8));
                scale[i] = ((const float*)(tile + 2 * kCacheTile * c.row_bytes))[part * kCacheTile + (t & 15)];
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int t = t0 + i * kRows;
            if (t >= c.capacity) break;
            float x[8];
            if (c.half) {
                const __half2* h = (const __half2*)&raw[i];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float2 f = __half22float2(h[k]);
                    x[2 * k] = f.x, x[2 * k + 1] = f.y;
                }
            } else {
                const uint32_t* q = (const uint32_t*)&raw[i];
#pragma unroll
                for (int k = 0; k < 8; k++)   // 2^23 + byte, as it is in f32
                    x[k] = (__uint_as_float(__byte_perm(q[k >> 2], 0x4b000000u, 0x7440 + (k & 3))) - (8388608.f + 128.f)) * scale[i];
            }
            T* const out = rows + (int64_t)t * c.dim;
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
    const bool along = p.tokens >= 16;
    const int per_block = 4 * 256 / threads, inner = along ? p.tokens : p.cache.heads;
    const int64_t outer = 2ll * p.cache.seqs * (along ? p.cache.heads : p.tokens);
    const dim3 grid((unsigned)((inner + per_block - 1) / per_block), (unsigned)std::min<int64_t>(outer, 65535));
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
