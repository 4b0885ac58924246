// Attention of new tokens against a decoder's cache.
//
//   p = prefix length + start[s] + t,   score_j = scale q . k_j,   cap tanh(score / cap),   - slope (p - j),
//   out = sum_j softmax(score)_j v_j   over   0 <= p - j < window
//
// One warp a row (a token's head): keys one after the other with the running maximum and sum of the softmax.
#include "cache.cuh"
#include "launch.cuh"

namespace kn {

CacheAttentionPlan cache_attention_plan(const CacheAttentionParams& p) {
    const int64_t rows = (int64_t)p.cache.seqs * p.tokens * p.heads;
    return {(int32_t)std::min<int64_t>((rows + 7) / 8, 1 << 20), 0, 0};
}

namespace {

template <typename T>
__global__ void __launch_bounds__(256) cache_attention_kernel(const __grid_constant__ CacheAttentionParams p) {
    pdl_enter();
    const int lane = threadIdx.x & 31, dim = p.cache.dim, group = p.heads / p.cache.heads;
    const int64_t rows = (int64_t)p.cache.seqs * p.tokens * p.heads;
    for (int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; r < rows; r += (int64_t)gridDim.x * 8) {
        const int h = (int)(r % p.heads);
        const int t = (int)(r / p.heads % p.tokens);
        const int64_t s = r / p.heads / p.tokens;
        const T* q = (const T*)p.query + s * p.q_strides[0] + t * p.q_strides[1] + h * p.q_strides[2];
        float qv[8], o[8] = {};
#pragma unroll
        for (int i = 0; i < 8; i++) qv[i] = lane + 32 * i < dim ? (float)q[(lane + 32 * i) * p.q_strides[3]] : 0.f;
        const int64_t shared = p.prefix.base ? min(max(*p.prefix_length, 0), p.prefix.capacity) : 0;
        const int64_t at = (int64_t)p.start[s] + t, position = shared + at;
        const bool live = at >= 0 && (p.count == nullptr || t < p.count[s]);
        const int64_t end = live ? min(position + 1, shared + p.cache.capacity) : 0;
        const int64_t first = p.window > 0 ? max(position - p.window + 1, (int64_t)0) : 0;
        float m = -INFINITY, l = 0.f;
        for (int64_t j = first; j < end; j++) {
            const CacheParams& c = j < shared ? p.prefix : p.cache;
            const int64_t key = j < shared ? j : j - shared, seq = j < shared ? 0 : s;
            float score = 0.f, v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int d = lane + 32 * i;
                v[i] = 0.f;
                if (d >= dim) continue;
                const int64_t kr = cache_row(c, 0, seq, h / group, key), vr = cache_row(c, 1, seq, h / group, key);
                const int x = cache_swizzle(c.row_bytes, (int)key);
                if (c.half) {
                    const int byte = (((d >> 3) ^ x) << 4) + 2 * (d & 7);
                    score += qv[i] * __half2float(*(const __half*)(c.base + kr * c.row_bytes + byte));
                    v[i] = __half2float(*(const __half*)(c.base + vr * c.row_bytes + byte));
                } else {
                    const int byte = (((d >> 4) ^ x) << 4) + (d & 15);
                    score += qv[i] * ((float)((int)c.base[kr * c.row_bytes + byte] - 128) * c.scales[kr]);
                    v[i] = (float)((int)c.base[vr * c.row_bytes + byte] - 128) * c.scales[vr];
                }
            }
#pragma unroll
            for (int n = 16; n > 0; n >>= 1) score += __shfl_xor_sync(0xffffffffu, score, n);
            score *= p.scale;
            if (p.softcap > 0.f) score = p.softcap * tanhf(score / p.softcap);
            if (p.slopes) score -= p.slopes[h] * (float)(position - j);
            const float most = fmaxf(m, score), base = most == -INFINITY ? 0.f : most;
            const float keep = expf(m - base), e = expf(score - base);
            l = l * keep + e;
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = o[i] * keep + e * v[i];
            m = most;
        }
        T* out = (T*)p.out + r * dim;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (lane + 32 * i < dim) out[lane + 32 * i] = (T)(first < end ? o[i] / l : 0.f);
    }
}

}  // namespace

int launch_cache_attention(const CacheAttentionParams& p, cudaStream_t stream) {
    if (p.half) launch_pdl(cache_attention_kernel<__half>, dim3(p.grid), dim3(256), 0, stream, p);
    else launch_pdl(cache_attention_kernel<float>, dim3(p.grid), dim3(256), 0, stream, p);
    return (int)cudaGetLastError();
}

}  // namespace kn
