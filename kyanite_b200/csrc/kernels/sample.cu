// One token for every row of logits, by temperature, top-k, top-p and min-p and a given random number.
//
// A token's weight exp((x - max) / T) is counted in whole steps of 2^-44 of the highest, from f64: sums of whole numbers are the
// same in any order.  What stays after top-k and top-p is the head of one order (falling logits, rising index among equals), so
// each is a cut: a key (the logit's bits in the order of whole numbers) and, among equal keys, an index.  A cut is found by
// eight bits of the key at a time, from counts or weights per value of them.
//
// One CTA a row.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../kernels.h"
#include "launch.cuh"

namespace kn {

namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024;

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T>
struct Row {
    const T* at;
    int64_t stride;
    float most;
    double inverse;   // 1 / temperature
    __device__ float logit(int i) const {
        const float x = (float)at[i * stride] + 0.f;   // (-0 + 0 = 0: equal logits have equal keys)
        return x != x ? -INFINITY : x;
    }
    __device__ u64 weight(float x) const {
        if (x == most) return 1ull << 44;
        if (x == -INFINITY || most == INFINITY) return 0;   // (also at an infinite temperature)
        return (u64)__double2ll_rn(exp(((double)x - (double)most) * inverse) * 17592186044416.0);
    }
};

// What stays: keys above `key`, and of those equal to it the indexes up to `index`
struct Cut {
    uint32_t key;
    int index;
    __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
};

template <typename V, typename F>
__device__ V block_reduce(V v, V* shared, F f) {   // to all threads
    const int lane = threadIdx.x & 31;
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = shared[lane];
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Sum of v over the threads in front of this one
__device__ u64 block_before(u64 v, u64* shared) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 up = v;
    for (int o = 1; o < 32; o <<= 1) {
        const u64 w = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += w;
    }
    __syncthreads();
    if (lane == 31) shared[warp] = up;
    __syncthreads();
    u64 front = 0;
    for (int w = 0; w < warp; w++) front += shared[w];
    return front + up - v;
}

struct Shared {
    u64 bins[256], scratch[32];
    float floats[32];
    int found;
    u64 before;
    int index;
};

// The shortest head of the order, within `within`, whose measure (amount(x) summed) reaches `goal` (1 or more)
template <typename T, typename A>
__device__ Cut find_cut(const Row<T>& row, int vocab, Cut within, u64 goal, A amount, Shared& sh) {
    uint32_t prefix = 0;
    u64 before = 0;   // measure of all keys above the ones that are left
    for (int shift = 24; shift >= 0; shift -= 8) {
        const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
        __syncthreads();
        if (threadIdx.x < 256) sh.bins[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < vocab; i += kThreads) {
            const float x = row.logit(i);
            const uint32_t k = key_of(x);
            if ((k & mask) == (prefix & mask) && within.keeps(k, i)) atomicAdd(&sh.bins[(k >> shift) & 255], amount(x));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 sum = before;
            int b = 255, last = -1;
            for (; b >= 0; b--) {
                if (sh.bins[b] == 0) continue;
                last = b;
                if (sum + sh.bins[b] >= goal) break;
                sum += sh.bins[b];
            }
            if (b < 0) b = last < 0 ? 0 : last, sum -= last < 0 ? 0 : sh.bins[last];   // (never, for a goal that all reach)
            sh.found = b;
            sh.before = sum;
        }
        __syncthreads();
        prefix |= (uint32_t)sh.found << shift;
        before = sh.before;
    }
    // of the equal keys the first so many
    u64 each = 0;
    int mine = 0;
    const int chunk = (vocab + kThreads - 1) / kThreads, from = threadIdx.x * chunk, until = min(vocab, from + chunk);
    for (int i = from; i < until; i++) {
        const float x = row.logit(i);
        if (key_of(x) == prefix && within.keeps(prefix, i)) mine++, each = amount(x);
    }
    each = block_reduce(each, sh.scratch, [](u64 a, u64 b) { return a > b ? a : b; });
    const u64 need = goal > before && each > 0 ? (goal - before + each - 1) / each : 1;
    const u64 front = block_before((u64)mine, sh.scratch);
    __syncthreads();
    if (threadIdx.x == 0) sh.index = vocab;
    __syncthreads();
    if (front < need && need <= front + mine) {
        u64 n = front;
        for (int i = from; i < until; i++)
            if (key_of(row.logit(i)) == prefix && within.keeps(prefix, i) && ++n == need) sh.index = i;
    }
    __syncthreads();
    return Cut{prefix, sh.index};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleParams p) {
    pdl_enter();
    __shared__ Shared sh;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        Row<T> row{(const T*)p.logits + r * p.row_stride, p.col_stride, 0.f, 0.0};
        const int vocab = p.vocab;
        const auto larger = [](float a, float b) { return fmaxf(a, b); };
        const auto sum = [](u64 a, u64 b) { return a + b; };
        const auto least = [](u64 a, u64 b) { return a < b ? a : b; };
        float most = -INFINITY;
        for (int i = threadIdx.x; i < vocab; i += kThreads) most = fmaxf(most, row.logit(i));
        row.most = most = block_reduce(most, sh.floats, larger);
        u64 first = ~0ull;
        for (int i = threadIdx.x; i < vocab; i += kThreads)
            if (row.logit(i) == most) first = first < (u64)i ? first : (u64)i;
        first = block_reduce(first, sh.scratch, least);
        const float temperature = p.temperature ? p.temperature[r] : 1.f;
        if (most == -INFINITY || !(temperature > 0.f)) {
            if (threadIdx.x == 0) p.out[r] = most == -INFINITY ? -1 : (int)first;
            __syncthreads();
            continue;
        }
        row.inverse = 1.0 / (double)temperature;
        Cut cut{0, vocab};
        const auto weight = [&](float x) { return row.weight(x); };
        const int k = p.top_k ? p.top_k[r] : 0;
        if (k > 0 && k < vocab) cut = find_cut(row, vocab, cut, (u64)k, [](float) { return 1ull; }, sh);
        if (p.top_p && !(p.top_p[r] >= 1.f)) {
            u64 mass = 0;
            for (int i = threadIdx.x; i < vocab; i += kThreads) {
                const float x = row.logit(i);
                if (cut.keeps(key_of(x), i)) mass += weight(x);
            }
            mass = block_reduce(mass, sh.scratch, sum);
            const double goal = ceil((double)p.top_p[r] * (double)mass);
            cut = find_cut(row, vocab, cut, goal >= 1.0 ? (u64)goal : 1ull, weight, sh);
        }
        const double least_weight = p.min_p ? (double)p.min_p[r] * 17592186044416.0 : 0.0;
        const auto stays = [&](float x, int i, u64 w) { return (u64)i == first || (cut.keeps(key_of(x), i) && (double)w >= least_weight); };
        u64 mass = 0;
        const int chunk = (vocab + kThreads - 1) / kThreads, from = threadIdx.x * chunk, until = min(vocab, from + chunk);
        for (int i = from; i < until; i++) {
            const float x = row.logit(i);
            const u64 w = weight(x);
            if (stays(x, i, w)) mass += w;
        }
        const u64 before = block_before(mass, sh.scratch), all = block_reduce(mass, sh.scratch, sum);
        const double goal = (double)p.uniform[r] * (double)all;
        u64 found = ~0ull, last = 0;
        u64 run = before;
        for (int i = from; i < until; i++) {
            const float x = row.logit(i);
            const u64 w = weight(x);
            if (!stays(x, i, w)) continue;
            run += w;
            if ((u64)i + 1 > last) last = (u64)i + 1;
            if (found == ~0ull && (double)run > goal) found = (u64)i;
        }
        found = block_reduce(found, sh.scratch, least);
        last = block_reduce(last, sh.scratch, [](u64 a, u64 b) { return a > b ? a : b; });
        if (threadIdx.x == 0) p.out[r] = (int)(found == ~0ull ? last - 1 : found);
        __syncthreads();
    }
}

}  // namespace

int launch_sample(const SampleParams& p, cudaStream_t stream) {
    const dim3 grid((unsigned)std::min<int64_t>(p.rows, 1 << 20));
    if (p.half) launch_pdl(sample_kernel<__half>, grid, dim3(kThreads), 0, stream, p);
    else launch_pdl(sample_kernel<float>, grid, dim3(kThreads), 0, stream, p);
    return (int)cudaGetLastError();
}

}  // namespace kn
