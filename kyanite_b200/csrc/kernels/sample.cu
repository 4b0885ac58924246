// One token for every row of logits, by temperature, top-k, top-p and min-p and a given random number.
//
// A token's weight exp((x - max) / T) is counted in whole steps of 2^-44 of the highest, from f64: sums of whole numbers are the
// same in any order.  What stays after top-k and top-p is the head of one order (falling logits, rising index among equals), so
// each is a cut: a key (the logit's bits in the order of whole numbers) and, among equal keys, an index.  A cut is found by
// eight bits of the key at a time, from counts or weights per value of them.
//
// A row is read once, into the shared memory of a cluster of up to eight CTAs that share it.  Cuts are found from counts or weights of 1024
// bins of the logits; a bin's tokens, if there are not too many, go to one CTA that ranks them all at once.  Weights are
// computed in f64 by a table of 256 powers and four terms of a series: ten operations, where the general exp has some thirty.
// Measured, step alone (of three executors side by side): 200 rows of 128256 f16 logits of which all tokens stay 70 us (57), one of 32000 f32
// 11.5 (4.8), with a top-k and a top-p 30 (11), greedy 3.8 (2.5).  51 MB of logits are 8 us of memory; issue slots are 56 % used, the f64 pipe
// 24 %: most of the time warps wait at barriers (of a row's CTAs and the cluster), of which each cut has four to six more.
// Rows that do not fit, or whose tokens do not lie together, are read again and again by one CTA.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "../kernels.h"
#include "launch.cuh"
#include "tc_ptx.cuh"

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
        const double goal = fmax((double)p.uniform[r] * (double)all, 0.0);
        u64 found = ~0ull, last = 0;
        u64 run = before;
        for (int i = from; i < until; i++) {
            const float x = row.logit(i);
            const u64 w = weight(x);
            if (!stays(x, i, w)) continue;
            run += w;
            if (w > 0 && (u64)i + 1 > last) last = (u64)i + 1;   // (of those that weigh something)
            if (found == ~0ull && (double)run > goal) found = (u64)i;
        }
        found = block_reduce(found, sh.scratch, least);
        last = block_reduce(last, sh.scratch, [](u64 a, u64 b) { return a > b ? a : b; });
        if (threadIdx.x == 0) p.out[r] = (int)(found == ~0ull ? last - 1 : found);
        __syncthreads();
    }
}

// ---- the usual rows: a cluster a row

constexpr int kCta = 512, kWarps = kCta / 32, kPieces = 8;   // a warp's part of a row is summed in eight pieces
constexpr int kBins = 1024, kList = 1024, kTable = 256;
constexpr int kMaxCluster = 8;
constexpr float kDepth = 32.f;   // weights below e^-32 count as 0 (2^-46 and less, in steps of 2^-44)

// A number of some tokens and their weight
struct Amount {
    u64 mass;
    uint32_t count;
};

// What the CTAs of a cluster tell each other, and what they share inside
struct ClusterShared {
    u64 bar;
    u64 slots[2][kMaxCluster];            // from each CTA, two exchanges in turn
    double table[kTable];                 // 2^44 2^(-k / 256)
    u64 pieces[kWarps * kPieces], scan[kWarps];
    uint32_t counts[kBins], limbs[3][kBins];   // weights of a bin in 15, 15 and 14 bits: no sum of 2^17 of them overflows
    // the leader's
    uint32_t list_key[kList], list_index[kList], listed;
    u64 list_weight[kList];
    // the leader's answer, to all
    int bin;
    uint32_t before_count, in_bin;
    u64 before_mass;
    uint32_t key, index;
    int found, at, abandon;
};

template <typename T>
struct Slice {
    const T* at;              // in shared memory
    int from, n;              // index of the first, how many
    float most;               // of the row
    float least;              // logits below it weigh nothing
    float depth;              // 2 kBins / (kDepth T): bins per unit of the logits' halves
    double rate;              // -256 log2(e) / T
    const double* table;
    __device__ __forceinline__ float logit(int i) const {
        const float x = (float)at[i] + 0.f;   // (-0 + 0 = 0: equal logits have equal keys)
        return x != x ? -INFINITY : x;
    }
    // 2^44 e^((x - most) / T), rounded, + 2^52, as the bits of an f64: the number is in the low 52.  2^(k / 256) from the table, the rest
    // by the series of 2^x.  (Finite `most`; of NaN, and of -infinity where `least` is above the lowest number, 0)
    __device__ __forceinline__ u64 weight_bits(float x) const {
        const double d = (double)most - (double)fmaxf(x, least), magic = 6755399441055744.0;   // 1.5 x 2^52: a sum's low word is the number, rounded
        const double t = __fma_rn(d, rate, magic);
        const int k = -__double2loint(t);   // (0 to 400 x 256: up to 256 steps of the temperature from one f32 to the next, times log2(e))
        const double r = __fma_rn(d, rate, -(t - magic));   // 256 times the rest, up to 1/2 either way
        constexpr double kLn = 0.69314718055994531 / 256;
        double p = __fma_rn(r, kLn * kLn * kLn * kLn / 24, kLn * kLn * kLn / 6);
        p = __fma_rn(p, r, kLn * kLn / 2);
        p = __fma_rn(p, r, kLn);
        p = __fma_rn(p, r, 1.0);
        const double w = p * table[k & (kTable - 1)];
        const double scaled = __hiloint2double(__double2hiint(w) - (int)((uint32_t)(k << 12) & 0xfff00000u), __double2loint(w));
        return (u64)__double_as_longlong(scaled + 4503599627370496.0);
    }
    __device__ __forceinline__ u64 weight(float x) const {
        if (most == INFINITY) return x == most ? 1ull << 44 : 0;
        return x > -INFINITY ? weight_bits(x) & 0xfffffffffffffull : 0;
    }
    // 0 .. kBins - 1 by falling logit; the last holds what weighs nothing
    __device__ __forceinline__ int bin(float x) const {
        if (x == most) return 0;
        const float b = (0.5f * most - 0.5f * x) * depth;   // (their difference may be too large)
        return b < (float)(kBins - 1) ? (int)b : kBins - 1;   // (also of -infinity, and under a highest logit of infinity)
    }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kCta, 2) sample_cluster_kernel(const __grid_constant__ SampleParams p, int slice) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(128) uint8_t raw[];
    __shared__ ClusterShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = cluster.num_blocks(), me = cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x / ctas;
    ClusterShared& leader = *cluster.map_shared_rank(&sh, 0);
    T* const x = (T*)raw;
    const int from = me * slice, n = max(0, min(slice, p.vocab - from));
    const uint32_t bar = tcp::smem_u32(&sh.bar);
    if (threadIdx.x == 0) {
        tcp::mbar_init(bar, 1);
        sh.abandon = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    auto started = cluster.barrier_arrive();   // (a CTA's memory is there once it runs)
    if (threadIdx.x < kTable) sh.table[threadIdx.x] = exp2(44.0 - (double)threadIdx.x / kTable);
    __syncthreads();
    pdl_enter();
    // ---- the slice
    const T* in = (const T*)p.logits + r * p.row_stride + from;
    constexpr int kUnit = 16 / sizeof(T);
    const bool bulk = p.row_stride % kUnit == 0 && (uintptr_t)p.logits % 16 == 0;   // (slices are multiples of 16 bytes)
    const int whole = bulk ? n / kUnit * kUnit : 0;
    if (whole > 0 && threadIdx.x == 0) {
        tcp::mbar_expect_tx(bar, whole * sizeof(T));
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tcp::smem_u32(x)), "l"(in),
                     "r"((uint32_t)(whole * sizeof(T))), "r"(bar) : "memory");
    }
    for (int i = whole + threadIdx.x; i < n; i += kCta) x[i] = in[i];
    if (threadIdx.x == 0 && (n & 1)) x[n] = (T)-INFINITY;
    const float temperature = p.temperature ? p.temperature[r] : 1.f, uniform = p.uniform[r], top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p ? p.min_p[r] : 0.f;
    const int top_k = p.top_k ? p.top_k[r] : 0;
    // (given up: the host learns of it.  The copy is still waited for: what is counted below must not change meanwhile)
    if (whole > 0 && !tcp::mbar_wait(bar, 0, &sh.abandon, p.status, 72u)) tcp::mbar_drain(bar, 0, clock64());
    __syncthreads();
    cluster.barrier_wait(std::move(started));
    // one number from each CTA; all get all of them
    int turn = 0;
    const auto exchange = [&](u64 v) {   // by thread 0
        if (threadIdx.x == 0)
            for (int c = 0; c < ctas; c++) cluster.map_shared_rank(&sh, c)->slots[turn][me] = v;
        cluster.sync();
        return sh.slots[turn++ & 1];
    };
    Slice<T> row{x, from, n, 0.f, 0.f, 0.f, 0.0, sh.table};
    // ---- highest logit
    using Two = typename std::conditional<sizeof(T) == 2, __half2, float2>::type;
    const auto two_of = [&](int i) {   // logits 2 i and 2 i + 1 of the slice
        const Two v = ((const Two*)x)[i];
        if constexpr (sizeof(T) == 2) return __half22float2(v);
        else return v;
    };
    const int pairs = (n + 1) / 2;   // (what is behind the last is -infinity)
    float most = -INFINITY;
    for (int i = threadIdx.x; i < pairs; i += kCta) {
        const float2 v = two_of(i);
        most = fmaxf(most, fmaxf(v.x, v.y));
    }
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) sh.scan[warp] = __float_as_uint(most);
    __syncthreads();
    for (int w = 0; w < kWarps; w++) most = fmaxf(most, __uint_as_float((uint32_t)sh.scan[w]));
    {
        const u64* all = exchange(__float_as_uint(most));
        for (int c = 0; c < ctas; c++) most = fmaxf(most, __uint_as_float((uint32_t)all[c]));
        turn &= 1;
    }
    row.most = most + 0.f;
    if (most == -INFINITY) {
        if (me == 0 && threadIdx.x == 0) p.out[r] = -1;
        return;   // (all CTAs of the cluster; nobody reads another's memory any more)
    }
    if (!(temperature > 0.f) || !(min_p <= 1.f)) {
        // the first of the highest is all that stays
        uint32_t first = 0xffffffffu;
        for (int i = threadIdx.x; i < n; i += kCta)
            if (row.logit(i) == row.most) first = min(first, (uint32_t)(from + i));
        first = __reduce_min_sync(0xffffffffu, first);
        __syncthreads();
        if (lane == 0) sh.scan[warp] = first;
        __syncthreads();
        for (int w = 0; w < kWarps; w++) first = min(first, (uint32_t)sh.scan[w]);
        const u64* all = exchange(first);
        for (int c = 0; c < ctas; c++) first = min(first, (uint32_t)all[c]);
        if (me == 0 && threadIdx.x == 0) p.out[r] = (int)first;
        return;
    }
    // No logit lies between the highest and the f32 below it.  Temperatures under 1/256 of that step leave weight to the highest alone, and count
    // as that much: nothing in the exponent's arithmetic overflows then.  `least` is rounded down, so that what it stands for weighs e^-44
    // and less, which is 2^-63, and never as much as the highest.
    const float gap = row.most - nextafterf(row.most, -INFINITY);
    const float heat = gap < INFINITY ? fmaxf(temperature, gap / 256.f) : temperature;
    row.rate = -256.0 * 1.4426950408889634074 / (double)heat;
    row.least = fmaxf(__fsub_rd(row.most, __fmul_ru(44.f, heat)), -FLT_MAX);
    row.depth = fminf(2.f * (float)kBins / kDepth / heat, 1e30f);
    Cut cut{0, INT_MAX};

    // In the order of the index: what each piece weighs by `amount`, summed over the cluster; then the first index at which the
    // running sum passes `goal` (a sum reaches it where `reach`).  Its number goes to all CTAs
    const int piece = (slice + 2 * kWarps * kPieces - 1) / (2 * kWarps * kPieces) * 2;
    const auto sums = [&](auto amount, u64 bias = 0) {   // bias: what each amount is too large by
        for (int q = 0; q < kPieces; q++) {
            const int a = (warp * kPieces + q) * piece, b = min(n, a + piece);
            u64 sum = 0;
            for (int i = a / 2 + lane; 2 * i < b; i += 32) {
                const float2 v = two_of(i);
                sum += amount(v.x, from + 2 * i) + amount(v.y, from + 2 * i + 1);
            }
            if (b > a) sum -= bias * (2 * (u64)max(0, (((b + 1) / 2 - a / 2) - lane + 31) / 32));
            sum = warp_sum(sum);
            if (lane == 0) sh.pieces[warp * kPieces + q] = sum;
        }
        __syncthreads();
        u64 all = threadIdx.x < kWarps * kPieces ? sh.pieces[threadIdx.x] : 0;
        all = warp_sum(all);
        if (lane == 0) sh.scan[warp] = all;
        __syncthreads();
        all = 0;
        for (int w = 0; w < kWarps * kPieces / 32; w++) all += sh.scan[w];
        return all;   // of this CTA
    };
    const auto search = [&](auto amount, auto passes, u64 front, u64 own) {   // front: of the CTAs in front, own: this one's
        if (own == 0 || !passes(front + own) || (front > 0 && passes(front))) return -1;   // (only the CTA in which it happens)
        if (threadIdx.x == 0) {
            u64 run = front;
            int q = 0;
            for (; q < kWarps * kPieces - 1; q++) {
                if (passes(run + sh.pieces[q])) break;
                run += sh.pieces[q];
            }
            sh.before_mass = run;
            sh.found = q;
            sh.at = -1;
        }
        __syncthreads();
        if (warp == 0) {
            u64 run = sh.before_mass;
            const int a = sh.found * piece, b = min(n, a + piece);
            for (int i0 = a; i0 < b; i0 += 32) {
                const int i = i0 + lane;
                const u64 v = i < b ? amount(row.logit(i), from + i) : 0;
                u64 up = v;
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 w = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += w;
                }
                const uint32_t over = __ballot_sync(0xffffffffu, v > 0 && passes(run + up));
                if (over) {
                    if (lane == 0) sh.at = from + i0 + __ffs(over) - 1;
                    break;
                }
                run += __shfl_sync(0xffffffffu, up, 31);
            }
        }
        __syncthreads();
        return sh.at;
    };

    // ---- a cut: the shortest head of the order, within `within`, of `k` tokens or of `share` of the weight (k == 0)
    const auto find_cut = [&](Cut within, int k, double share) {
        // bins: first of the logits, then, while one holds more tokens than the list, of their keys from low to high
        uint32_t low = 0, high = 0xffffffffu, before_count = 0;
        u64 before_mass = 0, goal = 0;
        int bin = -1;
        for (int level = 0;; level++) {
            const uint64_t range = (uint64_t)high - low + 1;
            const auto bin_of = [&](float x, uint32_t key) { return level == 0 ? row.bin(x) : (int)((uint64_t)(high - key) * kBins / range); };
            const auto member = [&](float x, uint32_t key, int i) { return within.keeps(key, i) && (level == 0 || (row.bin(x) == bin && key >= low && key <= high)); };
            for (int i = threadIdx.x; i < kBins; i += kCta) sh.counts[i] = sh.limbs[0][i] = sh.limbs[1][i] = sh.limbs[2][i] = 0;
            if (threadIdx.x == 0) sh.listed = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += kCta) {
                const float v = row.logit(i);
                const uint32_t key = key_of(v);
                if (!member(v, key, from + i)) continue;
                const int b = bin_of(v, key);
                if (level == 0 && b == kBins - 1) continue;   // weighs nothing
                atomicAdd(&sh.counts[b], 1u);
                if (k == 0) {
                    const u64 w = row.weight(v);
                    atomicAdd(&sh.limbs[0][b], (uint32_t)w & 0x7fffu);
                    atomicAdd(&sh.limbs[1][b], (uint32_t)(w >> 15) & 0x7fffu);
                    atomicAdd(&sh.limbs[2][b], (uint32_t)(w >> 30));
                }
            }
            cluster.sync();
            if (me == 0) {
                // two bins a thread: their sums, those of all in front, and where the goal is reached
                Amount mine[2];
                for (int j = 0; j < 2; j++) {
                    const int b = 2 * threadIdx.x + j;
                    mine[j] = {0, 0};
                    for (int c = 0; c < ctas; c++) {
                        const ClusterShared& o = *cluster.map_shared_rank(&sh, c);
                        mine[j].count += o.counts[b];
                        mine[j].mass += (u64)o.limbs[0][b] + ((u64)o.limbs[1][b] << 15) + ((u64)o.limbs[2][b] << 30);
                    }
                }
                const u64 measure[2] = {k > 0 ? mine[0].count : mine[0].mass, k > 0 ? mine[1].count : mine[1].mass};
                u64 up = measure[0] + measure[1];
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 w = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += w;
                }
                __syncthreads();
                if (lane == 31) sh.scan[warp] = up;
                if (threadIdx.x == 0) sh.bin = -1;
                __syncthreads();
                u64 all = 0;
                for (int w = 0; w < kWarps; w++) {
                    if (w < warp) up += sh.scan[w];
                    all += sh.scan[w];
                }
                if (level == 0) {
                    const double g = ceil(share * (double)all);
                    goal = k > 0 ? (u64)k : g >= 1.0 ? (u64)g : 1;
                }
                u64 run = (k > 0 ? before_count : before_mass) + up - measure[0] - measure[1];
                for (int j = 0; j < 2; j++) {
                    if (measure[j] > 0 && run < goal && goal <= run + measure[j]) {
                        sh.bin = 2 * threadIdx.x + j;
                        sh.before_mass = run;
                        sh.in_bin = mine[j].count;
                    }
                    run += measure[j];
                }
                __syncthreads();
                if (threadIdx.x == 0) {
                    const u64 run0 = sh.before_mass, g = goal;
                    const int b = sh.bin;
                    const uint32_t in_bin = sh.in_bin;
                    for (int c = 0; c < ctas; c++) {
                        ClusterShared& o = *cluster.map_shared_rank(&sh, c);
                        o.bin = b, o.before_mass = run0, o.in_bin = in_bin, o.scan[0] = g;
                    }
                }
            }
            cluster.sync();
            if (sh.bin < 0) return within;   // all that weighs anything stays
            goal = sh.scan[0];
            if (k > 0) before_count = (uint32_t)sh.before_mass;
            else before_mass = sh.before_mass;
            const int chosen = sh.bin;
            const uint32_t in_bin = sh.in_bin;
            const uint32_t old_high = high;
            if (level == 0) {
                bin = chosen;
            } else {
                // keys of which (high - key) kBins / range is `chosen`
                const uint64_t near = ((uint64_t)chosen * range + kBins - 1) / kBins, far = ((uint64_t)(chosen + 1) * range + kBins - 1) / kBins - 1;
                high = old_high - (uint32_t)near;
                low = old_high - (uint32_t)far;
            }
            const auto chosen_one = [&](float v, uint32_t key, int i) { return within.keeps(key, i) && row.bin(v) == bin && key >= low && key <= high; };
            if (in_bin <= kList) {
                // to the leader, who finds each one's place among them
                for (int i = threadIdx.x; i < n; i += kCta) {
                    const float v = row.logit(i);
                    const uint32_t key = key_of(v);
                    if (!chosen_one(v, key, from + i)) continue;
                    const uint32_t at = atomicAdd(&leader.listed, 1u);
                    leader.list_key[at] = key, leader.list_index[at] = from + i, leader.list_weight[at] = k > 0 ? 1 : row.weight(v);
                }
                cluster.sync();
                if (me == 0)
                    for (uint32_t e = threadIdx.x; e < in_bin; e += kCta) {
                        const uint32_t key = sh.list_key[e], index = sh.list_index[e];
                        u64 run = k > 0 ? before_count : before_mass;
                        for (uint32_t o = 0; o < in_bin; o++) {
                            const uint32_t other = sh.list_key[o];
                            if (other > key || (other == key && sh.list_index[o] < index)) run += sh.list_weight[o];
                        }
                        if (run < goal && goal <= run + sh.list_weight[e])
                            for (int c = 0; c < ctas; c++) {
                                ClusterShared& o = *cluster.map_shared_rank(&sh, c);
                                o.key = key, o.index = index;
                            }
                    }
                cluster.sync();
                const Cut found{sh.key, (int)sh.index};
                cluster.sync();   // (before anybody writes there again)
                return found;
            }
            if (low == high) {
                // equal logits: by index
                float value = 0.f;
                const uint32_t key = low;
                value = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
                const u64 each = k > 0 ? 1 : row.weight(value), need = (goal - (k > 0 ? before_count : before_mass) + each - 1) / each;
                const auto one = [&](float v, int i) { return (u64)(key_of(v + 0.f) == key && within.keeps(key, i) ? 1 : 0); };
                const u64 own = sums(one);
                const u64* all = exchange(own);
                turn &= 1;
                u64 front = 0;
                for (int c = 0; c < me; c++) front += all[c];
                const int at = search(one, [&](u64 s) { return s >= need; }, front, own);
                if (at >= 0 && threadIdx.x == 0)
                    for (int c = 0; c < ctas; c++) cluster.map_shared_rank(&sh, c)->index = at;
                cluster.sync();
                const Cut found{key, (int)sh.index};
                cluster.sync();
                return found;
            }
            if (level == 0) {
                // the keys of that bin
                uint32_t lo = 0xffffffffu, hi = 0;
                for (int i = threadIdx.x; i < n; i += kCta) {
                    const float v = row.logit(i);
                    const uint32_t key = key_of(v);
                    if (!chosen_one(v, key, from + i)) continue;
                    lo = min(lo, key), hi = max(hi, key);
                }
                lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
                __syncthreads();
                if (lane == 0) sh.scan[warp] = (u64)lo << 32 | hi;
                __syncthreads();
                for (int w = 0; w < kWarps; w++) lo = min(lo, (uint32_t)(sh.scan[w] >> 32)), hi = max(hi, (uint32_t)sh.scan[w]);
                const u64* all = exchange((u64)lo << 32 | hi);
                turn &= 1;
                for (int c = 0; c < ctas; c++) lo = min(lo, (uint32_t)(all[c] >> 32)), hi = max(hi, (uint32_t)all[c]);
                low = lo, high = hi;
            }
        }
    };
    if (top_k > 0 && top_k < p.vocab) cut = find_cut(cut, top_k, 0.0);
    if (p.top_p && !(top_p >= 1.f)) cut = find_cut(cut, 0, (double)top_p);

    // ---- the token
    const u64 least_weight = (u64)ceil(fmax((double)min_p, 0.0) * 17592186044416.0);
    const bool all_stay = cut.key == 0;
    const auto amount = [&](float v, int i) {
        const u64 w = row.weight(v);
        return w >= least_weight && (all_stay || cut.keeps(key_of(v + 0.f), i)) ? w : (u64)0;
    };
    // (all tokens, the usual kind: no more than their weights)
    const bool usual = all_stay && least_weight == 0 && row.most < INFINITY && row.least > -FLT_MAX;
    const u64 own = usual ? sums([&](float v, int) { return row.weight_bits(v); }, 0x4330000000000000ull) : sums(amount);
    const u64* all = exchange(own);
    u64 front = 0, total = 0;
    for (int c = 0; c < ctas; c++) {
        if (c < me) front += all[c];
        total += all[c];
    }
    const double goal = fmax((double)uniform * (double)total, 0.0);
    const auto passes = [&](u64 s) { return (double)s > goal || s == total; };   // (the last token for a number of 1 and more)
    const int token = search(amount, passes, front, own);
    if (token >= 0 && threadIdx.x == 0) p.out[r] = token;
    cluster.sync();   // (nobody leaves while another may still read its memory)
}

// CTAs of a row's cluster and tokens of each; 0: the row does not fit
int cluster_of(const SampleParams& p, int* slice) {
    const int size = p.half ? 2 : 4, unit = 16 / size;
    const auto tokens = [&](int ctas) { return ((p.vocab + ctas - 1) / ctas + unit - 1) / unit * unit; };
    int ctas = 1;
    // 64 KB a CTA, for two on an SM; and, of few rows, as many CTAs as have an SM's half, with 1024 tokens and more each.
    // (Step alone: 200 x 128256 f16 70.6 us with 64 KB, 75.8 with 180; 16 x 128256 18.8 spread, 22.8 not; 8 x 32000 f32 12.9 and 15.8.)
    while (ctas < kMaxCluster && ((int64_t)tokens(ctas) * size > 64 * 1024 || (p.rows * ctas * 2 <= 2 * 148 && p.vocab / (2 * ctas) >= 1024))) ctas *= 2;
    *slice = tokens(ctas);
    return p.col_stride != 1 || (int64_t)*slice * size > 180 * 1024 || p.rows * ctas > INT_MAX ? 0 : ctas;
}

template <typename T>
int launch_cluster(const SampleParams& p, int ctas, int slice, cudaStream_t stream) {
    static bool done[64];
    static std::mutex mu;
    const int err = allow_shared(sample_cluster_kernel<T>, 180 * 1024, done, mu);
    if (err != 0) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.rows * ctas));
    cfg.blockDim = dim3(kCta);
    cfg.dynamicSmemBytes = (size_t)slice * sizeof(T);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    (void)cudaLaunchKernelEx(&cfg, sample_cluster_kernel<T>, p, slice);   // a failure stays in cudaGetLastError()
    return 0;
}

}  // namespace

int launch_sample(const SampleParams& p, cudaStream_t stream) {
    int slice = 0;
    if (const int ctas = cluster_of(p, &slice)) {
        const int err = p.half ? launch_cluster<__half>(p, ctas, slice, stream) : launch_cluster<float>(p, ctas, slice, stream);
        return err != 0 ? err : (int)cudaGetLastError();
    }
    const dim3 grid((unsigned)std::min<int64_t>(p.rows, 1 << 20));
    if (p.half) launch_pdl(sample_kernel<__half>, grid, dim3(kThreads), 0, stream, p);
    else launch_pdl(sample_kernel<float>, grid, dim3(kThreads), 0, stream, p);
    return (int)cudaGetLastError();
}

}  // namespace kn
