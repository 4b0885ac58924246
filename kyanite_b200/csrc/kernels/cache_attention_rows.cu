// Attention of many rows against a decoder's cache of 8 bits, on the tensor cores' 128-row instructions: the next piece of a prompt
// (rows: the tokens and heads of a sequence that share keys), or what all sequences see of a prefix that they share (rows: those of
// all sequences; the results are parts that cache_attention_kernel joins with what each sequence sees of its own).
//
// A CTA has 256 rows, two accumulator tiles of 128, and takes 64 keys at a time:
//
//   warps 0..7      queries once; softmax: a row per thread, four warps a tile; the two tiles' exponentials run beside each other's products
//   warps 8..11     keys and values of 8 bits -> f16 in shared memory (exact; kernels/cache.cuh), three blocks of both in turn; their
//                   scales
//   warp 12, a lane MMA issuer: the next block's scores go ahead of this block's products with the values, tile by tile
//
// Scores of a block are one of a tile's two accumulators of 64 columns in tensor memory; its weights take their place as two halves of 11 bits
// in f16, 32 columns each, and are the A operands of the second product, whose accumulator stays.  (22 bits, as cache_attention_kernel has
// them: with the upper half alone results of f16 were 2.9e-4 from 64 bits, where their own rounding is 2.1e-4, and a sequence's
// result depended on how many others there were.  The lower half costs 128.7 -> 146.0 us at the size below, 71.1 -> 73.5 behind a
// prefix, step alone.)  Scales of keys multiply scores, those of values weights, in f32.  Weights go by a reference that no score is more
// than 2^8 above; it moves rarely, and then the thread rescales its row (once the block before has been added).  Where the items are
// fewer than the SMs their keys are split over several CTAs, and a second kernel joins the parts in order.
//
// Measured: 512 tokens of 2 sequences behind 4096 positions, 32 / 8 heads of 128 channels (73 GFLOP), step alone 146 us, 500
// TFLOP/s; of three executors side by side 129, 565 TFLOP/s.  Bound by the chain of a block's products and exponentials that wait for one
// another: the tensor pipe is busy 40 % of the time, issue slots 44 %.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "cache.cuh"
#include "launch.cuh"
#include "tc_ptx.cuh"

namespace kn {

namespace {

using namespace tcp;

constexpr int kRows = 256, kTileRows = 128, kKeys = 64, kStages = 3;
constexpr int kThreads = 13 * 32;
constexpr float kBottom = -3.402823466e38f, kAbove = 8.f;
constexpr uint32_t kSleepNs = 200;

template <int DB>   // 64-channel panels
struct RowsGeo {
    static constexpr int kDim = 64 * DB, kRowBytes = kDim;
    static constexpr int kQTile = DB * kTileRows * 128, kPart = DB * kKeys * 128;   // bytes: a tile's queries; a block's keys (or values)
    static constexpr int kStage = 2 * kPart;
    static constexpr int kScales = 2 * kQTile + kStages * kStage;   // [stage][keys, values][64] f32
    static constexpr int kBars = kScales + kStages * 2 * kKeys * 4;
    static constexpr int kShared = 1024 + kBars + 256;
    static constexpr int kChunks = kKeys * (kDim / 16) * 2 / 128;   // 16-byte pieces of a block per thread
};

__device__ __forceinline__ uint32_t two_low(uint32_t w) {
    const uint32_t raised = __byte_perm(w, 0x64646464u, 0x4140), off = 0x64806480u;
    const __half2 h = __hsub2(*(const __half2*)&raised, *(const __half2*)&off);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t two_high(uint32_t w) {
    const uint32_t raised = __byte_perm(w, 0x64646464u, 0x4342), off = 0x64806480u;
    const __half2 h = __hsub2(*(const __half2*)&raised, *(const __half2*)&off);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ void mma_f16_weights(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }

// Two products, or sums, in one instruction
__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b));
    return *(float2*)&d;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b));
    return *(float2*)&d;
}
__device__ __forceinline__ float max_of(float a, float b, float c) {   // (of numbers: a NaN is passed over)
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// What a row sees, in positions of a run (0: the prefix, 1: its sequence's own)
struct Sight {
    int low[2], high[2];
    bool live;
};

template <int DB>
__global__ void __launch_bounds__(kThreads, 1) cache_attention_rows_kernel(const __grid_constant__ CacheAttentionParams p) {
    using G = RowsGeo<DB>;
    constexpr int kDim = G::kDim;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + G::kBars;
    // per tile: queries are there; per stage full and empty, then per tile and parity of the block: scores complete, weights ready, values added; last, all products
    const uint32_t q_full = bars, full = bars + 16, empty = full + 8 * kStages, s_full = empty + 8 * kStages, p_ready = s_full + 32, pv_done = p_ready + 32, all_done = pv_done + 32;
    __shared__ uint32_t tmem_slot;
    __shared__ int abandon_flag, any_lo[2], any_hi[2], all_lo[2], all_hi[2];
    __shared__ float value_most[kStages][2];
    volatile int* const abandon = &abandon_flag;
    float* const scales = (float*)(gen + G::kScales);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 4), mbar_init(q_full + 8, 4);
        for (int i = 0; i < kStages; i++) mbar_init(full + 8 * i, 4), mbar_init(empty + 8 * i, 1);
        for (int i = 0; i < 4; i++) mbar_init(s_full + 8 * i, 1), mbar_init(p_ready + 8 * i, 4), mbar_init(pv_done + 8 * i, 1);
        mbar_init(all_done, 1);
        abandon_flag = 0;
        for (int r = 0; r < 2; r++) any_lo[r] = all_hi[r] = 1 << 30, any_hi[r] = all_lo[r] = -(1 << 30);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_enter();
    const bool prefix_only = p.many == 2;
    const int group = p.heads / p.cache.heads, splits = p.splits;
    const int rows = (prefix_only ? p.cache.seqs : 1) * p.tokens * group, row_tiles = (rows + kRows - 1) / kRows;
    const int item = blockIdx.x / splits, split = blockIdx.x % splits;
    // (the last rows first: they see the most)
    const int row0 = (row_tiles - 1 - item % row_tiles) * kRows, head = item / row_tiles % p.cache.heads, item_seq = item / row_tiles / p.cache.heads;
    const int shared = p.prefix.base ? min(max(*p.prefix_length, 0), p.prefix.capacity) : 0;
    const auto cut = [](int64_t x) { return (int)max(min(x, (int64_t)(1 << 30)), (int64_t)-(1 << 30)); };
    const auto seq_of = [&](int row) { return prefix_only ? row / group / p.tokens : item_seq; };
    const auto token_of = [&](int row) { return prefix_only ? row / group % p.tokens : row / group; };
    // this thread's row (softmax)
    const int row = row0 + (threadIdx.x & (kRows - 1));
    Sight sight{};
    int64_t position = 0;   // behind the prefix
    int counted = 0;        // what penalties count from, as in cache_attention.cu
    if (warp < 8 && row < rows) {
        const int s = seq_of(row), t = token_of(row);
        position = (int64_t)p.start[s] + t;
        counted = max(min(p.start[s], p.cache.capacity - 1), -(1 << 30)) + t;
        sight.live = position >= 0 && (p.count == nullptr || t < p.count[s]);
        sight.high[0] = shared, sight.high[1] = cut(min(position + 1, (int64_t)p.cache.capacity));
        sight.low[0] = p.window > 0 ? max(cut(shared + position - p.window + 1), 0) : 0;
        sight.low[1] = p.window > 0 ? max(cut(position - p.window + 1), 0) : 0;
    }
    __syncthreads();   // (before the range is agreed on)
    if (warp < 8) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const bool some = sight.live && sight.low[r] < sight.high[r];
            const int lo = __reduce_min_sync(0xffffffffu, some ? sight.low[r] : 1 << 30), hi = __reduce_max_sync(0xffffffffu, some ? sight.high[r] : -(1 << 30));
            const int high_lo = __reduce_max_sync(0xffffffffu, sight.live ? sight.low[r] : -(1 << 30)), low_hi = __reduce_min_sync(0xffffffffu, sight.live ? sight.high[r] : 1 << 30);
            if (lane == 0) atomicMin(&any_lo[r], lo), atomicMax(&any_hi[r], hi), atomicMax(&all_lo[r], high_lo), atomicMin(&all_hi[r], low_hi);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // blocks of 64 keys that some row sees: those of the prefix, then the sequence's own; of them this CTA's part
    const int first0 = any_lo[0] / kKeys, n0 = any_hi[0] > any_lo[0] ? (any_hi[0] + kKeys - 1) / kKeys - first0 : 0;
    const int first1 = any_lo[1] / kKeys, n1 = !prefix_only && any_hi[1] > any_lo[1] ? (any_hi[1] + kKeys - 1) / kKeys - first1 : 0;
    const int from = (int)((int64_t)(n0 + n1) * split / splits), n = (int)((int64_t)(n0 + n1) * (split + 1) / splits) - from;
    const int tiles = rows - row0 > kTileRows ? 2 : 1;

    if (warp >= 8 && warp < 12) {
        // ---------------- keys and values
        const int me = threadIdx.x - 256;
        const float log2e = 1.4426950408889634f;
        const float unit = p.softcap > 0.f ? p.scale * 2.f * log2e / p.softcap : p.scale * log2e;
        constexpr int kAcross = kDim / 16;
        // piece i of this thread: of part i / (pieces of a part), of key i x kApart + key_of_mine in it, always the same 16 channels
        constexpr int kApart = 128 / kAcross, kOfPart = G::kChunks / 2;
        const int my_key = me / kAcross, chunk = me % kAcross;   // (kApart is a multiple of 16: the order in a row is the key's)
        const int from_at = (my_key & 15) * G::kRowBytes + ((chunk ^ cache_swizzle(G::kRowBytes, my_key & 15)) << 4);
        const int to_at = (chunk >> 2) * (kKeys * 128) + my_key * 128, to_lo = (((chunk & 3) * 2) ^ (my_key & 7)) << 4, to_hi = (((chunk & 3) * 2 + 1) ^ (my_key & 7)) << 4;
        struct Block {
            uint4 raw[G::kChunks];
            float scale;
        };
        const auto load = [&](int j, Block& b) {
            const int run = from + j >= n0, kb = run ? first1 + from + j - n0 : first0 + from + j;
            const CacheParams& c = run ? p.cache : p.prefix;
            const uint8_t* const head_at = c.base + ((run ? (int64_t)item_seq * c.heads : 0) + head) * ((int64_t)c.tiles * c.tile_bytes);
            const uint8_t* const at = head_at + (int64_t)(kb * (kKeys / kCacheTile)) * c.tile_bytes + from_at;
            const int last = c.tiles - 1 - kb * (kKeys / kCacheTile);   // (behind it: any numbers will do, nobody sees them)
#pragma unroll
            for (int i = 0; i < G::kChunks; i++) {
                const int part = i / kOfPart, tile = (i % kOfPart * kApart + my_key) >> 4;
                b.raw[i] = __ldcg((const uint4*)(at + min(tile, last) * c.tile_bytes + part * kCacheTile * G::kRowBytes));
            }
            // a scale a thread: of keys, then of values; what no row sees has none
            const int part = me >> 6, key = kb * kKeys + (me & 63);
            b.scale = 0.f;
            if (key >= any_lo[run] && key < any_hi[run])
                b.scale = __ldcg((const float*)(head_at + (int64_t)(key >> 4) * c.tile_bytes + 2 * kCacheTile * G::kRowBytes) + part * kCacheTile + (key & 15));
            if (part == 0) b.scale *= unit;
        };
        const auto step = [&](int j, Block& now, Block& next) -> bool {
            const int st = j % kStages;
            if (j + 1 < n) load(j + 1, next);
            bool good = true;
            if (j >= kStages) good = mbar_wait(empty + 8 * st, (uint32_t)((j / kStages - 1) & 1), abandon, p.status, 81, kWaitCycles, kSleepNs);
            if (!__all_sync(0xffffffffu, good)) return false;
            uint8_t* const to = gen + 2 * G::kQTile + st * G::kStage + to_at;
#pragma unroll
            for (int i = 0; i < G::kChunks; i++) {
                uint8_t* const at = to + i / kOfPart * G::kPart + i % kOfPart * kApart * 128;
                const uint4 w = now.raw[i];
                *(uint4*)(at + to_lo) = make_uint4(two_low(w.x), two_high(w.x), two_low(w.y), two_high(w.y));
                *(uint4*)(at + to_hi) = make_uint4(two_low(w.z), two_high(w.z), two_low(w.w), two_high(w.w));
            }
            scales[(st * 2 + (me >> 6)) * kKeys + (me & 63)] = now.scale;
            if (me >= 64) {
                float most = now.scale;
                for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (lane == 0) value_most[st][warp & 1] = most;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) arrive(full + 8 * st);
            return true;
        };
        Block one, two;
        if (n > 0) load(0, one);
        for (int j = 0; j < n; j += 2)
            if (!step(j, one, two) || (j + 1 < n && !step(j + 1, two, one))) break;
    } else if (warp == 12) {
        if (elect_one() && n > 0) {
            // ---------------- MMA issuer (see kernels/flash.cu)
            const uint32_t idesc = (1u << 4) | ((uint32_t)(kTileRows >> 4) << 24), idesc_s = idesc | ((uint32_t)(kKeys >> 3) << 17);
            const uint32_t idesc_o = idesc | (1u << 16) | ((uint32_t)(kDim >> 3) << 17);
            const uint64_t v_desc = ((uint64_t)((kKeys * 128) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
            const auto scores = [&](int j) -> bool {
                const int st = j % kStages, b = j & 1;
                if (!mbar_wait(full + 8 * st, (uint32_t)((j / kStages) & 1), abandon, p.status, 82, kWaitCycles, kSleepNs)) return false;
                const uint32_t keys = base + 2 * G::kQTile + st * G::kStage;
                for (int tile = 0; tile < tiles; tile++) {
                    // (the weights of the block before the last lie where the scores go)
                    if (j > 1 && !mbar_wait(pv_done + 16 * tile + 8 * b, (uint32_t)(((j - 2) >> 1) & 1), abandon, p.status, 83, kWaitCycles, kSleepNs)) return false;
                    tc_fence_after();
                    for (int s = 0; s < kDim / 16; s++) {
                        const uint64_t da = smem_desc_sw128(base + tile * G::kQTile + (s >> 2) * (kTileRows * 128)) + 2u * (s & 3);
                        const uint64_t db = smem_desc_sw128(keys + (s >> 2) * (kKeys * 128)) + 2u * (s & 3);
                        mma_f16(tmem + tile * 256 + b * kKeys, da, db, idesc_s, s != 0 ? 1u : 0u);
                    }
                    mma_commit(s_full + 16 * tile + 8 * b);
                }
                return true;
            };
            bool ok = mbar_wait(q_full, 0, abandon, p.status, 84, kWaitCycles, kSleepNs) && (tiles == 1 || mbar_wait(q_full + 8, 0, abandon, p.status, 84, kWaitCycles, kSleepNs)) && scores(0);
            for (int j = 0; j < n && ok; j++) {
                const int st = j % kStages, b = j & 1;
                if (j + 1 < n && !scores(j + 1)) break;   // under this block's exponentials
                const uint32_t values = base + 2 * G::kQTile + st * G::kStage + G::kPart;
                for (int tile = 0; tile < tiles && ok; tile++) {
                    ok = mbar_wait(p_ready + 16 * tile + 8 * b, (uint32_t)((j >> 1) & 1), abandon, p.status, 85, kWaitCycles, kSleepNs);
                    if (!ok) break;
                    tc_fence_after();
                    for (int s = 0; s < 2 * (kKeys / 16); s++) {   // upper halves of the weights, then the lower ones
                        const uint64_t db = v_desc | (uint64_t)(((values + s % (kKeys / 16) * 16 * 128) & 0x3FFFFu) >> 4);
                        mma_f16_weights(tmem + tile * 256 + 128, tmem + tile * 256 + b * kKeys + s * 8, db, idesc_o, (j | s) != 0 ? 1u : 0u);
                    }
                    mma_commit(pv_done + 16 * tile + 8 * b);
                }
                if (ok && j + kStages < n) mma_commit(empty + 8 * st);   // (of the last ones nobody asks)
            }
            // (whoever has given up, and when: nothing reads shared memory or writes tensor memory any more)
            mma_commit(all_done);
            mbar_drain(all_done, 0, clock64());
        }
        __syncwarp();
    } else {
        // ---------------- softmax
        const int tile = warp >> 2;
        const uint32_t lane_bits = (uint32_t)((warp & 3) * 32) << 16, my_o = tmem + tile * 256 + 128 + lane_bits;
        const uint32_t my_s_full = s_full + 16 * tile, my_p_ready = p_ready + 16 * tile, my_pv_done = pv_done + 16 * tile;
        const auto wait = [&](uint32_t bar, uint32_t parity, uint32_t code) -> bool {   // one lane polls
            uint32_t good = 1;
            if (lane == 0) good = mbar_wait(bar, parity, abandon, p.status, code, kWaitCycles, kSleepNs) ? 1u : 0u;
            good = __shfl_sync(0xffffffffu, good, 0);
            tc_fence_after();
            return good != 0;
        };
        const bool used = tile < tiles && n > 0;
        // queries: of the warp's 32 rows, 16 bytes a lane
        if (used) {
            constexpr int kUnits = kDim / 8, kAtOnce = 32 / kUnits;   // units of 16 bytes of a row; rows of an access
#pragma unroll 8
            for (int i = 0; i < 32 / kAtOnce; i++) {
                const int r = (threadIdx.x & (kRows - 1) & ~31) + i * kAtOnce + lane / kUnits, unit = lane % kUnits, d = unit * 8, q_row = row0 + r;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (q_row < rows && d < p.cache.dim) {
                    const __half* at = (const __half*)p.query + (int64_t)seq_of(q_row) * p.q_strides[0] + (int64_t)token_of(q_row) * p.q_strides[1] +
                                       (int64_t)(head * group + q_row % group) * p.q_strides[2];
                    if (p.q_wide) {
                        v = *(const uint4*)(at + d);
                    } else {
                        __half h[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) h[k] = d + k < p.cache.dim ? at[(d + k) * p.q_strides[3]] : __half(0.f);
                        v = *(const uint4*)h;
                    }
                }
                *(uint4*)(gen + tile * G::kQTile + (unit >> 3) * (kTileRows * 128) + (r % kTileRows) * 128 + (((unit & 7) ^ (r & 7)) << 4)) = v;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) arrive(q_full + 8 * tile);
        }
        const float log2e = 1.4426950408889634f, cap = p.softcap * log2e;
        const float slope = p.slopes && row < rows ? p.slopes[head * group + row % group] * log2e : 0.f;
        // weights are 2^(x - reference): what the reference is above is 2^7 times a weight over the values' scale, so that weights times
        // scales of values lie under 2^15 in f16
        float highest = kBottom, reference = kBottom, sum = 0.f, value_ref = 0.f, shift = 0.f;
        bool ok = true;
        for (int j = 0; used && j < n; j++) {
            const int st = j % kStages, b = j & 1;
            const uint32_t my_s = tmem + tile * 256 + b * kKeys + lane_bits;
            // (the second wait, for what is there already, is for the scales)
            if (!wait(my_s_full + 8 * b, (uint32_t)((j >> 1) & 1), 86) || !wait(full + 8 * st, (uint32_t)((j / kStages) & 1), 86)) { ok = false; break; }
            const int run = from + j >= n0, key0 = (run ? first1 + from + j - n0 : first0 + from + j) * kKeys;
            uint32_t v[2][32];
            tmem_load_32_nowait(my_s, v[0]);
            tmem_load_32_nowait(my_s + 32u, v[1]);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            const float4* const ks = (const float4*)(scales + st * 2 * kKeys);
            const float4* const vs = ks + kKeys / 4;
            float2 x[32];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float4 k = ks[i];
                const int c = 4 * i & 31;
                x[2 * i] = mul_pair(make_float2(__uint_as_float(v[i >> 3][c]), __uint_as_float(v[i >> 3][c + 1])), make_float2(k.x, k.y));
                x[2 * i + 1] = mul_pair(make_float2(__uint_as_float(v[i >> 3][c + 2]), __uint_as_float(v[i >> 3][c + 3])), make_float2(k.z, k.w));
            }
            if (p.softcap > 0.f) {
                const auto capped = [&](float y) { return cap - __fdividef(2.f * cap, 1.f + exp2_approx(min_keeping_nan(y, 126.f))); };   // tanh(y) = 1 - 2 / (1 + e^(2y))
#pragma unroll
                for (int i = 0; i < 32; i++) x[i] = make_float2(capped(x[i].x), capped(x[i].y));
            }
            if (p.slopes) {
                const float away = (float)(counted + (run ? 0 : shared) - key0);
#pragma unroll
                for (int i = 0; i < 32; i++) x[i].x -= slope * (away - (float)(2 * i)), x[i].y -= slope * (away - (float)(2 * i + 1));
            }
            const bool masked = key0 < all_lo[run] || key0 + kKeys > all_hi[run];   // some row does not see all of it
            const int lo = sight.low[run] - key0, hi = sight.live ? sight.high[run] - key0 : 0;
            if (masked) {
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    if (2 * i < lo || 2 * i >= hi) x[i].x = -INFINITY;
                    if (2 * i + 1 < lo || 2 * i + 1 >= hi) x[i].y = -INFINITY;
                }
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i++) tops[i & 3] = max_of(tops[i & 3], x[i].x, x[i].y);
            const float top = max_of(fmaxf(tops[0], tops[1]), tops[2], tops[3]);
            // ---- the reference
            const float value_top = fmaxf(value_most[st][0], value_most[st][1]);
            const bool wider = value_top > value_ref || value_ref == 0.f;
            if (__any_sync(0xffffffffu, wider || top > highest + kAbove)) {
                float factor = 1.f;
                if (wider) {
                    const int e = min(max((__float_as_int(value_top) >> 23) + 1, 32), 254);
                    const float next_ref = __int_as_float(e << 23);
                    factor = value_ref > 0.f ? value_ref / next_ref : 0.f;
                    value_ref = next_ref;
                    shift = 7.f - (float)(e - 127);
                }
                if (top > highest + kAbove) {
                    factor *= exp2_approx(highest - top);
                    highest = top;
                }
                reference = highest - shift;
                sum *= factor;
                if (j > 0 && __any_sync(0xffffffffu, factor != 1.f)) {
                    if (!wait(my_pv_done + 8 * ((j - 1) & 1), (uint32_t)(((j - 1) >> 1) & 1), 87)) { ok = false; break; }
#pragma unroll 1
                    for (int c = 0; c < kDim / 16; c++) {
                        uint32_t o[16];
                        tmem_load_16_nowait(my_o + c * 16, o);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                        tmem_store_16(my_o + c * 16, o);
                    }
                }
            }
            // ---- weights.  (One that is hidden is 0, whatever its position's scale: 0 times a scale that is none is a NaN)
            const float2 down = make_float2(-reference, -reference);
            float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const float2 y = add_pair(x[i], down);
                x[i] = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                sums[i & 1] = add_pair(sums[i & 1], x[i]);
            }
            sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float4 f = vs[i];
                x[2 * i] = mul_pair(x[2 * i], make_float2(f.x, f.y)), x[2 * i + 1] = mul_pair(x[2 * i + 1], make_float2(f.z, f.w));
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    if (2 * i < lo || 2 * i >= hi) x[i].x = 0.f;
                    if (2 * i + 1 < lo || 2 * i + 1 >= hi) x[i].y = 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const __half2 hi = __floats2half2_rn(x[i].x, x[i].y);
                const float2 back = __half22float2(hi), rest = add_pair(x[i], make_float2(-back.x, -back.y));
                const __half2 lo = __floats2half2_rn(rest.x, rest.y);
                v[0][i] = *(const uint32_t*)&hi, v[1][i] = *(const uint32_t*)&lo;
            }
            tmem_store_32(my_s, v[0]);
            tmem_store_32(my_s + 32u, v[1]);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive(my_p_ready + 8 * b);
        }
        if (used) ok = ok && wait(my_pv_done + 8 * ((n - 1) & 1), (uint32_t)(((n - 1) >> 1) & 1), 88);
        const bool sees = sight.live && (sight.low[0] < sight.high[0] || sight.low[1] < sight.high[1]);
        const bool whole = splits == 1 && !prefix_only;
        if (tile < tiles && ok) {
            float* const part = p.pre + ((int64_t)blockIdx.x * kRows + (threadIdx.x & (kRows - 1))) * (kDim + 4);
            __half* const out = (__half*)p.out + (((int64_t)seq_of(row) * p.tokens + token_of(row)) * p.heads + head * group + row % group) * p.cache.dim;
            const float inverse = 1.f / sum;
#pragma unroll 1
            for (int c = 0; c < kDim / 32; c++) {
                uint32_t o[32];
                if (n > 0) tmem_load_32(my_o + c * 32, o);
                if (row < rows) {
                    if (!whole) {
                        if (n > 0) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *(float4*)(part + c * 32 + i) = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                        }
                    } else if (p.cache.dim % 8 == 0) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            if (c * 32 + i >= p.cache.dim) continue;
                            uint32_t h[4];
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const __half2 pair = __floats2half2_rn(sees ? __uint_as_float(o[i + 2 * q]) * inverse : 0.f, sees ? __uint_as_float(o[i + 2 * q + 1]) * inverse : 0.f);
                                h[q] = *(const uint32_t*)&pair;
                            }
                            *(uint4*)(out + c * 32 + i) = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (c * 32 + i < p.cache.dim) out[c * 32 + i] = __float2half_rn(sees ? __uint_as_float(o[i]) * inverse : 0.f);
                    }
                }
                __syncwarp();
            }
            if (!whole && row < rows) part[kDim] = n > 0 ? reference : kBottom, part[kDim + 1] = n > 0 ? sum : 0.f;
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// The parts of a row, a warp each
template <int DB>
__global__ void __launch_bounds__(256) cache_attention_join_kernel(const __grid_constant__ CacheAttentionParams p) {
    constexpr int kDim = 64 * DB, kEach = kDim / 32;   // channels of a lane
    pdl_enter();
    const int group = p.heads / p.cache.heads, rows = p.tokens * group, row_tiles = (rows + kRows - 1) / kRows, lane = threadIdx.x & 31;
    const int shared = p.prefix.base ? min(max(*p.prefix_length, 0), p.prefix.capacity) : 0;
    const int64_t index = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);   // of all rows of all sequences and heads
    if (index >= (int64_t)p.cache.seqs * p.cache.heads * rows) return;
    const int row = (int)(index % rows), head = (int)(index / rows % p.cache.heads), seq = (int)(index / rows / p.cache.heads), t = row / group;
    const int64_t item = ((int64_t)seq * p.cache.heads + head) * row_tiles + row_tiles - 1 - row / kRows;
    const float* const part = p.pre + (item * p.splits * kRows + row % kRows) * (kDim + 4);
    const int64_t step = (int64_t)kRows * (kDim + 4);
    // (a part that saw nothing has no sum, and may have written no more than that)
    const float2 mine = lane < p.splits ? __ldcg((const float2*)(part + lane * step + kDim)) : make_float2(kBottom, 0.f);
    const float top = [&] {
        float m = mine.y != 0.f ? mine.x : kBottom;
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        return m;
    }();
    const float factor = mine.y != 0.f ? exp2_approx(mine.x - top) : 0.f;
    float all = mine.y != 0.f ? factor * mine.y : 0.f, v[kEach] = {};
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
#pragma unroll 8
    for (int k = 0; k < p.splits; k++) {
        const float f = __shfl_sync(0xffffffffu, factor, k);
        const bool some = __shfl_sync(0xffffffffu, mine.y, k) != 0.f;
#pragma unroll
        for (int c = 0; c < kEach; c++) {
            const float x = __ldcg(part + k * step + lane * kEach + c);
            v[c] += some ? f * x : 0.f;
        }
    }
    const int64_t at = (int64_t)p.start[seq] + t, last = min(at + shared, (int64_t)shared + p.cache.capacity - 1);
    const bool sees = at >= 0 && (p.count == nullptr || t < p.count[seq]) && (p.window == 0 || last > at + shared - p.window);
    __half* const out = (__half*)p.out + (((int64_t)seq * p.tokens + t) * p.heads + head * group + row % group) * p.cache.dim + lane * kEach;
#pragma unroll
    for (int c = 0; c < kEach; c++)
        if (lane * kEach + c < p.cache.dim) out[c] = __float2half_rn(sees ? v[c] / all : 0.f);
}

}  // namespace

// `many` 1: all of a sequence's keys, 2: the prefix for the rows of all sequences
CacheRowsPlan cache_attention_rows_plan(const CacheAttentionParams& p, int many) {
    CacheRowsPlan plan{};
    const int64_t rows = (int64_t)(many == 2 ? p.cache.seqs : 1) * p.tokens * (p.heads / p.cache.heads), dim = (p.cache.dim + 63) / 64 * 64;
    plan.items = (rows + kRows - 1) / kRows * p.cache.heads * (many == 2 ? 1 : p.cache.seqs);
    const int64_t blocks = (p.prefix.dim ? (p.prefix.capacity + kKeys - 1) / kKeys : 0) + (many == 2 ? 0 : (p.cache.capacity + kKeys - 1) / kKeys);
    // parts of 8 blocks and more, for as many CTAs as there are SMs (of a prefix: as many as cache_attention_kernel takes)
    plan.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({148 / plan.items, blocks / 8, many == 2 ? 8 : 32}));
    plan.part_floats = plan.splits > 1 || many == 2 ? plan.items * plan.splits * kRows * (dim + 4) : 0;
    return plan;
}

int launch_cache_attention_rows(const CacheAttentionParams& p, cudaStream_t stream) {
    const int blocks = (p.cache.dim + 63) / 64;
    static bool done[2][64];
    static std::mutex mu;
    const int err = blocks == 1 ? allow_shared(cache_attention_rows_kernel<1>, RowsGeo<1>::kShared, done[0], mu)
                                : allow_shared(cache_attention_rows_kernel<2>, RowsGeo<2>::kShared, done[1], mu);
    if (err != 0) return err;
    const dim3 grid((unsigned)(p.row_items * p.splits));
    if (blocks == 1) launch_pdl(cache_attention_rows_kernel<1>, grid, dim3(kThreads), RowsGeo<1>::kShared, stream, p);
    else launch_pdl(cache_attention_rows_kernel<2>, grid, dim3(kThreads), RowsGeo<2>::kShared, stream, p);
    if (p.many == 1 && p.splits > 1) {
        const int64_t rows = (int64_t)p.cache.seqs * p.tokens * p.heads;
        launch_pdl(blocks == 1 ? cache_attention_join_kernel<1> : cache_attention_join_kernel<2>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream, p);
    }
    return (int)cudaGetLastError();
}

}  // namespace kn
