// Attention of new tokens against a decoder's cache.
//
//   p = prefix length + start[s] + t,   score_j = scale q . k_j,   cap tanh(score / cap),   - slope (p - j),
//   out = sum_j softmax(score)_j v_j   over   0 <= p - j < window
//
// Bound by the cache's bytes (one token of 64 sequences of up to 8192 positions, 32 / 8 heads of 128 channels: 694 MB against 5.4
// GFLOP), so the kernel is built around reading them once, evenly and without a pause:
//
//  * Query rows that share keys (heads / cache heads x tokens) are the 8 or 16 columns of a matrix product; more are further items.
//  * The work of all items (sequence, head of the cache, rows) is one list of units of kWarps tiles of 16 positions, cut into equal
//    ranges, one per CTA, by the lengths that the sequences have now: a batch of any lengths keeps every SM busy to the end.  Where a
//    cut falls inside an item its CTAs leave their parts in memory and the last to arrive joins them, in the order of the keys: the
//    result does not depend on who is last.
//  * A warp takes one tile of each unit and has its own ring of shared memory that bulk copies fill ahead of it, across the ends of
//    items; warps meet only at an item's end.
//  * Products are keys . queries^T and values^T . weights^T: 16 positions, or 16 channels, by 8 rows, so that the few rows of one
//    token fill them.  Between the two the weights are transposed in registers.  The order of channels and positions inside a
//    product is free: both are chosen so that a lane's operands are 16 bytes of one row of shared memory.
//  * Numbers of 8 bits become f16 exactly (two instructions for two of them, cache.cuh), their scales multiply scores and weights
//    in f32.  Weights, and f32 queries, are taken as two halves of 11 bits, a product each, and keep 22.
//
// Measured, step alone: 133 us for the sizes above (5.2 TB/s, 80 % of a copy), 59 us for one sequence of 131072 (276.8 MB, 72 %; 54 of
// three executors side by side, whose ends overlap).
//
// Softmax statistics and sums are f32.  A row's reference is not its maximum but one that no score is more than 2^8 above: it moves
// rarely, and only then do lanes compare notes.
//
// A 16-bit cache may hold infinities and NaN (numbers of f32 past 65504 are such).  A product would make NaN of an infinity and a weight's lower
// half, so every tile is asked whether its values are finite, and one that says no takes the code of tiles that rows see in part, which
// keeps them out of the products and adds them row by row.  What the question costs, without -> with: 64 x 8192 216.4 -> 219.9 us,
// 24 x 1500 f32 30.8 -> 32.0, 5 tokens of 256 channels 84.5 -> 93.4, 256 tokens of 2 x 2048 178 -> 189 (step alone, L2 warm).
#include "cache.cuh"
#include "launch.cuh"
#include "tc_ptx.cuh"

#include <type_traits>

namespace kn {

namespace {

constexpr int kTile = kCacheTile;
constexpr uint32_t kWaitCode = 71;
constexpr float kBottom = -3.402823466e38f;   // a row's reference before it has seen a score
constexpr float kAbove = 8.f;                 // of a score over its row's reference, as a power of two
constexpr float kWeight = 128.f;              // what a weight of 1 is in f16: up to 2^15 with kAbove, down to 2^-21 with all its bits

// COLS: 8 query rows, once or twice.  F32Q: f32 queries
template <bool HALF, bool F32Q, int COLS, int DB>   // storage of 16 bits; 64-channel blocks
struct Geo {
    static constexpr int kDim = 64 * DB, kRowBytes = kDim * (HALF ? 2 : 1);
    static constexpr int kRows = 8 * COLS;                   // query rows of an item
    static constexpr int kStage = 2 * kTile * kRowBytes + (HALF ? 0 : 128);
    // as many warps as registers and shared memory allow (3 stages and more): 16 a SM, 12 with two times 8 rows of 128 channels
    static constexpr int kWarps = kRowBytes >= 512 ? 4 : kRowBytes == 128 && COLS == 2 ? 12 : 8;
    static constexpr int kPerSm = kRowBytes < 128 || (kRowBytes == 128 && COLS == 1) ? 2 : 1;
    static constexpr int kE = HALF ? 8 : DB % 2 == 0 ? 16 : 8;   // channels of a value row that a lane takes at a time
    static constexpr int kBlocks = kDim / (8 * kE);
    static constexpr int kGroups = kRowBytes / 64;           // 64-byte groups of a key row: one 16-byte chunk a lane
    static constexpr int kSteps = HALF ? 2 : 4;              // products of 16 channels in one
    // floats: what the warps exchange at a time, 32 channels of all rows, or 128 where two stages leave room
    static constexpr int kJoinTimes = kPerSm == 1 && kRowBytes >= 256 && kRowBytes != 384 && COLS == 2 ? 4 : 1;
    static constexpr int kJoin = kWarps * kRows * 32 * kJoinTimes;
    static constexpr int kRoom = (220 * 1024 / kPerSm - kJoin * 4) / (kWarps * kStage);
    static constexpr int kStages = kRoom < 4 ? kRoom : 4;
    static constexpr int kShared = kWarps * kStages * kStage + kJoin * 4;
    static_assert(kStages >= 2, "shared memory");
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 8 x 8 numbers of 16 bits, a row per four lanes, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*(const __half2*)&x); }
// Bytes K and K + 1 of `w`, whole numbers + 128, as two f16
template <int K>
__device__ __forceinline__ uint32_t two_of(uint32_t w) {
    const uint32_t raised = __byte_perm(w, 0x64646464u, K == 0 ? 0x4140 : 0x4342);   // 1024 + byte
    const uint32_t off = 0x64806480u;                                                // 1152
    const __half2 h = __hsub2(*(const __half2*)&raised, *(const __half2*)&off);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What the rows of a sequence see, in tiles: first those of the prefix, then its own
struct Span {
    int64_t start;           // of its first new token, behind the prefix
    int t_lo, t_hi;          // new tokens that count
    int pre_tile, own_tile;  // first tiles
    int pre_tiles, tiles;    // the prefix's, all
};

__device__ __forceinline__ Span span_of(const CacheAttentionParams& p, int s, int shared) {
    Span z;
    z.start = p.start[s];
    z.t_hi = p.count ? min(max(p.count[s], 0), p.tokens) : p.tokens;
    z.t_lo = (int)min(max(-z.start, (int64_t)0), (int64_t)p.tokens);
    const int64_t seen = p.window > 0 ? shared + z.start + z.t_lo - p.window + 1 : 0;   // first position that any row sees
    const int64_t own_first = max(seen - shared, (int64_t)0), own_end = min(z.start + z.t_hi, (int64_t)p.cache.capacity);
    const int64_t pre_first = max(seen, (int64_t)0);
    z.pre_tile = z.own_tile = z.pre_tiles = z.tiles = 0;
    if (z.t_lo >= z.t_hi) return z;
    if (pre_first < shared && p.many != 2) {   // (else others see to the prefix)
        z.pre_tile = (int)(pre_first / kTile);
        z.pre_tiles = (shared + kTile - 1) / kTile - z.pre_tile;
    }
    z.tiles = z.pre_tiles;
    if (own_first < own_end) {
        z.own_tile = (int)(own_first / kTile);
        z.tiles += (int)((own_end + kTile - 1) / kTile) - z.own_tile;
    }
    return z;
}

// The tiles of one run (0: the prefix, 1: a sequence's own) that a warp has in units [from, until) of an item: the first, as the run
// counts them, and how many; each is `warps` behind the one before
struct Run {
    int first, count;
};
__device__ __forceinline__ Run run_of(const Span& z, int run, int from, int until, int warp, int warps) {
    const int lo = run ? z.pre_tiles : 0, hi = min(run ? z.tiles : z.pre_tiles, until * warps);   // in the list of both
    int t = from * warps + warp;
    if (t < lo) t += (lo - t + warps - 1) / warps * warps;
    return {(run ? z.own_tile : z.pre_tile) + t - lo, t < hi ? (hi - t + warps - 1) / warps : 0};
}

template <bool HALF, bool F32Q, int COLS, int DB>
__global__ void __launch_bounds__(Geo<HALF, F32Q, COLS, DB>::kWarps * 32, Geo<HALF, F32Q, COLS, DB>::kPerSm)
cache_attention_kernel(const __grid_constant__ CacheAttentionParams p) {
    using G = Geo<HALF, F32Q, COLS, DB>;
    constexpr int kWarps = G::kWarps, kThreads = kWarps * 32, kStages = G::kStages, kE = G::kE, RB = G::kRowBytes, kDim = G::kDim;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) unsigned long long bars[kWarps * kStages];
    __shared__ int scan_sum[kWarps], scan_at, scan_seq, abandon, is_last;
    __shared__ int64_t row_to[G::kRows];
    __shared__ bool row_sees[G::kRows];
    __shared__ float row_most[kWarps][G::kRows], row_sum[kWarps][G::kRows], row_all[G::kRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    float* const join = (float*)(smem + kWarps * kStages * G::kStage);
    uint8_t* const ring = smem + warp * kStages * G::kStage;
    const uint32_t ring_at = tcp::smem_u32(ring), bar_at = tcp::smem_u32(&bars[warp * kStages]);
    if (lane == 0)
        for (int i = 0; i < kStages; i++) tcp::mbar_init(bar_at + 8 * i, 1);
    if (threadIdx.x == 0) abandon = 0, scan_seq = -1, scan_at = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_enter();
    const int group = p.heads / p.cache.heads, rows = group * p.tokens;
    const int row_tiles = (rows + G::kRows - 1) / G::kRows, items = p.cache.heads * row_tiles;   // of a sequence
    const int shared = p.prefix.base ? min(max(*p.prefix_length, 0), p.prefix.capacity) : 0;
    __syncthreads();

    // ---- what this CTA does: `todo` units from unit first_from of item first_item of sequence first_seq on
    const auto units_of = [&](const Span& z) { return max(1, (z.tiles + kWarps - 1) / kWarps); };
    const auto units_at = [&](int s) { return units_of(span_of(p, s, shared)); };
    // sum over the sequences of a chunk up to and with this thread's, of f(units of an item)
    const auto scan = [&](int chunk, int& mine, auto f) {
        const int s = chunk * kThreads + threadIdx.x;
        mine = s < p.cache.seqs ? f(units_at(s)) * items : 0;
        int up = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += w;
        }
        __syncthreads();
        if (lane == 31) scan_sum[warp] = up;
        __syncthreads();
        for (int w = 0; w < warp; w++) up += scan_sum[w];
        return up;
    };
    // the sequence in whose part of that sum `x` lies
    const auto find = [&](int x, auto f) {
        int front = 0;
        for (int i = 0; i * kThreads < p.cache.seqs; i++) {
            int mine;
            const int at = front + scan(i, mine, f) - mine;
            if (at <= x && x < at + mine) scan_seq = i * kThreads + threadIdx.x, scan_at = at;
            for (int w = 0; w < kWarps; w++) front += scan_sum[w];
        }
        __syncthreads();
    };
    const int grid = gridDim.x;
    int total = 0, most = 0;   // units; in a part, see below
    // Up to 64 sequences every warp shares out for itself, two a lane, without a barrier.  (Step alone, all barriers and equal ranges -> this:
    // 16 x 2048 26.6 -> 20.8 us, 64 x 300 28.4 -> 28.1, 64 x 8192 135.5 -> 133.3)
    const bool few = p.cache.seqs <= 64;
    int mine[2] = {0, 0};
    if (few) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (2 * lane + i < p.cache.seqs) mine[i] = units_at(2 * lane + i);
        total = __reduce_add_sync(0xffffffffu, mine[0] + mine[1]) * items;
        // Items in whole parts of up to `most` units, one part per CTA, where that is hardly longer than equal ranges: a CTA does not change
        // items then.  (A change and a join are about as long as two units.  Step alone, equal ranges -> parts: 16 x 512 19.6 -> 14.5 us,
        // 16 x 2048 25.8 -> 20.8, one of 131072 69.1 -> 58.7; 64 x 8192 133 and 133.)
        const int least = (total + grid - 1) / grid;
        for (int q = least; q <= least + 2 && most == 0; q++)
            if (__reduce_add_sync(0xffffffffu, (mine[0] + q - 1) / q + (mine[1] + q - 1) / q) * items <= grid) most = q;
    } else {
        for (int i = 0; i * kThreads < p.cache.seqs; i++) {
            int one;
            scan(i, one, [](int n) { return n; });
            for (int w = 0; w < kWarps; w++) total += scan_sum[w];
        }
    }
    // in equal ranges the first `longer` CTAs have one unit more
    const int ctas = min(grid, total), each = total / ctas, longer = total - each * ctas;
    const auto cta_of = [&](int u) { return u < longer * (each + 1) ? u / (each + 1) : longer + (u - longer * (each + 1)) / each; };
    const auto start_of = [&](int b) { return b * each + min(b, longer); };
    const int u0 = start_of(blockIdx.x);   // (equal ranges)
    if (most == 0 && (int)blockIdx.x >= ctas) return;
    int first_seq, first_units, place;   // where the CTA begins: its place among the units (or parts) of that sequence
    if (few) {
        const auto parts_of = [&](int n) { return (most > 0 ? (n + most - 1) / most : n) * items; };
        const int x = most > 0 ? (int)blockIdx.x : u0, a = parts_of(mine[0]), b = parts_of(mine[1]);
        int front = a + b;
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, front, o);
            if (lane >= o) front += w;
        }
        front -= a + b;
        const uint32_t hit = __ballot_sync(0xffffffffu, front <= x && x < front + a + b);
        if (hit == 0) return;
        const int from = __ffs(hit) - 1, second = x >= front + a ? 1 : 0;
        first_seq = __shfl_sync(0xffffffffu, 2 * lane + second, from);
        first_units = __shfl_sync(0xffffffffu, mine[second], from);
        place = __shfl_sync(0xffffffffu, x - front - (second ? a : 0), from);
    } else {
        find(u0, [](int n) { return n; });
        first_seq = scan_seq;
        first_units = units_at(first_seq);
        place = u0 - scan_at;
    }
    int first_item, first_from, todo, part = 0;
    if (most > 0) {
        const int parts = (first_units + most - 1) / most;
        first_item = place / parts;
        part = place - first_item * parts;
        const int least = first_units / parts, more = first_units - least * parts;   // the first `more` parts have one unit more
        first_from = part * least + min(part, more);
        todo = least + (part < more ? 1 : 0);
    } else {
        first_item = place / first_units;
        first_from = place - first_item * first_units;
        todo = each + ((int)blockIdx.x < longer ? 1 : 0);
    }
    int issued = 0, consumed = 0;

    // ---- bulk copies of this warp's tiles, as far ahead as the ring goes: run after run, item after item
    Span next_span = span_of(p, first_seq, shared);
    int next_s = first_seq, next_units = units_of(next_span), next_run = -1, next_left = 0;
    int next_item = first_item, next_from = first_from, next_todo = todo, next_stage = 0;
    const uint8_t* next_tile = nullptr;
    const auto issue = [&]() {
        while (issued - consumed < kStages) {
            while (next_left == 0) {   // the next run that has a tile for this warp
                if (next_run == 1) {
                    next_todo -= next_units - next_from;
                    next_from = 0;
                    next_run = -1;
                    if (++next_item == items) {
                        next_item = 0;
                        if (next_todo > 0) {
                            next_span = span_of(p, ++next_s, shared);
                            next_units = units_of(next_span);
                        }
                    }
                }
                if (next_todo <= 0) return;
                const int until = min(next_units, next_from + next_todo);
                const Run r = run_of(next_span, ++next_run, next_from, until, warp, kWarps);
                next_left = r.count;
                const CacheParams& k = next_run ? p.cache : p.prefix;
                next_tile = cache_tile(k, (next_run ? (int64_t)next_s * k.heads : 0) + (row_tiles == 1 ? next_item : next_item / row_tiles), r.first * kTile);
            }
            if (tcp::elect_one()) {
                tcp::mbar_expect_tx(bar_at + 8 * next_stage, G::kStage);
                bulk_load(ring_at + next_stage * G::kStage, next_tile, G::kStage, bar_at + 8 * next_stage);
            }
            next_stage = next_stage + 1 == kStages ? 0 : next_stage + 1;
            next_tile += kWarps * G::kStage;
            next_left--;
            issued++;
        }
    };
    // (the same answer for all lanes, also where the wait runs out)
    int stage_at = 0, phase = 0;   // of the tile that is waited for
    const auto wait_tile = [&]() { return __all_sync(0xffffffffu, tcp::mbar_wait(bar_at + 8 * stage_at, phase, &abandon, p.status, kWaitCode)); };
    const auto done_tile = [&]() {
        consumed++;
        if (++stage_at == kStages) stage_at = 0, phase ^= 1;
    };

    // ---- where this lane's operands lie in a tile: keys at positions token[0] and token[1], a row of the first product each; values at
    // the positions that are columns 2 c, 2 c + 1, 2 c + 8 and 2 c + 9 of the second
    const int token[2] = {4 * (g >> 1) + ((g & 1) + (g >> 1) & 3), 4 * (g >> 1) + (2 + (g & 1) + (g >> 1) & 3)};
    int key_at[2], value_at[4], value_token[4];
#pragma unroll
    for (int j = 0; j < 2; j++) key_at[j] = token[j] * RB + ((c ^ cache_swizzle(RB, token[j])) << 4);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        value_token[r] = 4 * c + ((r + c) & 3);
        const int x = cache_swizzle(RB, value_token[r]);
        value_at[r] = kTile * RB + value_token[r] * RB + (kE * (HALF ? 2 : 1) == 16 ? (g ^ x) << 4 : (((g >> 1) ^ x) << 4) + 8 * (g & 1));
    }
    const float log2e = 1.4426950408889634f;
    const bool capped = p.softcap > 0.f;
    // 2^x of how far a reference lies under another; of 16-bit caches no 0, so that a sum that is infinite stays so
    const auto under = [](float x) { return HALF ? fmaxf(exp2_fast(x), 1.17549435e-38f) : exp2_fast(x); };

    bool dead = false;
    Span span = next_span;
    int u = u0;   // (equal ranges)
    for (int seq = first_seq, item = first_item, first_unit = first_from; todo > 0;) {
        // ---- an item, or the part of it that is this CTA's: units [first_unit, until) of its own
        const int head = row_tiles == 1 ? item : item / row_tiles, row0 = row_tiles == 1 ? 0 : (item % row_tiles) * G::kRows;
        const int units = units_of(span);
        const int until = min(units, first_unit + todo);
        if (!dead) issue();
        // queries: row g of each eight
        uint32_t q[COLS][F32Q ? 2 : 1][G::kGroups][G::kSteps][2];
        float factor[COLS][2];   // of this lane's columns, 2 c and 2 c + 1: what a sum of products times the key's scale is multiplied with
#pragma unroll
        for (int n = 0; n < COLS; n++) {
            constexpr int kN = HALF ? 8 : 16;   // channels of a lane's chunk
            const int row = row0 + 8 * n + g;
            const bool has = row < rows;
            const int64_t from = seq * p.q_strides[0] + (row / group) * p.q_strides[1] + (head * group + row % group) * p.q_strides[2];
            float amount = 1.f;
            int by = 0;
            if constexpr (F32Q) {
                // brought near 2^14, so that the lower half keeps its bits in f16
                const float* at = (const float*)p.query + from;
                float most = 0.f;
                if (has && p.q_wide) {
#pragma unroll
                    for (int d = 4 * c; d < kDim; d += 16)
                        if (d < p.cache.dim) {
                            const float4 x = *(const float4*)(at + d);
                            most = fmaxf(most, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
                        }
                } else if (has) {
                    for (int d = c; d < p.cache.dim; d += 4) most = fmaxf(most, fabsf(at[d * p.q_strides[3]]));
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const int e = (__float_as_int(most) >> 23) - 127;   // (of an infinity 128: the row's result is NaN then)
                by = most > 0.f ? min(max(13 - e, -126), 126) : 0;
                amount = __int_as_float((127 + by) << 23);
            }
#pragma unroll
            for (int k = 0; k < 2; k++) factor[n][k] = p.scale * (F32Q ? __int_as_float((127 - __shfl_sync(0xffffffffu, by, 4 * (2 * c + k))) << 23) : 1.f);
#pragma unroll
            for (int k = 0; k < G::kGroups; k++) {
                const int d0 = k * 4 * kN + c * kN;   // channels d0 to d0 + kN - 1 of the row
                if constexpr (F32Q) {
                    const float* at = (const float*)p.query + from;
                    float x[kN];
#pragma unroll
                    for (int i = 0; i < kN; i++) x[i] = 0.f;
                    if (has && p.q_wide) {
#pragma unroll
                        for (int i = 0; i < kN; i += 4)
                            if (d0 + i < p.cache.dim) *(float4*)(x + i) = *(const float4*)(at + d0 + i);
                    } else if (has) {
#pragma unroll
                        for (int i = 0; i < kN; i++)
                            if (d0 + i < p.cache.dim) x[i] = at[(d0 + i) * p.q_strides[3]];
                    }
#pragma unroll
                    for (int i = 0; i < kN; i += 2) {
                        const uint32_t hi = pack(x[i] * amount, x[i + 1] * amount);
                        const float2 back = unpack(hi);
                        q[n][0][k][i >> 2][i >> 1 & 1] = hi;
                        q[n][F32Q ? 1 : 0][k][i >> 2][i >> 1 & 1] = pack(x[i] * amount - back.x, x[i + 1] * amount - back.y);
                    }
                } else {
                    const __half* at = (const __half*)p.query + from;
                    uint32_t x[kN / 2];
#pragma unroll
                    for (int i = 0; i < kN / 2; i++) x[i] = 0;
                    if (has && p.q_wide) {
#pragma unroll
                        for (int i = 0; i < kN / 2; i += 4)
                            if (d0 + 2 * i < p.cache.dim) {
                                const uint4 raw = *(const uint4*)(at + d0 + 2 * i);
                                x[i] = raw.x, x[i + 1] = raw.y, x[i + 2] = raw.z, x[i + 3] = raw.w;
                            }
                    } else if (has) {
#pragma unroll
                        for (int i = 0; i < kN; i++)
                            if (d0 + i < p.cache.dim) x[i >> 1] |= (uint32_t)__half_as_ushort(at[(d0 + i) * p.q_strides[3]]) << (16 * (i & 1));
                    }
#pragma unroll
                    for (int i = 0; i < kN / 2; i++) q[n][0][k][i >> 1][i & 1] = x[i];
                }
            }
        }
        // this lane's columns
        float slope[COLS][2];
        int t_of[COLS][2];
#pragma unroll
        for (int n = 0; n < COLS; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int row = row0 + 8 * n + 2 * c + k;
                t_of[n][k] = row / group;
                slope[n][k] = p.slopes && row < rows ? p.slopes[head * group + row % group] * log2e : 0.f;
                if (!capped) factor[n][k] *= log2e;
                else factor[n][k] *= (F32Q ? 1.f : 2.f * log2e) / p.softcap;
            }
        const float cap = p.softcap * log2e;
        // rows of the item that count
        const int t_first = max(row0 / group, span.t_lo), t_last = min((min(row0 + G::kRows, rows) - 1) / group, span.t_hi - 1);

        float o[COLS][G::kBlocks][kE / 2][4];
        float ref[COLS][2], sum[COLS][2];
#pragma unroll
        for (int n = 0; n < COLS; n++) {
#pragma unroll
            for (int b = 0; b < G::kBlocks; b++)
#pragma unroll
                for (int i = 0; i < kE / 2; i++) o[n][b][i][0] = o[n][b][i][1] = o[n][b][i][2] = o[n][b][i][3] = 0.f;
            ref[n][0] = ref[n][1] = kBottom;
            sum[n][0] = sum[n][1] = 0.f;
        }
        float value_ref = 0.f, weight_scale = HALF ? kWeight : 0.f;   // values' scales are counted in `value_ref`, a power of two above all

#pragma unroll 1
        for (int run = 0; run < 2 && !dead; run++) {
            Run tiles = run_of(span, run, first_unit, until, warp, kWarps);
            if (tiles.count == 0) continue;
            // In positions of the run: a row at `zero` + t sees [low, high); all rows see [all_lo, all_hi), one at least [any_lo, any_hi)
            const auto cut = [](int64_t x) { return (int)max(min(x, (int64_t)(1 << 30)), (int64_t)-(1 << 30)); };
            const int64_t zero = span.start + (run ? 0 : shared), end = run ? p.cache.capacity : shared;
            const auto high = [&](int t) { return cut(min(zero + t + 1, end)); };
            const auto low = [&](int t) { return p.window > 0 ? cut(zero + t - p.window + 1) : -(1 << 30); };
            const int all_hi = high(t_first), any_hi = high(t_last), all_lo = low(t_last), any_lo = low(t_first);
            // whether some value of a tile is no finite number: 0 times all others is 0
            const auto holds_others = [&](const uint8_t* stage) {
                const __half2 zero = __float2half2_rn(0.f);
                __half2 none[4] = {zero, zero, zero, zero};
#pragma unroll
                for (int i = 0; i < kTile * RB / 512; i++) {
                    const uint4 raw = *(const uint4*)(stage + kTile * RB + (32 * i + lane) * 16);
                    none[0] = __hfma2(*(const __half2*)&raw.x, zero, none[0]), none[1] = __hfma2(*(const __half2*)&raw.y, zero, none[1]);
                    none[2] = __hfma2(*(const __half2*)&raw.z, zero, none[2]), none[3] = __hfma2(*(const __half2*)&raw.w, zero, none[3]);
                }
                const __half2 all = __hadd2(__hadd2(none[0], none[1]), __hadd2(none[2], none[3]));
                return __any_sync(0xffffffffu, (*(const uint32_t*)&all & 0x7fff7fffu) != 0) != 0;
            };
            // one tile, with or without positions that some row does not see (and values that are no finite numbers)
            const auto do_tile = [&](auto tag, int at, const uint8_t* stage) {
                constexpr bool MASKED = decltype(tag)::value;
                // ---- scores: 16 positions x 8 rows
                // (8 rows: two sums, of every other group of channels, so that a product waits for the one before the last; of f32 queries and
                // keys that may be infinite the queries' upper and lower halves)
                constexpr bool TWO = COLS == 1 && G::kGroups > 1, BY_HALF = HALF && F32Q;
                static_assert(TWO || !BY_HALF);
                float s[COLS][4] = {}, other[4] = {};
#pragma unroll
                for (int k = 0; k < G::kGroups; k++) {
                    uint32_t w[2][4];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint4 raw = *(const uint4*)(stage + (RB % 128 == 0 ? (key_at[j] ^ ((k & 1) << 6)) + 128 * (k >> 1) : key_at[j] + 64 * k));
                        w[j][0] = raw.x, w[j][1] = raw.y, w[j][2] = raw.z, w[j][3] = raw.w;
                    }
#pragma unroll
                    for (int st = 0; st < G::kSteps; st++) {
                        uint32_t a[4];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            a[j] = HALF ? w[j][(2 * st) & 3] : two_of<0>(w[j][st]);
                            a[2 + j] = HALF ? w[j][(2 * st + 1) & 3] : two_of<2>(w[j][st]);
                        }
#pragma unroll
                        for (int n = 0; n < COLS; n++)
#pragma unroll
                            for (int half = 0; half < (F32Q ? 2 : 1); half++) mma(TWO && (BY_HALF ? half : k & 1) ? other : s[n], a, q[n][half][k][st][0], q[n][half][k][st][1]);
                    }
                }
                if constexpr (TWO) {
#pragma unroll
                    for (int i = 0; i < 4; i++)   // (an infinite key has its sign from the upper half)
                        if (!BY_HALF || fabsf(s[0][i]) < INFINITY) s[0][i] += other[i];
                }
                float key_scale[2] = {1.f, 1.f}, value_scale[2] = {1.f, 1.f};
                if constexpr (!HALF) {
                    const float* scales = (const float*)(stage + 2 * kTile * RB);
#pragma unroll
                    for (int j = 0; j < 2; j++) key_scale[j] = scales[token[j]], value_scale[j] = scales[kTile + token[j]];
                }
                // s[n][2 j + k]: position token[j], row 2 c + k
#pragma unroll
                for (int n = 0; n < COLS; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[n][i] *= HALF ? factor[n][i & 1] : key_scale[i >> 1] * factor[n][i & 1];
                if (capped) {
                    // tanh(y) = 1 - 2 / (1 + e^(2y)): off by 2^-22 of the cap, which f32 results do not take
#pragma unroll
                    for (int n = 0; n < COLS; n++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if constexpr (F32Q) s[n][i] = cap * tanhf(s[n][i]);
                            else s[n][i] = cap - __fdividef(2.f * cap, 1.f + exp2_fast(tcp::min_keeping_nan(s[n][i], 126.f)));
                        }
                }
                if (p.slopes) {
                    // (of sequences behind the capacity not from their positions: all scores of a row are higher by as much then, so that f32 holds
                    // them.  Kept out of registers between tiles)
                    int away = cut(min(span.start, (int64_t)p.cache.capacity - 1)) + (run ? 0 : shared) - at;
                    asm volatile("" : "+r"(away));
#pragma unroll
                    for (int n = 0; n < COLS; n++)
#pragma unroll
                        for (int i = 0; i < 4; i++) s[n][i] -= slope[n][i & 1] * (float)(away + t_of[n][i & 1] - token[i >> 1]);   // (positions may be past 2^24, where f32 are two apart)
                }
                bool hidden[COLS][4] = {};
                if constexpr (MASKED) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int key = at + token[j];
#pragma unroll
                        for (int n = 0; n < COLS; n++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                hidden[n][2 * j + k] = key < low(t_of[n][k]) || key >= high(t_of[n][k]);
                                if (hidden[n][2 * j + k]) s[n][2 * j + k] = -INFINITY;
                            }
                        if (!HALF && (key < any_lo || key >= any_hi)) value_scale[j] = 0.f;
                    }
                }
                // ---- references: of the rows, and of the values' scales
                bool moves = !HALF && fmaxf(value_scale[0], value_scale[1]) > value_ref;
                float above[COLS][4];   // scores, from the reference on
#pragma unroll
                for (int n = 0; n < COLS; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        above[n][i] = __fsub_rn(s[n][i], ref[n][i & 1]);   // (0 for the highest itself, whose weight is 1 to the last bit)
                        moves = moves || above[n][i] > kAbove;
                    }
                if (__any_sync(0xffffffffu, moves)) {
                    const auto of_column = [](float v) {   // over the eight lanes of a column
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                        return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                    };
                    float shrink = 1.f;
                    if constexpr (!HALF) {
                        const float top = of_column(fmaxf(value_scale[0], value_scale[1]));
                        if (top > value_ref) {
                            // (the next power of two, but none so small that its inverse times kWeight overflows)
                            const float next = __int_as_float(min(max((__float_as_int(top) >> 23) + 1, 32), 254) << 23);
                            shrink = value_ref > 0.f ? value_ref / next : 0.f;
                            value_ref = next;
                            weight_scale = kWeight / next;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < COLS; n++) {
                        float keep[2];
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const float top = fmaxf(ref[n][k], of_column(fmaxf(s[n][k], s[n][2 + k])));
                            keep[k] = under(ref[n][k] - top);
                            ref[n][k] = top;
                            above[n][k] = __fsub_rn(s[n][k], top);
                            above[n][2 + k] = __fsub_rn(s[n][2 + k], top);
                            sum[n][k] *= keep[k];
                            keep[k] *= shrink;
                        }
#pragma unroll
                        for (int b = 0; b < G::kBlocks; b++)
#pragma unroll
                            for (int i = 0; i < kE / 2; i++)
#pragma unroll
                                for (int x = 0; x < 4; x++) o[n][b][i][x] *= keep[x & 1];
                    }
                }
                // ---- weights, in two halves, transposed: of row g, positions 2 c and 2 c + 1, 2 c + 8 and 2 c + 9 of the product
                uint32_t weight[COLS][2][2];
#pragma unroll
                for (int n = 0; n < COLS; n++) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float e = exp2_fast(above[n][i]);
                        sum[n][i & 1] += e;
                        w[i] = e * (HALF ? kWeight : value_scale[i >> 1] * weight_scale);
                        if (MASKED && hidden[n][i]) w[i] = 0.f;
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint32_t hi = pack(w[2 * j], w[2 * j + 1]);
                        const float2 back = unpack(hi);
                        weight[n][0][j] = transposed(hi);
                        weight[n][1][j] = transposed(pack(w[2 * j] - back.x, w[2 * j + 1] - back.y));
                    }
                }
                // ---- values^T . weights^T.  f32: the tile's products by themselves, then added (the matrix unit cuts off what it adds)
                const auto times = [&](int b, int i, const uint32_t (&a)[4]) {
#pragma unroll
                    for (int n = 0; n < COLS; n++) {
                        if constexpr (F32Q) {
                            float part[4] = {};
                            mma(part, a, weight[n][1][0], weight[n][1][1]);
                            mma(part, a, weight[n][0][0], weight[n][0][1]);
#pragma unroll
                            for (int x = 0; x < 4; x++) o[n][b][i][x] += part[x];
                        } else {
                            mma(o[n][b][i], a, weight[n][1][0], weight[n][1][1]);
                            mma(o[n][b][i], a, weight[n][0][0], weight[n][0][1]);
                        }
                    }
                };
                bool odd = false;
#pragma unroll
                for (int b = 0; b < G::kBlocks; b++) {
                    constexpr int kWords = kE * (HALF ? 2 : 1) / 4;
                    uint32_t w[4][kWords];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint8_t* from = stage + value_at[r] + b * 8 * kE * (HALF ? 2 : 1);
                        if constexpr (kWords == 4) {
                            const uint4 raw = *(const uint4*)from;
                            w[r][0] = raw.x, w[r][1] = raw.y, w[r][2] = raw.z, w[r][3] = raw.w;
                        } else {
                            const uint2 raw = *(const uint2*)from;
                            w[r][0] = raw.x, w[r][1] = raw.y;
                        }
                    }
                    if constexpr (HALF) {
                        if constexpr (MASKED) {
                            // what nobody sees, and infinities and NaN (added row by row below), count as 0
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const bool seen = at + value_token[r] >= any_lo && at + value_token[r] < any_hi;
#pragma unroll
                                for (int x = 0; x < kWords; x++) {
                                    const bool lo = (w[r][x] & 0x7c00u) == 0x7c00u, hi = (w[r][x] & 0x7c000000u) == 0x7c000000u;
                                    odd = odd || (seen && (lo || hi));
                                    w[r][x] = seen ? w[r][x] & (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0xffffu : 0xffffffffu) : 0u;
                                }
                            }
                        }
#pragma unroll
                        for (int x = 0; x < kWords; x++) {
                            const uint32_t a[4] = {__byte_perm(w[0][x], w[1][x], 0x5410), __byte_perm(w[0][x], w[1][x], 0x7632),
                                                   __byte_perm(w[2][x], w[3][x], 0x5410), __byte_perm(w[2][x], w[3][x], 0x7632)};
                            times(b, x, a);
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < kWords; x++) {
                            const uint32_t lo01 = __byte_perm(w[0][x], w[1][x], 0x5140), lo23 = __byte_perm(w[2][x], w[3][x], 0x5140);
                            const uint32_t hi01 = __byte_perm(w[0][x], w[1][x], 0x7362), hi23 = __byte_perm(w[2][x], w[3][x], 0x7362);
                            const uint32_t a[4] = {two_of<0>(lo01), two_of<2>(lo01), two_of<0>(lo23), two_of<2>(lo23)};
                            times(b, 2 * x, a);
                            const uint32_t a2[4] = {two_of<0>(hi01), two_of<2>(hi01), two_of<0>(hi23), two_of<2>(hi23)};
                            times(b, 2 * x + 1, a2);
                        }
                    }
                }
                if constexpr (HALF && MASKED)
                    if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
                        for (int r = 0; r < 16; r++) {   // position token[r / 8] of lanes 4 (r % 8) and on
                            const int key = at + __shfl_sync(0xffffffffu, r < 8 ? token[0] : token[1], 4 * (r & 7));
                            if (key < any_lo || key >= any_hi) continue;
#pragma unroll
                            for (int n = 0; n < COLS; n++)
#pragma unroll
                                for (int k = 0; k < 2; k++) {
                                    if (key < low(t_of[n][k]) || key >= high(t_of[n][k])) continue;
                                    // (what the weight is does not matter: an infinity stays one)
#pragma unroll
                                    for (int b = 0; b < G::kBlocks; b++)
#pragma unroll
                                        for (int d = 0; d < kE; d++) {
                                            const int chunk = g ^ cache_swizzle(RB, key);
                                            const float v = __half2float(*(const __half*)(stage + (kTile + (key & 15)) * RB + b * 128 + (chunk << 4) + 2 * d));
                                            if (!(fabsf(v) <= 65504.f)) o[n][b][d >> 1][2 * (d & 1) + k] += v;
                                        }
                                }
                        }
                    }
            };
#pragma unroll 1
            for (; tiles.count > 0; tiles.count--, tiles.first += kWarps) {
                if (!wait_tile()) {
                    dead = true;
                    break;
                }
                const int at = tiles.first * kTile;
                const uint8_t* stage = ring + stage_at * G::kStage;
                if (t_first <= t_last) {   // (else rows of nothing but padding, of a sequence that has others)
                    if (at < all_lo || at + kTile > all_hi || (HALF && holds_others(stage))) do_tile(std::true_type{}, at, stage);
                    else do_tile(std::false_type{}, at, stage);
                }
                done_tile();
                __syncwarp();
                issue();
            }
        }

        // ---- the warps' parts become one
#pragma unroll
        for (int n = 0; n < COLS; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float v = sum[n][k];
                for (int x = 4; x < 32; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
                if (g == 0) row_most[warp][8 * n + 2 * c + k] = ref[n][k], row_sum[warp][8 * n + 2 * c + k] = v;
            }
        __syncthreads();
        const auto most_of = [&](int r) {
            float m = row_most[0][r];
            for (int w = 1; w < kWarps; w++) m = fmaxf(m, row_most[w][r]);
            return m;
        };
        if (threadIdx.x < G::kRows) {
            const int r = threadIdx.x;
            const float m = most_of(r);
            float all = 0.f;
            for (int w = 0; w < kWarps; w++) all += row_sum[w][r] * exp2_fast(row_most[w][r] - m);
            // (read behind the next barrier)
            row_all[r] = all;
            const int row = row0 + r, t = row / group;
            const int64_t pos = shared + span.start + t, last = min(pos, (int64_t)shared + p.cache.capacity - 1);
            row_sees[r] = row < rows && t >= span.t_lo && t < span.t_hi && last >= 0 && (p.window == 0 || last > pos - p.window);
            row_to[r] = (((int64_t)seq * p.tokens + t) * p.heads + head * group + row % group) * p.cache.dim;
        }
        float times[COLS][2];
#pragma unroll
        for (int n = 0; n < COLS; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float m = most_of(8 * n + 2 * c + k);
                times[n][k] = under(ref[n][k] - m) * ((HALF ? 1.f : value_ref) / kWeight);
            }
        const bool whole = first_unit == 0 && until == units;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (most > 0 || u == u0 ? 0 : 1);
        float* const partial = p.partial + slot * (G::kRows * (kDim + 2));
        const int rows_here = min(G::kRows, rows - row0);
        // `v` of weight `all`, by reference `ref_of`
        const auto store = [&](int r, int d, float v, float ref_of, float all) {
            if (d >= p.cache.dim) return;
            if (p.many == 2) {   // and what the row sees of the prefix, in up to eight parts (of no sum where it sees nothing)
                const int row = (seq * p.tokens) * group + row0 + r, tiles = (p.cache.seqs * rows + 255) / 256, tile = row / 256;
                const float* const part = p.pre + ((int64_t)(head * tiles + tiles - 1 - tile) * p.splits * 256 + row % 256) * (kDim + 4);
                float2 state[8];
                float x[8], top = all > 0.f ? ref_of : kBottom;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float* const at = part + (int64_t)min(i, p.splits - 1) * 256 * (kDim + 4);
                    state[i] = __ldcg((const float2*)(at + kDim));
                    x[i] = __ldcg(at + d);
                    if (i >= p.splits) state[i].y = 0.f;
                    if (state[i].y != 0.f) top = fmaxf(top, state[i].x);
                }
                const float f = all > 0.f ? exp2_fast(ref_of - top) : all == 0.f ? 0.f : 1.f;
                v *= f, all *= f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float g = exp2_fast(state[i].x - top);
                    if (state[i].y != 0.f) v += g * x[i], all += g * state[i].y;
                }
            }
            v = row_sees[r] ? v / all : 0.f;
            if constexpr (F32Q) ((float*)p.out)[row_to[r] + d] = v;
            else ((__half*)p.out)[row_to[r] + d] = __float2half_rn(v);
        };
        // 32 of a block's channels (four of each lane's) of all rows, or more of them of fewer rows, at a time
        constexpr int kPieces = G::kBlocks * kE / 4;
        const int row_bits = rows_here <= 1 ? 0 : rows_here <= 2 ? 1 : rows_here <= 4 ? 2 : rows_here <= 8 ? 3 : 4;
        const int at_once = min((G::kRows >> row_bits) * G::kJoinTimes, kPieces);   // pieces (all powers of two, or all there are)
#pragma unroll
        for (int piece = 0; piece < kPieces; piece++) {
            const int b = piece / (kE / 4), i0 = piece % (kE / 4) * 2, place = piece % at_once;
#pragma unroll
            for (int n = 0; n < COLS; n++)
#pragma unroll
                for (int k = 0; k < 2; k++)
                    if (8 * n + 2 * c + k < rows_here)
                        *(float4*)(join + (((warp * at_once + place) << row_bits) + 8 * n + 2 * c + k) * 32 + 4 * g) =
                            make_float4(o[n][b][i0][k] * times[n][k], o[n][b][i0][2 + k] * times[n][k], o[n][b][i0 + 1][k] * times[n][k], o[n][b][i0 + 1][2 + k] * times[n][k]);
            if (place != at_once - 1 && piece != kPieces - 1) continue;
            __syncthreads();
            const int from = piece - place;
            for (int at = threadIdx.x; at < (((place + 1) << row_bits) << 5); at += kThreads) {
                const int r = (at >> 5) & ((1 << row_bits) - 1), which = from + (at >> (5 + row_bits));
                if (r >= rows_here) continue;
                const int d = which / (kE / 4) * 8 * kE + kE * ((at & 31) >> 2) + which % (kE / 4) * 4 + (at & 3);
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) v += join[((w * at_once) << (row_bits + 5)) + at];
                if (whole) store(r, d, v, most_of(r), row_all[r]);
                else partial[r * kDim + d] = v;
            }
            __syncthreads();
        }
        if (!whole) {
            if (threadIdx.x < G::kRows) {
                partial[G::kRows * kDim + 2 * threadIdx.x] = most_of(threadIdx.x);
                partial[G::kRows * kDim + 2 * threadIdx.x + 1] = row_all[threadIdx.x];
            }
            // ---- whoever is last joins the item's parts: of CTAs c0 to c1, the first one's its second where it has something in front
            const int item_u = u - first_unit;   // the item's first unit
            int c0, parts;
            bool second = false;
            if (most > 0) {
                parts = (units + most - 1) / most;
                c0 = blockIdx.x - part;
            } else {
                c0 = cta_of(item_u);
                parts = cta_of(item_u + units - 1) - c0 + 1;
                second = start_of(c0) < item_u;
            }
            __syncthreads();
            if (threadIdx.x == 0) {
                __threadfence();   // (of all that the CTA has written: the barrier came first)
                uint32_t* arrived = p.arrived + (int64_t)seq * items + item;
                const uint32_t before = atomicAdd(arrived, 1u);
                is_last = before == (uint32_t)(parts - 1);
                if (is_last) *arrived = 0;
                __threadfence();
            }
            __syncthreads();
            if (is_last) {
                constexpr int64_t kPart = G::kRows * (kDim + 2);
                const float* const first = p.partial + (2 * (int64_t)c0 + (second ? 1 : 0)) * kPart;
                const auto part_of = [&](int i) { return i == 0 ? first : p.partial + 2 * (int64_t)(c0 + i) * kPart; };
                for (int at = threadIdx.x; at < rows_here * kDim / 4; at += kThreads) {
                    const int r = at / (kDim / 4), d = at % (kDim / 4) * 4;
                    float m = kBottom, all = 0.f;
                    float4 v = make_float4(0, 0, 0, 0);
                    for (int i0 = 0; i0 < parts; i0 += 8) {   // eight parts' loads in flight
                        float2 state[8];
                        float4 x[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float* const at_part = part_of(min(i0 + i, parts - 1));
                            state[i] = __ldcg((const float2*)(at_part + G::kRows * kDim + 2 * r));
                            x[i] = __ldcg((const float4*)(at_part + r * kDim + d));
                        }
                        float top = m;
#pragma unroll
                        for (int i = 0; i < 8; i++) top = fmaxf(top, state[i].x);
                        const float keep = under(m - top);
                        m = top;
                        all *= keep, v.x *= keep, v.y *= keep, v.z *= keep, v.w *= keep;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float f = i0 + i < parts ? under(state[i].x - m) : 0.f;
                            if (i0 + i < parts) all += f * state[i].y, v.x += f * x[i].x, v.y += f * x[i].y, v.z += f * x[i].z, v.w += f * x[i].w;
                        }
                    }
                    store(r, d, v.x, m, all);
                    store(r, d + 1, v.y, m, all);
                    store(r, d + 2, v.z, m, all);
                    store(r, d + 3, v.w, m, all);
                }
            }
            __syncthreads();
        }
        u += until - first_unit;
        todo -= until - first_unit;
        first_unit = 0;
        if (++item == items) {
            item = 0;
            if (todo > 0) span = span_of(p, ++seq, shared);
        }
    }
    // (given up: what is under way still writes to this CTA's shared memory)
    if (dead)
        for (const long long since = clock64(); consumed < issued; done_tile()) tcp::mbar_drain(bar_at + 8 * stage_at, phase, since);
}

// f(Geo, kernel) of the variant that takes p
template <bool HALF, bool F32Q, int COLS, typename F>
void with_dim(int blocks, F f) {
    if (blocks == 1) f(Geo<HALF, F32Q, COLS, 1>{}, cache_attention_kernel<HALF, F32Q, COLS, 1>);
    if (blocks == 2) f(Geo<HALF, F32Q, COLS, 2>{}, cache_attention_kernel<HALF, F32Q, COLS, 2>);
    if (blocks == 3) f(Geo<HALF, F32Q, COLS, 3>{}, cache_attention_kernel<HALF, F32Q, COLS, 3>);
    if (blocks == 4) f(Geo<HALF, F32Q, COLS, 4>{}, cache_attention_kernel<HALF, F32Q, COLS, 4>);
}
template <bool HALF, typename F>
void with_rows(const CacheAttentionParams& p, F f) {
    const int blocks = (p.cache.dim + 63) / 64;
    const int64_t rows = (int64_t)p.tokens * (p.heads / p.cache.heads);
    if (!p.half) with_dim<HALF, true, 1>(blocks, f);
    else rows <= 8 ? with_dim<HALF, false, 1>(blocks, f) : with_dim<HALF, false, 2>(blocks, f);
}
template <typename F>
void with_variant(const CacheAttentionParams& p, F f) {
    p.cache.half ? with_rows<true>(p, f) : with_rows<false>(p, f);
}

}  // namespace

CacheAttentionPlan cache_attention_plan(const CacheAttentionParams& p) {
    CacheAttentionPlan plan{};
    with_variant(p, [&](auto geo, auto) {
        using G = decltype(geo);
        const int64_t rows = (int64_t)p.tokens * (p.heads / p.cache.heads);
        plan.items = p.cache.seqs * p.cache.heads * ((rows + G::kRows - 1) / G::kRows);
        const int64_t tiles = (p.cache.capacity + kTile - 1) / kTile + (p.prefix.dim ? (p.prefix.capacity + kTile - 1) / kTile : 0);
        const double most = (double)plan.items * ((tiles + G::kWarps - 1) / G::kWarps);
        plan.units = most;
        plan.grid = (int32_t)std::min<double>(148 * G::kPerSm, most);
        plan.partial_floats = 2ll * plan.grid * G::kRows * (G::kDim + 2);
    });
    return plan;
}

int launch_cache_attention(const CacheAttentionParams& p, cudaStream_t stream) {
    int err = 0;
    if (p.many != 0) err = launch_cache_attention_rows(p, stream);
    if (err != 0 || p.many == 1) return err;
    with_variant(p, [&](auto geo, auto kernel) {
        using G = decltype(geo);
        static bool done[64];
        static std::mutex mu;
        err = allow_shared(kernel, G::kShared, done, mu);
        if (err == 0) launch_pdl(kernel, dim3(p.grid), dim3(G::kWarps * 32), G::kShared, stream, p);
    });
    return err != 0 ? err : (int)cudaGetLastError();
}

}  // namespace kn
