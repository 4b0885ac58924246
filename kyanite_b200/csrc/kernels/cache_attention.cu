// Attention of new tokens against a decoder's cache.
//
//   p = prefix length + start[s] + t,   score_j = scale q . k_j,   cap tanh(score / cap),   - slope (p - j),
//   out = sum_j softmax(score)_j v_j   over   0 <= p - j < window
//
// Bound by the cache's bytes (one token of 64 sequences of 8192 positions, 32 / 8 heads of 128 channels: 694 MB against 5.4 GFLOP), so
// the kernel is built around reading them once, evenly and without a pause:
//
//  * All query rows that share keys (heads / cache heads x tokens) are the 16 rows of a matrix product; more of them are further items.
//  * The work of all items (sequence, head of the cache, 16 rows) is one list of units of kWarps tiles of 16 positions, cut into equal
//    ranges, one per CTA, by the lengths that the sequences have now: a batch of any lengths keeps every SM busy to the end.  Where a
//    cut falls inside an item its CTAs leave their parts in memory and the last to arrive joins them, in the order of the keys: the
//    result does not depend on who is last.
//  * A warp takes one tile of each unit and has its own ring of shared memory that bulk copies fill ahead of it, across the ends of
//    items; warps meet only at an item's end.
//  * Keys of 8 bits become f16 exactly (two instructions for two of them, cache.cuh), their scales multiply scores and weights in f32.
//    Rows of 16 bits of f32 queries are taken as two halves of 11 bits, a row of the product each: scores, and weights split the same
//    way, keep 22 bits.  The order of channels and positions inside a product is free: both are chosen so that a lane's
//    operands are 16 bytes of one row of shared memory.
//
// Softmax statistics and sums are f32; weights are rounded to f16 (once, or to two halves) relative to the row's running maximum.
#include "cache.cuh"
#include "launch.cuh"
#include "tc_ptx.cuh"

namespace kn {

namespace {

constexpr int kTile = 16;      // positions of a tile
constexpr uint32_t kWaitCode = 71;

template <bool HALF, bool F32Q, int DB>   // storage of 16 bits; f32 queries; 64-channel blocks
struct Geo {
    static constexpr int kDim = 64 * DB, kRowBytes = kDim * (HALF ? 2 : 1);
    static constexpr int kRows = F32Q ? 8 : 16;              // query rows of an item
    static constexpr int kStage = 2 * kTile * kRowBytes + (HALF ? 0 : 128);
    static constexpr int kWarps = kRowBytes >= 512 ? 4 : 8;
    static constexpr int kPerSm = kRowBytes <= 128 ? 2 : 1;  // CTAs: those whose registers allow two
    static constexpr int kStages = kRowBytes <= 64 ? 4 : kRowBytes <= 128 ? 2 : kRowBytes == 384 ? 2 : 3;
    static constexpr int kE = HALF ? 8 : DB % 2 == 0 ? 16 : 8;   // channels of a value row that a lane takes at a time
    static constexpr int kBlocks = kDim / (8 * kE);
    static constexpr int kGroups = kRowBytes / 64;           // 64-byte groups of a key row: one 16-byte chunk a lane
    static constexpr int kSteps = HALF ? 2 : 4;              // products of 16 channels in one
    static constexpr int kJoin = kWarps * kRows * 32;        // floats: what the warps exchange at a time, 32 channels
    static constexpr int kShared = kWarps * kStages * kStage + kJoin * 4;
    static_assert(kShared * kPerSm <= 220 * 1024, "shared memory");
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}
// Bytes k and k + 1 of `w`, whole numbers + 128, as two f16
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
    int shared;              // positions of the prefix
    int t_lo, t_hi;          // new tokens that count
    int pre_tile, own_tile;  // first tiles
    int pre_tiles, tiles;    // the prefix's, all
};

__device__ __forceinline__ Span span_of(const CacheAttentionParams& p, int s, int shared) {
    Span z;
    z.start = p.start[s];
    z.shared = shared;
    z.t_hi = p.count ? min(max(p.count[s], 0), p.tokens) : p.tokens;
    z.t_lo = (int)min(max(-z.start, (int64_t)0), (int64_t)p.tokens);
    const int64_t seen = p.window > 0 ? shared + z.start + z.t_lo - p.window + 1 : 0;   // first position that any row sees
    const int64_t own_first = max(seen - shared, (int64_t)0), own_end = min(z.start + z.t_hi, (int64_t)p.cache.capacity);
    const int64_t pre_first = max(seen, (int64_t)0);
    z.pre_tile = z.own_tile = z.pre_tiles = z.tiles = 0;
    if (z.t_lo >= z.t_hi) return z;
    if (pre_first < shared) {
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

// A place in the list of units
struct Cursor {
    Span span;
    int s, item;             // sequence, item of it: head of the cache x rows
    int unit, units;         // of the item
    __device__ __forceinline__ void enter(const CacheAttentionParams& p, int warps) {
        span = span_of(p, s, span.shared);
        units = max(1, (span.tiles + warps - 1) / warps);
    }
    __device__ __forceinline__ void next(const CacheAttentionParams& p, int warps, int items) {
        if (++unit < units) return;
        unit = 0;
        if (++item < items) return;
        item = 0;
        if (++s < p.cache.seqs) enter(p, warps);
    }
};

template <bool HALF, bool F32Q, int DB>
__global__ void __launch_bounds__(Geo<HALF, F32Q, DB>::kWarps * 32, Geo<HALF, F32Q, DB>::kPerSm)
cache_attention_kernel(const __grid_constant__ CacheAttentionParams p) {
    using G = Geo<HALF, F32Q, DB>;
    constexpr int kWarps = G::kWarps, kThreads = kWarps * 32, kStages = G::kStages, kE = G::kE, RB = G::kRowBytes, kDim = G::kDim;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) unsigned long long bars[kWarps * kStages];
    __shared__ int64_t scan_sum[8], scan_at;
    __shared__ int scan_seq, abandon, is_last;
    __shared__ float row_most[kWarps][16], row_sum[kWarps][16], row_all[16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    float* const join = (float*)(smem + kWarps * kStages * G::kStage);
    uint8_t* const ring = smem + warp * kStages * G::kStage;
    const uint32_t ring_at = tcp::smem_u32(ring), bar_at = tcp::smem_u32(&bars[warp * kStages]);
    if (lane == 0)
        for (int i = 0; i < kStages; i++) tcp::mbar_init(bar_at + 8 * i, 1);
    if (threadIdx.x == 0) abandon = 0, scan_seq = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_enter();
    const int group = p.heads / p.cache.heads, rows = group * p.tokens;
    const int row_tiles = (rows + G::kRows - 1) / G::kRows, items = p.cache.heads * row_tiles;
    const int shared = p.prefix.base ? min(max(*p.prefix_length, 0), p.prefix.capacity) : 0;
    __syncthreads();

    // ---- this CTA's range of the list: units [u0, u1), where u0 lies
    const auto scan = [&](int chunk, int64_t& mine) {   // sum over the sequences of a chunk up to and with this thread's
        const int s = chunk * kThreads + threadIdx.x;
        mine = 0;
        if (s < p.cache.seqs) mine = (int64_t)max(1, (span_of(p, s, shared).tiles + kWarps - 1) / kWarps) * items;
        int64_t up = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t w = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += w;
        }
        __syncthreads();
        if (lane == 31) scan_sum[warp] = up;
        __syncthreads();
        for (int w = 0; w < warp; w++) up += scan_sum[w];
        return up;
    };
    const int chunks = (p.cache.seqs + kThreads - 1) / kThreads;
    int64_t total = 0, mine = 0, upto = 0;
    for (int i = 0; i < chunks; i++) {
        upto = scan(i, mine);
        for (int w = 0; w < kWarps; w++) total += scan_sum[w];
    }
    // (as many CTAs as there are units at most: each has some, and counts where an item's parts are joined)
    const int64_t ctas = min((int64_t)gridDim.x, total), u0 = total * blockIdx.x / ctas, u1 = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : u0;
    int64_t front = 0;
    for (int i = 0; i < chunks; i++) {
        if (chunks > 1) upto = scan(i, mine);
        const int64_t at = front + upto - mine;
        if (at <= u0 && u0 < at + mine) scan_seq = i * kThreads + threadIdx.x, scan_at = at;
        for (int w = 0; w < kWarps; w++) front += scan_sum[w];
    }
    __syncthreads();
    if (u0 >= u1) return;
    Cursor ahead, here;
    ahead.s = scan_seq;
    ahead.span.shared = shared;
    ahead.enter(p, kWarps);
    ahead.item = (int)((u0 - scan_at) / ahead.units);
    ahead.unit = (int)((u0 - scan_at) % ahead.units);
    here = ahead;
    int64_t ahead_u = u0, u = u0;
    int issued = 0, consumed = 0;

    // ---- bulk copies of this warp's tiles, as far ahead as the ring goes
    const auto issue = [&]() {
        while (issued - consumed < kStages && ahead_u < u1) {
            const int tile = ahead.unit * kWarps + warp;
            if (tile < ahead.span.tiles) {
                if (lane == 0) {
                    const bool pre = tile < ahead.span.pre_tiles;
                    const CacheParams& k = pre ? p.prefix : p.cache;
                    const int64_t row = cache_row(k, 0, pre ? 0 : ahead.s, ahead.item / row_tiles, (int64_t)kTile * (pre ? ahead.span.pre_tile + tile : ahead.span.own_tile + tile - ahead.span.pre_tiles));
                    const int stage = issued % kStages;
                    const uint32_t to = ring_at + stage * G::kStage, bar = bar_at + 8 * stage;
                    tcp::mbar_expect_tx(bar, G::kStage);
                    bulk_load(to, k.base + row * RB, kTile * RB, bar);
                    bulk_load(to + kTile * RB, k.base + (row + k.part_rows) * RB, kTile * RB, bar);
                    if constexpr (!HALF) {
                        bulk_load(to + 2 * kTile * RB, k.scales + row, 64, bar);
                        bulk_load(to + 2 * kTile * RB + 64, k.scales + row + k.part_rows, 64, bar);
                    }
                }
                issued++;
            }
            ahead.next(p, kWarps, items);
            ahead_u++;
        }
    };

    // (the same answer for all lanes, also where the wait runs out)
    const auto wait_tile = [&]() {
        return __all_sync(0xffffffffu, tcp::mbar_wait(bar_at + 8 * (consumed % kStages), (consumed / kStages) & 1, &abandon, p.status, kWaitCode));
    };

    // ---- where this lane's operands lie in a tile
    const int key_row[2] = {4 * (g >> 1) + ((g & 1) + (g >> 1) & 3), 4 * (g >> 1) + (2 + (g & 1) + (g >> 1) & 3)};
    int key_at[2], value_at[4], token[4];
#pragma unroll
    for (int j = 0; j < 2; j++) key_at[j] = key_row[j] * RB + ((c ^ cache_swizzle(RB, key_row[j])) << 4);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        token[r] = 4 * c + ((r + c) & 3);
        const int x = cache_swizzle(RB, token[r]);
        value_at[r] = kTile * RB + token[r] * RB + (kE * (HALF ? 2 : 1) == 16 ? (g ^ x) << 4 : (((g >> 1) ^ x) << 4) + 8 * (g & 1));
    }
    const float log2e = 1.4426950408889634f;

    bool dead = false;
    while (u < u1) {
        // ---- an item, or the part of it that is this CTA's
        const Span span = here.span;
        const int seq = here.s, head = here.item / row_tiles, row0 = (here.item % row_tiles) * G::kRows;
        const int first_unit = here.unit, units = here.units;
        const int until = (int)min((int64_t)units, first_unit + (u1 - u));
        if (!dead) issue();
        // this lane's rows: g and g + 8 (f32 queries: g, in two halves)
        const int row_a = row0 + g, row_b = row0 + 8 + g;
        const int ta = row_a / group, tb = row_b / group;
        const int head_a = head * group + row_a % group, head_b = head * group + row_b % group;
        const bool has_a = row_a < rows, has_b = !F32Q && row_b < rows;
        uint32_t q[G::kGroups][G::kSteps][4];
        float factor = p.scale;     // what a sum of products times the key's scale is multiplied with
        {
            constexpr int kN = HALF ? 8 : 16;   // channels of a lane's chunk
            float amount = 1.f;
            if constexpr (F32Q) {
                // brought near 2^14, so that the lower half keeps its bits in f16
                const float* from = (const float*)p.query + seq * p.q_strides[0] + ta * p.q_strides[1] + head_a * p.q_strides[2];
                float most = 0.f;
                if (has_a)
                    for (int d = c; d < p.cache.dim; d += 4) most = fmaxf(most, fabsf(from[d * p.q_strides[3]]));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const int e = (__float_as_int(most) >> 23) - 127;   // (of a NaN or an infinity 128: the row's result is one then)
                const int by = most > 0.f ? min(max(13 - e, -126), 126) : 0;
                amount = __int_as_float((127 + by) << 23);
                factor = p.scale * __int_as_float((127 - by) << 23);
            }
#pragma unroll
            for (int k = 0; k < G::kGroups; k++) {
                const int d0 = k * 4 * kN + c * kN;
#pragma unroll
                for (int half = 0; half < (F32Q ? 1 : 2); half++) {
                    const bool has = half ? has_b : has_a;
                    const int64_t from = seq * p.q_strides[0] + (half ? tb : ta) * p.q_strides[1] + (half ? head_b : head_a) * p.q_strides[2];
#pragma unroll
                    for (int st = 0; st < G::kSteps; st++)
#pragma unroll
                        for (int pair = 0; pair < 2; pair++) {
                            const int d = d0 + 4 * st + 2 * pair;
                            const bool one = has && d < p.cache.dim, two = has && d + 1 < p.cache.dim;
                            if constexpr (F32Q) {
                                const float* at = (const float*)p.query + from;
                                const float x = one ? at[d * p.q_strides[3]] * amount : 0.f, y = two ? at[(d + 1) * p.q_strides[3]] * amount : 0.f;
                                const uint32_t hi = pack(x, y);
                                const float2 back = __half22float2(*(const __half2*)&hi);
                                q[k][st][2 * pair] = hi;
                                q[k][st][2 * pair + 1] = pack(x - back.x, y - back.y);
                            } else {
                                const __half* at = (const __half*)p.query + from;
                                const __half x = one ? at[d * p.q_strides[3]] : __half(0.f), y = two ? at[(d + 1) * p.q_strides[3]] : __half(0.f);
                                const __half2 both = __halves2half2(x, y);
                                q[k][st][2 * pair + half] = *(const uint32_t*)&both;
                            }
                        }
                }
            }
        }
        const float slope_a = p.slopes && has_a ? p.slopes[head_a] * log2e : 0.f, slope_b = p.slopes && has_b ? p.slopes[head_b] * log2e : 0.f;
        const bool capped = p.softcap > 0.f;
        const float to_cap = capped ? (F32Q ? 1.f : 2.f * log2e) * factor / p.softcap : 0.f, cap = p.softcap * log2e, scaled = factor * log2e;
        const int64_t pos_a = span.shared + span.start + ta, pos_b = span.shared + span.start + tb;   // of the rows
        // positions that all rows of the item see: [all_lo, all_hi), and that one of them does
        const int t_first = max(row0 / group, span.t_lo), t_last = min((min(row0 + G::kRows, rows) - 1) / group, span.t_hi - 1);
        const int64_t all_hi = span.shared + span.start + t_first + 1, any_hi = min(span.shared + span.start + t_last + 1, (int64_t)span.shared + p.cache.capacity);
        const int64_t all_lo = p.window > 0 ? span.shared + span.start + t_last - p.window + 1 : 0, any_lo = p.window > 0 ? span.shared + span.start + t_first - p.window + 1 : 0;

        float o[G::kBlocks][kE][4];
#pragma unroll
        for (int b = 0; b < G::kBlocks; b++)
#pragma unroll
            for (int i = 0; i < kE; i++) o[b][i][0] = o[b][i][1] = o[b][i][2] = o[b][i][3] = 0.f;
        float most_a = -INFINITY, most_b = -INFINITY, sum_a = 0.f, sum_b = 0.f;
        float ref = 0.f, weight_scale = HALF ? 16384.f : 0.f;   // values' scales are counted in `ref`, a power of two; weights are up to 2^14

        for (int unit = first_unit; unit < until && !dead; unit++) {
            const int tile = unit * kWarps + warp;
            if (tile >= span.tiles || t_first > t_last) {
                if (tile < span.tiles) {   // (rows of nothing but padding, of a sequence that has others)
                    dead = !wait_tile();
                    consumed++;
                    if (!dead) issue();
                }
                continue;
            }
            const bool pre = tile < span.pre_tiles;
            const int64_t at = pre ? (int64_t)(span.pre_tile + tile) * kTile : span.shared + (int64_t)(span.own_tile + tile - span.pre_tiles) * kTile;   // position of the tile's first key
            const int64_t end = pre ? (int64_t)span.shared : (int64_t)span.shared + p.cache.capacity;
            const uint8_t* stage = ring + (consumed % kStages) * G::kStage;
            if (!wait_tile()) {
                dead = true;
                break;
            }
            // ---- scores: 16 rows x 16 keys
            float s[2][4] = {};
#pragma unroll
            for (int k = 0; k < G::kGroups; k++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int offset = RB % 128 == 0 ? (key_at[j] ^ ((k & 1) << 6)) + 128 * (k >> 1) : key_at[j] + 64 * k;
                    const uint4 raw = *(const uint4*)(stage + offset);
                    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
                    if constexpr (HALF) {
                        mma(s[j], q[k][0], w[0], w[1]);
                        mma(s[j], q[k][1], w[2], w[3]);
                    } else {
#pragma unroll
                        for (int st = 0; st < 4; st++) mma(s[j], q[k][st], two_of<0>(w[st]), two_of<2>(w[st]));
                    }
                }
            const float* scales = (const float*)(stage + 2 * kTile * RB);
            float value_scale[4];
            const bool masked = at < all_lo || at + kTile > min(all_hi, end);
            float xa[4], xb[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {   // r: column r % 2 of product r / 2
                xa[r] = s[r >> 1][r & 1];
                xb[r] = s[r >> 1][2 + (r & 1)];
                if constexpr (F32Q) xa[r] += xb[r];
                if constexpr (!HALF) {
                    const float ks = scales[token[r]];
                    value_scale[r] = scales[16 + token[r]];
                    xa[r] *= ks;
                    if constexpr (!F32Q) xb[r] *= ks;
                }
                if (!capped) {
                    xa[r] *= scaled;
                    if constexpr (!F32Q) xb[r] *= scaled;
                }
            }
            if (capped) {
                // tanh(y) = 1 - 2 / (1 + e^(2y)): off by 2^-22 of the cap, which f32 results do not take
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (F32Q) {
                        xa[r] = cap * tanhf(xa[r] * to_cap);
                    } else {
                        xa[r] = cap - __fdividef(2.f * cap, 1.f + exp2_fast(fminf(xa[r] * to_cap, 126.f)));
                        xb[r] = cap - __fdividef(2.f * cap, 1.f + exp2_fast(fminf(xb[r] * to_cap, 126.f)));
                    }
                }
            }
            if (p.slopes) {
                const float away_a = (float)(pos_a - at), away_b = (float)(pos_b - at);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    xa[r] -= slope_a * (away_a - (float)token[r]);
                    if constexpr (!F32Q) xb[r] -= slope_b * (away_b - (float)token[r]);
                }
            }
            uint32_t see = 0xfff;   // per position of this lane: a row sees it (bits 0 to 3: g, 4 to 7: g + 8, 8 to 11: any of the item)
            if (masked) {
                const auto within = [&](int64_t x) { return (int)min(max(x - at, (int64_t)-1), (int64_t)kTile); };   // in positions of the tile
                const int hi_a = min(within(pos_a + 1), within(end)), hi_b = min(within(pos_b + 1), within(end)), hi = min(within(any_hi), within(end));
                const int lo_a = p.window > 0 ? within(pos_a - p.window + 1) : 0, lo_b = p.window > 0 ? within(pos_b - p.window + 1) : 0, lo = within(any_lo);
                see = 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool a = token[r] >= lo_a && token[r] < hi_a, b = token[r] >= lo_b && token[r] < hi_b, any = token[r] >= lo && token[r] < hi;
                    see |= (a ? 1u << r : 0u) | (b ? 16u << r : 0u) | (any ? 256u << r : 0u);
                    if (!a) xa[r] = -INFINITY;
                    if (!b) xb[r] = -INFINITY;
                    if (!HALF && !any) value_scale[r] = 0.f;
                }
            }
            // ---- running maximum and sum
            const auto quad_most = [](float v) {
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
            };
            const float new_a = fmaxf(most_a, quad_most(fmaxf(fmaxf(xa[0], xa[1]), fmaxf(xa[2], xa[3]))));
            const float base_a = new_a == -INFINITY ? 0.f : new_a;
            const float keep_a = exp2_fast(most_a - base_a);
            float keep_b = 1.f, base_b = 0.f;
            most_a = new_a;
            if constexpr (!F32Q) {
                const float new_b = fmaxf(most_b, quad_most(fmaxf(fmaxf(xb[0], xb[1]), fmaxf(xb[2], xb[3]))));
                base_b = new_b == -INFINITY ? 0.f : new_b;
                keep_b = exp2_fast(most_b - base_b);
                most_b = new_b;
            }
            bool larger = false;
            if constexpr (!HALF) {
                const float top = fmaxf(fmaxf(value_scale[0], value_scale[1]), fmaxf(value_scale[2], value_scale[3]));
                larger = top > ref;
            }
            float shrink = 1.f;
            if constexpr (!HALF)
                if (__any_sync(0xffffffffu, larger)) {
                    const float top = quad_most(fmaxf(fmaxf(value_scale[0], value_scale[1]), fmaxf(value_scale[2], value_scale[3])));
                    // (the next power of two, but none so small that its inverse times 2^14 overflows)
                    const int e = min(max((__float_as_int(fmaxf(top, ref)) >> 23) + 1, 32), 254);
                    const float next = __int_as_float(e << 23);
                    shrink = ref > 0.f ? ref / next : 0.f;
                    ref = next;
                    weight_scale = 16384.f / next;
                }
            sum_a *= keep_a, sum_b *= keep_b;
            if (__any_sync(0xffffffffu, keep_a * shrink != 1.f || keep_b * shrink != 1.f)) {
                const float ka = keep_a * shrink, kb = (F32Q ? keep_a : keep_b) * shrink;
#pragma unroll
                for (int b = 0; b < G::kBlocks; b++)
#pragma unroll
                    for (int i = 0; i < kE; i++) o[b][i][0] *= ka, o[b][i][1] *= ka, o[b][i][2] *= kb, o[b][i][3] *= kb;
            }
            // ---- weights
            float wa[4], wb[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float vs = HALF ? weight_scale : value_scale[r] * weight_scale;
                const float ea = exp2_fast(xa[r] - base_a);
                sum_a += ea;
                wa[r] = see >> r & 1 ? ea * vs : 0.f;
                if constexpr (!F32Q) {
                    const float eb = exp2_fast(xb[r] - base_b);
                    sum_b += eb;
                    wb[r] = see >> r & 16 ? eb * vs : 0.f;
                }
            }
            uint32_t a[4];
            a[0] = pack(wa[0], wa[1]);
            a[2] = pack(wa[2], wa[3]);
            if constexpr (F32Q) {
                const float2 x = __half22float2(*(const __half2*)&a[0]), y = __half22float2(*(const __half2*)&a[2]);
                a[1] = pack(wa[0] - x.x, wa[1] - x.y);
                a[3] = pack(wa[2] - y.x, wa[3] - y.y);
            } else {
                a[1] = pack(wb[0], wb[1]);
                a[3] = pack(wb[2], wb[3]);
            }
            // ---- weights . values.  f32: the tile's products by themselves, then added (the matrix unit cuts off what it adds to a sum)
            const auto times = [&](float (&acc)[4], uint32_t b0, uint32_t b1) {
                if constexpr (F32Q) {
                    float part[4] = {};
                    mma(part, a, b0, b1);
#pragma unroll
                    for (int n = 0; n < 4; n++) acc[n] += part[n];
                } else {
                    mma(acc, a, b0, b1);
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
                    if (masked) {
                        // what nobody sees, and infinities and NaN that some rows do not see (they are added row by row below), count as 0
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const bool seen = see >> r & 256;
#pragma unroll
                            for (int n = 0; n < kWords; n++) {
                                const bool lo = (w[r][n] & 0x7c00u) == 0x7c00u, hi = (w[r][n] & 0x7c000000u) == 0x7c000000u;
                                odd = odd || (seen && (lo || hi));
                                w[r][n] = seen ? w[r][n] & (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0xffffu : 0xffffffffu) : 0u;
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < kWords; n++) {
                        times(o[b][2 * n], __byte_perm(w[0][n], w[1][n], 0x5410), __byte_perm(w[2][n], w[3][n], 0x5410));
                        times(o[b][2 * n + 1], __byte_perm(w[0][n], w[1][n], 0x7632), __byte_perm(w[2][n], w[3][n], 0x7632));
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < kWords; n++) {
                        const uint32_t lo01 = __byte_perm(w[0][n], w[1][n], 0x5140), lo23 = __byte_perm(w[2][n], w[3][n], 0x5140);
                        const uint32_t hi01 = __byte_perm(w[0][n], w[1][n], 0x7362), hi23 = __byte_perm(w[2][n], w[3][n], 0x7362);
                        times(o[b][4 * n], two_of<0>(lo01), two_of<0>(lo23));
                        times(o[b][4 * n + 1], two_of<2>(lo01), two_of<2>(lo23));
                        times(o[b][4 * n + 2], two_of<0>(hi01), two_of<0>(hi23));
                        times(o[b][4 * n + 3], two_of<2>(hi01), two_of<2>(hi23));
                    }
                }
            }
            if constexpr (HALF)
                if (__any_sync(0xffffffffu, odd)) {
                    for (int k = 0; k < kTile; k++) {
                        // the weight of key k, of which lane 4 g + k / 4 has it as its number (k - k / 4) % 4
                        const int r = (k - (k >> 2)) & 3, from = (lane & ~3) | (k >> 2);
                        float na = -1.f, nb = -1.f;   // hidden
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (i == r && (see >> i & 1)) na = wa[i];
                            if constexpr (!F32Q)
                                if (i == r && (see >> i & 16)) nb = wb[i];
                        }
                        const float ka = __shfl_sync(0xffffffffu, na, from), kb = __shfl_sync(0xffffffffu, nb, from);
                        if (!(__shfl_sync(0xffffffffu, see >> r, from) & 256)) continue;
#pragma unroll
                        for (int b = 0; b < G::kBlocks; b++)
#pragma unroll
                            for (int i = 0; i < kE; i++)
#pragma unroll
                                for (int n = 0; n < 2; n++) {
                                    const int d = kE * (2 * c + n) + i;
                                    const int chunk = (d >> 3) ^ cache_swizzle(RB, k);
                                    const float v = __half2float(*(const __half*)(stage + kTile * RB + k * RB + b * 128 + (chunk << 4) + 2 * (d & 7)));
                                    if (fabsf(v) <= 65504.f) continue;
                                    if (ka >= 0.f) o[b][i][n] += ka * v;
                                    if (kb >= 0.f) o[b][i][2 + n] += kb * v;
                                }
                    }
                }
            consumed++;
            __syncwarp();
            issue();
        }

        // ---- the warps' parts become one
        sum_a += __shfl_xor_sync(0xffffffffu, sum_a, 1);
        sum_a += __shfl_xor_sync(0xffffffffu, sum_a, 2);
        sum_b += __shfl_xor_sync(0xffffffffu, sum_b, 1);
        sum_b += __shfl_xor_sync(0xffffffffu, sum_b, 2);
        if (c == 0) {
            row_most[warp][g] = most_a, row_sum[warp][g] = sum_a;
            if constexpr (!F32Q) row_most[warp][g + 8] = most_b, row_sum[warp][g + 8] = sum_b;
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
            float sum = 0.f;
            for (int w = 0; w < kWarps; w++) sum += row_sum[w][r] * (m == -INFINITY ? 0.f : exp2_fast(row_most[w][r] - m));
            row_all[r] = sum;   // (read behind the next barrier)
        }
        const float unscale = (HALF ? 1.f : ref) * (1.f / 16384.f);
        const float all_a = most_of(g), all_b = F32Q ? all_a : most_of((g + 8) & 15);
        const float times_a = all_a == -INFINITY ? 0.f : exp2_fast(most_a - all_a) * unscale;
        const float times_b = F32Q ? times_a : all_b == -INFINITY ? 0.f : exp2_fast(most_b - all_b) * unscale;
        const bool whole = first_unit == 0 && until == units;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (u == u0 ? 0 : 1);
        float* const partial = p.partial + slot * (G::kRows * (kDim + 2));
        const auto visible = [&](int row) {   // does this row see anything
            const int t = row / group;
            if (row >= rows || t < span.t_lo || t >= span.t_hi) return false;
            const int64_t pos = span.shared + span.start + t, last = min(pos, (int64_t)span.shared + p.cache.capacity - 1);
            return last >= 0 && (p.window == 0 || last > pos - p.window);
        };
        const auto store = [&](int row, int d, float v) {
            if (row >= rows || d >= p.cache.dim) return;
            const int64_t to = (((int64_t)seq * p.tokens + row / group) * p.heads + head * group + row % group) * p.cache.dim + d;
            if constexpr (F32Q) ((float*)p.out)[to] = v;
            else ((__half*)p.out)[to] = __float2half_rn(v);
        };
        constexpr int kI = 4;   // kI of a lane's channels of a block at a time: 8 kI channels of the block
#pragma unroll
        for (int b = 0; b < G::kBlocks; b++)
#pragma unroll
            for (int i0 = 0; i0 < kE; i0 += kI) {
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    float* to = join + (warp * G::kRows + g) * 32 + (2 * c + n) * kI;
                    float va[kI], vb[kI];
#pragma unroll
                    for (int i = 0; i < kI; i++) {
                        va[i] = o[b][i0 + i][n] * times_a;
                        vb[i] = o[b][i0 + i][2 + n] * times_b;
                        if constexpr (F32Q) va[i] += vb[i];
                    }
                    *(float4*)to = make_float4(va[0], va[1], va[2], va[3]);
                    if constexpr (!F32Q) *(float4*)(to + 8 * 32) = make_float4(vb[0], vb[1], vb[2], vb[3]);
                }
                __syncthreads();
                for (int at = threadIdx.x; at < G::kRows * 32; at += kThreads) {
                    const int r = at >> 5, n = (at & 31) / kI, i = (at & 31) % kI, d = b * 8 * kE + kE * n + i0 + i;
                    if (row0 + r >= rows) continue;
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; w++) v += join[(w * G::kRows + r) * 32 + (at & 31)];
                    if (whole) {
                        store(row0 + r, d, visible(row0 + r) ? v / row_all[r] : 0.f);
                    } else {
                        partial[r * kDim + d] = v;
                    }
                }
                __syncthreads();
            }
        if (!whole) {
            if (threadIdx.x < G::kRows) {
                const int r = threadIdx.x;
                partial[G::kRows * kDim + 2 * r] = most_of(r);
                partial[G::kRows * kDim + 2 * r + 1] = row_all[r];
            }
            // ---- whoever is last joins the item's parts
            const int64_t item_u = u - first_unit;   // the item's first unit; CTA b has units from total b / ctas on
            const int64_t c0 = ((item_u + 1) * ctas - 1) / total, c1 = ((item_u + units) * ctas - 1) / total;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                uint32_t* arrived = p.arrived + (int64_t)seq * items + here.item;
                const uint32_t before = atomicAdd(arrived, 1u);
                is_last = before == (uint32_t)(c1 - c0);
                if (is_last) *arrived = 0;
                __threadfence();
            }
            __syncthreads();
            if (is_last) {
                const auto part_of = [&](int64_t b) { return p.partial + (2 * b + (b == c0 && total * b / ctas < item_u ? 1 : 0)) * (G::kRows * (kDim + 2)); };
                for (int at = threadIdx.x; at < G::kRows * kDim / 4; at += kThreads) {
                    const int r = at / (kDim / 4), d = at % (kDim / 4) * 4;
                    if (row0 + r >= rows) continue;
                    float m = -INFINITY, sum = 0.f;
                    for (int64_t b = c0; b <= c1; b++) m = fmaxf(m, __ldcg(part_of(b) + G::kRows * kDim + 2 * r));
                    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
                    for (int64_t b = c0; b <= c1; b++) {
                        const float* part = part_of(b);
                        const float2 state = __ldcg((const float2*)(part + G::kRows * kDim + 2 * r));
                        const float4 x = __ldcg((const float4*)(part + r * kDim + d));
                        const float f = m == -INFINITY ? 0.f : exp2_fast(state.x - m);
                        sum += f * state.y;
                        v.x += f * x.x, v.y += f * x.y, v.z += f * x.z, v.w += f * x.w;
                    }
                    const bool some = visible(row0 + r);
                    store(row0 + r, d, some ? v.x / sum : 0.f);
                    store(row0 + r, d + 1, some ? v.y / sum : 0.f);
                    store(row0 + r, d + 2, some ? v.z / sum : 0.f);
                    store(row0 + r, d + 3, some ? v.w / sum : 0.f);
                }
            }
            __syncthreads();
        }
        u += until - first_unit;
        here.unit = until - 1;
        here.next(p, kWarps, items);
    }
    // (given up: what is under way still writes to this CTA's shared memory)
    for (; dead && consumed < issued; consumed++) wait_tile();
}

// f(Geo, kernel) of the variant that takes p
template <bool HALF, bool F32Q, typename F>
void with_dim(int blocks, F f) {
    if (blocks == 1) f(Geo<HALF, F32Q, 1>{}, cache_attention_kernel<HALF, F32Q, 1>);
    if (blocks == 2) f(Geo<HALF, F32Q, 2>{}, cache_attention_kernel<HALF, F32Q, 2>);
    if (blocks == 3) f(Geo<HALF, F32Q, 3>{}, cache_attention_kernel<HALF, F32Q, 3>);
    if (blocks == 4) f(Geo<HALF, F32Q, 4>{}, cache_attention_kernel<HALF, F32Q, 4>);
}
template <typename F>
void with_variant(const CacheAttentionParams& p, F f) {
    const int blocks = (p.cache.dim + 63) / 64;
    if (p.cache.half) p.half ? with_dim<true, false>(blocks, f) : with_dim<true, true>(blocks, f);
    else p.half ? with_dim<false, false>(blocks, f) : with_dim<false, true>(blocks, f);
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
        plan.grid = (int32_t)std::min<double>(148 * G::kPerSm, most);
        plan.partial_floats = 2ll * plan.grid * G::kRows * (G::kDim + 2);
    });
    return plan;
}

int launch_cache_attention(const CacheAttentionParams& p, cudaStream_t stream) {
    int err = 0;
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
