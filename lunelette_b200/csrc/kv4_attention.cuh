// Causal attention over the paged 4-bit KV cache for few query rows: decode
// steps over many sequences, and short runs of tokens.
//
// HBM-bound by design: a block of the cache (one page of one KV head, 9216 bytes for
// 128 dims) is copied once into shared memory, K with its scales and V with its
// scales by bulk copies of their own, and serves all the query rows of its KV head.
//
// Work is dealt out page by page: the pages of all (sequence, KV head, row tile) items
// make one list, of which every warp of the grid takes an equal, contiguous share, found
// from the lengths on the device. So a call's time does not depend on how its lengths
// are spread. A warp walks its share with its own ring of half blocks, whatever items
// it crosses; a whole item is written out, the ends of others leave parts that the
// combine kernel adds up in order. Where a block's warps share one item (long
// sequences), they merge first, through shared memory. Where there are fewer pages
// than a quarter of the warps, a share is counted in 16 keys instead.
//
// The products run on mma.sync m16n8k16 with FP16 operands and FP32 sums: a
// decode step has 1 to 16 query rows a KV head, so a tcgen05 tile of 128 rows would be
// mostly padding, while here the rows sit in the n = 8 side. FP32 rows of q and
// weights of the softmax enter as FP16 hi + lo parts in neighbouring columns
// (22 bits together), so one MMA serves 4 rows at FP32 grade; of 16-bit rows the 11
// bits of one FP16 are taken (q exact after a power-of-two scaling but for what lies
// 2^-17 below the row's largest; a weight off by 2^-12 of itself, under the rounding of the
// output), 8 rows an MMA.
//   S = K Q^T     A: 16 keys x 16 dims of integers c - 8 straight from the
//                 codes (exact); a group's sum is scaled by d in FP32 after its
//                 two MMAs, so K needs no multiplication per element.
//   O^T = V^T P^T A: 16 dims x 16 keys of d * (c - 8), exact in FP16; B: the
//                 weights, moved from S's layout by movmatrix.
// A code becomes FP16 by OR-ing it into the mantissa of 1024 (low nibble of a
// byte) or of 1024 scaled by 16 (high nibble) and subtracting: both exact.
#pragma once
#include "async.cuh"
#include "attention.cuh"
#include "kv4.cuh"

namespace lun {

constexpr int kKv4Timeout = 4;  // status bit: a bounded wait gave up, outputs are not valid

struct Kv4AttnParams {
    Kv4Cache cache;
    Kv4Rows rows;
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    int group;     // query heads per KV head
    float scale2;  // scale * log2 e
    int tiles;     // decode kernel: row tiles of a (sequence, KV head), at most
    int most;      // decode kernel: its sequences have at most so many rows a KV head
    int split_pages, splits;  // block kernel: pages of a split; splits, 1: the kernel writes the output itself
    bool wide;
    // unnormalised o, m, l, D + 2 floats a row: [2 warp + (0 the warp's first item, 1 its last)][row of
    // the tile] of the decode kernel, [row][query head][split] of the block kernel
    float *part;
    int2 *items;  // decode kernel: an item's first part (-1: it is written out) and last warp
    int *status;
};

// A bounded wait of one thread on an mbarrier phase. The clock and the abort word
// are read only after 64 polls: reading %globaltimer on the first poll that fails
// costs more than most waits here last. False when the CTA gave up.
__device__ __forceinline__ bool kv4_wait(uint64_t *bar, unsigned parity, volatile int *abort_word)
{
    unsigned long long start = 0;
    for (unsigned spins = 1; !mbar_try_wait(bar, parity); spins++) {
        if (spins < 64 || (spins & 15u)) continue;
        const unsigned long long now = wait_clock_ns();
        if (spins == 64) start = now;
        if (*abort_word) return false;
        if (now - start > kWaitLimitNs) {
            *abort_word = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool kv4_warp_wait(uint64_t *bar, unsigned parity, volatile int *abort_word)
{
    return __all_sync(0xffffffffu, kv4_wait(bar, parity, abort_word));
}

// The softmax's weights are taken times 2^14, and l with them: the largest is
// 16384, and the FP16 parts of a weight keep 22 bits down to 2^-28 of it, where a
// largest weight of 1 would leave small ones on the 2^-24 grid of FP16's
// subnormals.
constexpr float kWeightShift = 14.0f;

#ifndef KV4_SLOTS
#define KV4_SLOTS 4
#define KV4_CTAS 3
#endif
constexpr int kDecodeWarps = 4, kDecodeSlots = KV4_SLOTS, kDecodeCtas = KV4_CTAS;

template <int D, typename T, int NT> struct Kv4Decode {
    static constexpr bool split = sizeof(T) == 4;    // hi and lo columns
    static constexpr int lane_rows = split ? 1 : 2;  // query rows of a lane and n tile
    static constexpr int rows = 4 * NT * lane_rows;  // query rows of a tile
    static constexpr int half = Kv4Layout<D>::block / 2;
    static constexpr int ring = kDecodeWarps * kDecodeSlots * half;
    static constexpr int merge = kDecodeWarps * rows * (D + 2) * 4;
    static constexpr int bars = (ring > merge ? ring : merge);
    static constexpr int prefix = bars + kDecodeWarps * kDecodeSlots * 8;  // 33 * kDecodeWarps long longs
    static constexpr int smem = prefix + (32 * kDecodeWarps + 1) * 8 + 16;
};

__device__ __forceinline__ float exp2_fast(float x)  // 2 ulp; 0 below 2^-126
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Four codes in the bytes' low and high nibbles of both halves -> c - 8 in FP16:
// a = (nibble 0, nibble 4), b = (nibble 1, nibble 5) of a word.
__device__ __forceinline__ uint32_t kv4_low(uint32_t w)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(r) : "r"(w));
    const __half2 h = __hsub2(*reinterpret_cast<__half2 *>(&r), __half2half2(__ushort_as_half(0x6408)));  // 1032
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t kv4_high(uint32_t w)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(r) : "r"(w));
    // (1024 + 16 c) / 16 - 72
    const __half2 h = __hfma2(*reinterpret_cast<__half2 *>(&r), __half2half2(__ushort_as_half(0x2c00)),
                              __half2half2(__ushort_as_half(0xd480)));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t kv4_times(uint32_t v, uint32_t d)
{
    const __half2 h = __hmul2(*reinterpret_cast<__half2 *>(&v), *reinterpret_cast<__half2 *>(&d));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float low_half(uint32_t v) { return __low2float(*reinterpret_cast<__half2 *>(&v)); }
__device__ __forceinline__ float high_half(uint32_t v) { return __high2float(*reinterpret_cast<__half2 *>(&v)); }

// 2^-e with 2^e the power of two at or below x's magnitude, e within +-120;
// 1 for zero, NaN and infinities.
__device__ __forceinline__ float power_scale(float x, float &back)
{
    int e = (int)(__float_as_uint(x) >> 23 & 255) - 127;
    if (x == 0.0f || e == 128) e = 0;
    e = max(-120, min(120, e));
    back = __uint_as_float((uint32_t)(127 + e) << 23);
    return __uint_as_float((uint32_t)(127 - e) << 23);
}


// What the decode kernel does of a sequence: units of KT * 16 keys an item, items.
struct Kv4Share {
    int units, tiles;
    long long all;  // units of all its items
};
template <int KT, int ROWS>
__device__ __forceinline__ Kv4Share kv4_share(const Kv4AttnParams &p, const Kv4Sequence &q)
{
    Kv4Share w = {0, 0, 0};
    const int rows = q.count * p.group;
    if (!q.ok || rows == 0 || rows > p.most) return w;
    w.units = (q.length + 16 * KT - 1) / (16 * KT);
    w.tiles = (rows + ROWS - 1) / ROWS;
    w.all = (long long)w.units * p.cache.heads * w.tiles;
    return w;
}

// Grid: any number of blocks; items [sequence][KV head][row tile of p.tiles].
template <int D, typename T, int NT, int KT>
static __global__ void __launch_bounds__(32 * kDecodeWarps, NT == 1 ? kDecodeCtas : 2) kv4_decode_kernel(Kv4AttnParams p)
{
    using L = Kv4Layout<D>;
    using K = Kv4Decode<D, T, NT>;
    constexpr int G = L::groups, MT = D / 16, RP = K::lane_rows, W = kDecodeWarps, SLOTS = kDecodeSlots;
    constexpr int row_bytes = D / 2;
    extern __shared__ __align__(128) uint8_t kv4_smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(kv4_smem + K::bars);
    long long *prefix = reinterpret_cast<long long *>(kv4_smem + K::prefix);  // of 128 runs of sequences
    volatile int *abort_word = reinterpret_cast<volatile int *>(prefix + 32 * W + 1);
    volatile int *merged_word = abort_word + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint64_t *bar = bars + warp * SLOTS;
    if (threadIdx.x == 0) *abort_word = 0;
    if (lane < SLOTS) mbar_init(&bar[lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_wait();
    pdl_launch_dependents();

    // ---- this warp's units [u0, u1) of the list
    const int run = (p.rows.sequences + 32 * W - 1) / (32 * W);  // sequences of a thread
    {
        long long sum = 0;
        for (int i = 0; i < run; i++) {
            const int s = threadIdx.x * run + i;
            if (s >= p.rows.sequences) break;
            const Kv4Sequence q = kv4_sequence(p.rows, s);
            if (!q.ok && blockIdx.x == 0) kv4_report(p.status, kKv4BadRows);
            sum += kv4_share<KT, K::rows>(p, q).all;
        }
        long long upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        if (lane == 31) prefix[32 * W - warp] = upto;  // the warps' totals, for a moment
        __syncthreads();
        long long before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const long long all = prefix[32 * W - w];
            if (w < warp) before += all;
            total += all;
        }
        __syncthreads();
        prefix[threadIdx.x] = before + upto - sum;
        if (threadIdx.x == 0) prefix[32 * W] = total;
        __syncthreads();
    }
    const long long total = prefix[32 * W];
    const long long warps = min((long long)gridDim.x * W, total);
    const long long me = (long long)blockIdx.x * W + warp;
    if ((long long)blockIdx.x * W >= warps) return;
    auto share_of = [&](long long i) { return i >= warps ? total : total / warps * i + total % warps * i / warps; };
    const long long u0 = share_of(me), u1 = share_of(me + 1);
    const int n = (int)(u1 - u0);
    // the sequence of u0 and its first unit
    int s = 0;
    long long base = 0;
    if (n > 0) {
        int k = -1;
        for (int i = 0; i < W; i++) {
            const unsigned at = __ballot_sync(0xffffffffu, prefix[32 * i + lane] <= u0);
            if (at) k = 32 * i + 31 - __clz(at);
        }
        s = k * run;
        base = prefix[k];
        for (;;) {
            const long long all = kv4_share<KT, K::rows>(p, kv4_sequence(p.rows, s)).all;
            if (u0 < base + all) break;
            base += all;
            s++;
        }
    }
    // unit base_i + lane of the list: its block in the layer (or none) and its item
    auto map = [&](int i, uint32_t &block, int &item, int &unit) {
        block = 0xffffffffu;
        item = -1;
        unit = 0;
        const long long u = u0 + i;
        if (u >= u1) return;
        Kv4Share w;
        for (;;) {
            w = kv4_share<KT, K::rows>(p, kv4_sequence(p.rows, s));
            if (u < base + w.all) break;
            base += w.all;
            s++;
        }
        const long long rest = u - base;
        const int of = (int)(rest / w.units), kvh = of / w.tiles;
        unit = (int)(rest - (long long)of * w.units);
        item = (s * p.cache.heads + kvh) * p.tiles + of - kvh * w.tiles;
        const int id = p.rows.page_tables[s * p.rows.table_stride + (KT == 4 ? unit : unit >> 2)];
        if ((unsigned)id < (unsigned)p.cache.pages) block = (uint32_t)id * (uint32_t)p.cache.heads + kvh;
        else kv4_report(p.status, kKv4BadPage);
    };
    // two sets of 32 units, a lane each; the walk is in one while the other is fetched
    uint32_t block_a, block_b = 0xffffffffu;
    int item_a, item_b = -1, unit_a, unit_b;
    map(lane, block_a, item_a, unit_a);
    auto block_at = [&](int i) { return __shfl_sync(0xffffffffu, i & 32 ? block_b : block_a, i & 31); };
    auto item_at = [&](int i) { return __shfl_sync(0xffffffffu, i & 32 ? item_b : item_a, i & 31); };
    int unit = __shfl_sync(0xffffffffu, unit_a, 0);  // of the current item

    uint8_t *buffers = kv4_smem + warp * SLOTS * K::half;
    // half h of the walk: K (even) or V (odd) of unit h / 2
    int issue_unit = unit, issue_item = item_at(0);  // the unit within its item of the next half
    auto issue = [&](int h, int slot) {
        const uint32_t id = block_at(h >> 1);
        int quarter = 0;
        if (KT == 1) {  // which 16 keys of the page
            const int item = item_at(h >> 1);
            if (item != issue_item) issue_item = item, issue_unit = 0;
            quarter = issue_unit & 3;
            if (h & 1) issue_unit++;
        }
        if (lane || id == 0xffffffffu) return;
        const uint8_t *src = p.cache.layer + (size_t)id * L::block + (h & 1 ? K::half : 0);
        uint8_t *dst = buffers + slot * K::half;
        if (KT == 4) {
            mbar_expect_tx(&bar[slot], K::half);
            bulk_g2s(dst, src, K::half, &bar[slot]);
        } else {
            constexpr int codes = 16 * row_bytes, scales = 32 * G;
            mbar_expect_tx(&bar[slot], codes + scales);
            bulk_g2s(dst + quarter * codes, src + quarter * codes, codes, &bar[slot]);
            bulk_g2s(dst + L::codes + quarter * scales, src + L::codes + quarter * scales, scales, &bar[slot]);
        }
    };
#pragma unroll
    for (int h = 0; h < SLOTS; h++)
        if (h < 2 * n) issue(h, h);
    // whether the block's warps share one item
    if (warp == 0) {
        const Kv4Share all = kv4_share<KT, K::rows>(p, kv4_sequence(p.rows, item_at(0) / p.tiles / p.cache.heads));
        if (lane == 0)
            *merged_word = (long long)blockIdx.x * W + W <= warps && u0 + all.units - unit >= share_of(me + W);
    }
    __syncthreads();
    const bool merged = *merged_word != 0;

    // byte offsets of the lane's first reads in a half block; 16 keys on are 16 rows on, the swizzle the same
    const int k_at = g * row_bytes + 4 * G * t, ks_at = L::k_scale(g, 0);
    const int v_even = L::v_word(2 * t, g * (MT / 4)) - K::half, v_odd = v_even ^ row_bytes;
    const int vs_at = L::v_scale(2 * t, g * (D / 8) / 32) - K::half;
    bool ok = true, ends = false;
    unsigned phases = 0;  // parity of each slot's next wait
    int slot = 0;
    auto next = [&](int h) {  // done with half h: every lane has read it; refill its slot
        __syncwarp();
        if (h + SLOTS < 2 * n) issue(h + SLOTS, slot);
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
    };
    float m[NT][RP], l[NT][RP], o[NT][MT][4];
    int item = 0, begin = 0, r0 = 0, kvh = 0;
    Kv4Sequence q = {0, 0, 0, false};
    for (int i = 0; i < n && ok;) {
        // ---- an item
        const bool first_item = i == 0;
        item = item_at(i);
        begin = unit;
        r0 = item % p.tiles * K::rows;
        kvh = item / p.tiles % p.cache.heads;
        q = kv4_sequence(p.rows, item / p.tiles / p.cache.heads);
        const int n_rows = q.count * p.group, units = (q.length + 16 * KT - 1) / (16 * KT);
        // q as B: column g of n tile nt belongs to row (split: 4 nt + g / 2, part g % 2; else 8 nt + g)
        uint32_t qb[NT][D / 16][2];
        float back[NT][RP];  // what a score is multiplied with, of the lane's rows 4 nt + t or 8 nt + 2 t + (0, 1)
        int limit[NT][RP];   // those rows' last visible position
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = r0 + (K::split ? 4 * nt + (g >> 1) : 8 * nt + g);
            const bool live = r < n_rows;
            const int token = live ? r / p.group : 0, head = kvh * p.group + (live ? r - token * p.group : 0);
            const T *src = static_cast<const T *>(p.q) + (size_t)(q.first + token) * p.q_stride + (size_t)head * D + 8 * t;
            float x[G][8], top = 0.0f;
#pragma unroll
            for (int j = 0; j < G; j++) {
                load8(src + 32 * j, p.wide, x[j]);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (!live) x[j][e] = 0.0f;
                    top = fmaxf(top, fabsf(x[j][e]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float undo;
            const float f = power_scale(top, undo);
#pragma unroll
            for (int j = 0; j < G; j++)
#pragma unroll
                for (int hw = 0; hw < 2; hw++)
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        uint32_t hi, lo;
                        split_half2(x[j][2 * hw + b] * f, x[j][2 * hw + b + 4] * f, hi, lo);
                        qb[nt][2 * j + hw][b] = K::split && (g & 1) ? lo : hi;
                    }
#pragma unroll
            for (int e = 0; e < RP; e++) {
                // the row's factors sit in the lanes of its (first) column
                back[nt][e] = __shfl_sync(0xffffffffu, undo, 4 * (2 * t + e)) * p.scale2;
                const int row = r0 + (K::split ? 4 * nt + t : 8 * nt + 2 * t + e);
                limit[nt][e] = row < n_rows ? q.length - q.count + row / p.group : -1;
                m[nt][e] = -INFINITY;
                l[nt][e] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < MT; j++) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.0f;
        }
        const int all_see = q.length - q.count + r0 / p.group;  // every row of the tile sees keys up to here
        do {
            if ((i & 31) == 0 && i + 32 < n) {  // the other set of units, long before it is asked for
                s = __shfl_sync(0xffffffffu, s, 31);
                base = __shfl_sync(0xffffffffu, base, 31);
                if (i & 32) map(i + 32 + lane, block_a, item_a, unit_a);
                else map(i + 32 + lane, block_b, item_b, unit_b);
            }
            if (block_at(i) == 0xffffffffu) {
                next(2 * i);
                next(2 * i + 1);
                continue;
            }
            if (!(ok = kv4_warp_wait(&bar[slot], phases >> slot & 1, abort_word))) break;
            phases ^= 1u << slot;
            const int p0 = unit * 16 * KT, tile0 = KT == 4 ? 0 : unit & 3;
            const uint8_t *block = buffers + slot * K::half + tile0 * 16 * row_bytes;
            const uint8_t *block_scales = buffers + slot * K::half + tile0 * 32 * G;
            float sc[KT][NT][2][RP];
#pragma unroll
            for (int tile = 0; tile < KT; tile++) {
                float acc[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
                uint32_t ka[G], kb[G], da[G / 2], db[G / 2];
                const uint8_t *row = block + k_at + 16 * tile * row_bytes, *scale = block_scales + ks_at + 32 * G * tile;
                if constexpr (G == 4) {
                    *reinterpret_cast<uint4 *>(ka) = *reinterpret_cast<const uint4 *>(row);
                    *reinterpret_cast<uint4 *>(kb) = *reinterpret_cast<const uint4 *>(row + 8 * row_bytes);
                    *reinterpret_cast<uint2 *>(da) = *reinterpret_cast<const uint2 *>(scale);
                    *reinterpret_cast<uint2 *>(db) = *reinterpret_cast<const uint2 *>(scale + 16 * G);
                } else {
                    *reinterpret_cast<uint2 *>(ka) = *reinterpret_cast<const uint2 *>(row);
                    *reinterpret_cast<uint2 *>(kb) = *reinterpret_cast<const uint2 *>(row + 8 * row_bytes);
                    da[0] = *reinterpret_cast<const uint32_t *>(scale);
                    db[0] = *reinterpret_cast<const uint32_t *>(scale + 16 * G);
                }
#pragma unroll
                for (int j = 0; j < G; j++) {
                    const uint32_t a0[4] = {kv4_low(ka[j]), kv4_low(kb[j]), kv4_high(ka[j]), kv4_high(kb[j])};
                    const uint32_t a1[4] = {kv4_low(ka[j] >> 8), kv4_low(kb[j] >> 8), kv4_high(ka[j] >> 8),
                                            kv4_high(kb[j] >> 8)};
                    const float d0 = j & 1 ? high_half(da[j >> 1]) : low_half(da[j >> 1]);
                    const float d1 = j & 1 ? high_half(db[j >> 1]) : low_half(db[j >> 1]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_16816(c, a0, qb[nt][2 * j][0], qb[nt][2 * j][1]);
                        mma_16816(c, a1, qb[nt][2 * j + 1][0], qb[nt][2 * j + 1][1]);
                        acc[nt][0] = fmaf(d0, c[0], acc[nt][0]);
                        acc[nt][1] = fmaf(d0, c[1], acc[nt][1]);
                        acc[nt][2] = fmaf(d1, c[2], acc[nt][2]);
                        acc[nt][3] = fmaf(d1, c[3], acc[nt][3]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int k8 = 0; k8 < 2; k8++) {
                        if constexpr (K::split) {
                            sc[tile][nt][k8][0] = (acc[nt][2 * k8] + acc[nt][2 * k8 + 1]) * back[nt][0];
                        } else {
                            sc[tile][nt][k8][0] = acc[nt][2 * k8] * back[nt][0];
                            sc[tile][nt][k8][1] = acc[nt][2 * k8 + 1] * back[nt][1];
                        }
                    }
            }
            next(2 * i);
            if (p0 + 16 * KT - 1 > all_see) {
#pragma unroll
                for (int tile = 0; tile < KT; tile++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int k8 = 0; k8 < 2; k8++)
#pragma unroll
                            for (int e = 0; e < RP; e++)
                                if (p0 + 16 * tile + 8 * k8 + g > limit[nt][e]) sc[tile][nt][k8][e] = -INFINITY;
            }
            uint32_t pb[KT][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                // the maximum moves seldom once a few pages are in: the warp agrees on whether one does
                float corr[RP], zero[RP];
                bool raised = false;
                float high[RP];
#pragma unroll
                for (int e = 0; e < RP; e++) {
                    float mx = sc[0][nt][0][e];
#pragma unroll
                    for (int tile = 0; tile < KT; tile++) mx = fmaxf(mx, fmaxf(sc[tile][nt][0][e], sc[tile][nt][1][e]));
                    high[e] = mx;
                    raised = raised || mx > m[nt][e];
                    corr[e] = 1.0f;
                }
                if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
                    for (int e = 0; e < RP; e++) {
                        float mx = fmaxf(high[e], m[nt][e]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        corr[e] = mx == m[nt][e] ? 1.0f : exp2_fast(m[nt][e] - mx);
                        m[nt][e] = mx;
                        l[nt][e] *= corr[e];
                    }
#pragma unroll
                    for (int j = 0; j < MT; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[nt][j][e] *= corr[K::split ? 0 : e & 1];
                }
                // a row without any key yet: exp2(-inf - 0) = 0
#pragma unroll
                for (int e = 0; e < RP; e++) zero[e] = m[nt][e] == -INFINITY ? 0.0f : m[nt][e] - kWeightShift;
#pragma unroll
                for (int tile = 0; tile < KT; tile++)
#pragma unroll
                    for (int k8 = 0; k8 < 2; k8++) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < RP; e++) {
                            w[e] = exp2_fast(sc[tile][nt][k8][e] - zero[e]);
                            l[nt][e] += w[e];
                        }
                        __half2 two;
                        if constexpr (K::split) {
                            const __half h = __float2half_rn(w[0]);
                            two = __halves2half2(h, __float2half_rn(w[0] - __half2float(h)));
                        } else {
                            two = __floats2half2_rn(w[0], w[1]);
                        }
                        pb[tile][nt][k8] = movmatrix_trans(*reinterpret_cast<const uint32_t *>(&two));
                    }
            }
            if (!(ok = kv4_warp_wait(&bar[slot], phases >> slot & 1, abort_word))) break;
            phases ^= 1u << slot;
            uint8_t *vblock = buffers + slot * K::half;
            uint8_t *vscales = vblock + L::codes + tile0 * 32 * G;  // [position / 2][group][position % 2]
            {
                // scales behind the last position (whatever those slots hold) and NaNs become zeros
                // before the MMAs, in which a weight of zero would not keep a NaN away from a row
                // that does not see its position; the rows that do see a NaN take it here
                constexpr int words = KT * 8 * G, each = (words + 31) / 32;
                uint32_t *mine = reinterpret_cast<uint32_t *>(vscales) + lane;
                uint32_t d[each], nan = 0;
                const int valid = q.length - p0;
#pragma unroll
                for (int e = 0; e < each; e++) {
                    d[e] = words % 32 == 0 || lane + 32 * e < words ? mine[32 * e] : 0;
                    nan |= __hneu2_mask(*reinterpret_cast<__half2 *>(&d[e]), *reinterpret_cast<__half2 *>(&d[e]));
                }
                if (valid < 16 * KT || __any_sync(0xffffffffu, nan != 0)) {
                    for (int key = 0; key < min(valid, 16 * KT); key++) {
                        const int at = ((key >> 1) * G + g * (D / 8) / 32) * 2 + (key & 1);
                        const float x = __half2float(reinterpret_cast<const __half *>(vscales)[at]);
                        if (x != x)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int e = 0; e < RP; e++)
                                    if (p0 + key <= limit[nt][e])
#pragma unroll
                                        for (int j = 0; j < MT; j++) o[nt][j][e] = o[nt][j][2 + e] = x;
                    }
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < each; e++) {
                        d[e] &= ~__hneu2_mask(*reinterpret_cast<__half2 *>(&d[e]), *reinterpret_cast<__half2 *>(&d[e]));
                        const int key = (lane + 32 * e) / G * 2;
                        if (key >= valid) d[e] = 0;
                        else if (key + 1 >= valid) d[e] &= 0xffffu;
                        if (words % 32 == 0 || lane + 32 * e < words) mine[32 * e] = d[e];
                    }
                    fence_proxy_async_smem();  // before the slot's next bulk copy
                    __syncwarp();
                }
            }
#pragma unroll
            for (int tile = 0; tile < KT; tile++) {
                uint32_t d2[2], v[4][MT / 4];
                const uint8_t *rows16 = vblock + 16 * (tile0 + tile) * row_bytes;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    d2[e] = *reinterpret_cast<const uint32_t *>(vblock + vs_at + (16 * (tile0 + tile) + 8 * e) * 2 * G);
#pragma unroll
                    for (int odd = 0; odd < 2; odd++) {
                        const uint8_t *at = rows16 + (odd ? v_odd : v_even) + 8 * e * row_bytes;
                        if constexpr (MT == 8) *reinterpret_cast<uint2 *>(v[2 * e + odd]) = *reinterpret_cast<const uint2 *>(at);
                        else v[2 * e + odd][0] = *reinterpret_cast<const uint32_t *>(at);
                    }
                }
#pragma unroll
                for (int w = 0; w < MT / 4; w++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const uint32_t x0 = __byte_perm(v[0][w], v[1][w], half ? 0x7632 : 0x5410);
                        const uint32_t x1 = __byte_perm(v[2][w], v[3][w], half ? 0x7632 : 0x5410);
#pragma unroll
                        for (int two = 0; two < 2; two++) {
                            const uint32_t y0 = two ? x0 >> 8 : x0, y1 = two ? x1 >> 8 : x1;
                            const uint32_t a[4] = {kv4_times(kv4_low(y0), d2[0]), kv4_times(kv4_high(y0), d2[0]),
                                                   kv4_times(kv4_low(y1), d2[1]), kv4_times(kv4_high(y1), d2[1])};
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
                                mma_16816(o[nt][4 * w + 2 * half + two], a, pb[tile][nt][0], pb[tile][nt][1]);
                        }
                    }
            }
            next(2 * i + 1);
        } while (unit++, ++i < n && item_at(i) == item);
        ends = unit == units;
        if (ok && !merged) {
            // the item's end in this warp: the output where all of it was, else a part
            const bool whole = begin == 0 && ends;
            const int at = 2 * (int)me + (first_item ? 0 : 1);
            if (lane == 0) {
                if (begin == 0) p.items[item].x = whole ? -1 : at;
                if (ends && !whole) p.items[item].y = (int)me;
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < RP; e++) {
                    float sum = l[nt][e];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    const int r = K::split ? 4 * nt + t : 8 * nt + 2 * t + e;
                    if (r0 + r >= n_rows) continue;
                    const float inverse = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
                    const int token = (r0 + r) / p.group, head = kvh * p.group + (r0 + r) - token * p.group;
                    T *out = static_cast<T *>(p.out) + (size_t)(q.first + token) * p.out_stride + (size_t)head * D + g * MT * 2;
                    float *part = p.part + ((size_t)at * K::rows + r) * (D + 2);
#pragma unroll
                    for (int j = 0; j < MT; j += 4) {
                        float x[8];
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            x[2 * c] = (K::split ? o[nt][j + c][0] + o[nt][j + c][1] : o[nt][j + c][e]) * inverse;
                            x[2 * c + 1] = (K::split ? o[nt][j + c][2] + o[nt][j + c][3] : o[nt][j + c][2 + e]) * inverse;
                        }
                        if (whole) {
                            store8(out + 2 * j, p.wide, x);
                        } else {
#pragma unroll
                            for (int c = 0; c < 8; c += 2)
                                *reinterpret_cast<float2 *>(part + g * MT * 2 + 2 * j + c) = make_float2(x[c], x[c + 1]);
                        }
                    }
                    if (!whole && g == 0) *reinterpret_cast<float2 *>(part + D) = make_float2(m[nt][e], sum);
                }
        }
        unit = 0;  // the next item begins at its first
    }
    if (!ok) {
        // copies may be in flight: see them land (bounded) before the CTA's memory goes
        for (int i = 0; i < SLOTS; i++)
            for (unsigned spin = 0; spin < 1024 && !mbar_test_wait(&bar[i], phases >> i & 1); spin++) __nanosleep(500);
    }
    __syncthreads();
    if (*abort_word) {
        if (threadIdx.x == 0) kv4_report(p.status, kKv4Timeout);
        return;
    }
    if (!merged) return;
    // ---- merge the warps' parts of the block's one item, in warp order
    float *mo = reinterpret_cast<float *>(kv4_smem), *ml = mo + W * K::rows * D;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < RP; e++) {
            float sum = l[nt][e];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const int r = warp * K::rows + (K::split ? 4 * nt + t : 8 * nt + 2 * t + e);
            float *dst = mo + r * D + g * MT * 2;
#pragma unroll
            for (int i = 0; i < MT; i++)
                *reinterpret_cast<float2 *>(dst + 2 * i) =
                    K::split ? make_float2(o[nt][i][0] + o[nt][i][1], o[nt][i][2] + o[nt][i][3])
                             : make_float2(o[nt][i][e], o[nt][i][2 + e]);
            if (g == 0) {
                ml[2 * r] = m[nt][e];
                ml[2 * r + 1] = sum;
            }
        }
    // whether the item begins here (the first warp knows) and ends here (the last one does)
    if (threadIdx.x == 0) *merged_word = begin == 0 ? 2 : 1;
    __syncthreads();
    if (threadIdx.x == 32 * (W - 1) && ends) *abort_word = 1;
    __syncthreads();
    const bool starts_here = *merged_word == 2, ends_here = *abort_word != 0, whole = starts_here && ends_here;
    const int at = 2 * blockIdx.x * W, n_rows = q.count * p.group;
    if (threadIdx.x == 0) {
        if (starts_here) p.items[item].x = whole ? -1 : at;
        if (ends_here && !whole) p.items[item].y = blockIdx.x * W + W - 1;
    }
    if (!whole)  // the other warps' parts are empty
        for (int i = threadIdx.x; i < (W - 1) * K::rows; i += 32 * W)
            *reinterpret_cast<float2 *>(p.part + ((size_t)(at + 2 * (1 + i / K::rows)) * K::rows + i % K::rows) * (D + 2) + D) =
                make_float2(-INFINITY, 0.0f);
    constexpr int per = D / 8;  // threads of a row, 8 dims each
    for (int i = threadIdx.x; i < K::rows * per; i += 32 * W) {
        const int r = i / per, d = i % per * 8;
        if (r0 + r >= n_rows) continue;
        float top = -INFINITY, sum = 0.0f, x[8] = {};
#pragma unroll
        for (int w = 0; w < W; w++) top = fmaxf(top, ml[2 * (w * K::rows + r)]);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const int from = w * K::rows + r;
            // a part without keys has l = 0; one whose scores are NaN has l = NaN and stays
            const float weight = ml[2 * from + 1] == 0.0f ? 0.0f : ml[2 * from] == top ? 1.0f : exp2_fast(ml[2 * from] - top);
            sum = fmaf(weight, ml[2 * from + 1], sum);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = fmaf(weight, mo[from * D + d + e], x[e]);
        }
        if (whole) {
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] *= inverse;
            const int token = (r0 + r) / p.group, head = kvh * p.group + (r0 + r) - token * p.group;
            store8(static_cast<T *>(p.out) + (size_t)(q.first + token) * p.out_stride + (size_t)head * D + d, p.wide, x);
        } else {
            float *part = p.part + ((size_t)at * K::rows + r) * (D + 2);
#pragma unroll
            for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2 *>(part + d + e) = make_float2(x[e], x[e + 1]);
            if (d == 0) *reinterpret_cast<float2 *>(part + D) = make_float2(top, sum);
        }
    }
}

// `Warps` warps: the parts of an item's row, in a fixed order, to a row's head. at(i) is
// part i's D + 2 floats. Every thread of the block calls it.
template <int D, typename T, int Warps, typename At>
__device__ __forceinline__ void kv4_combine(const Kv4AttnParams &p, At &&at, int parts, int row, int head)
{
    constexpr int per = D / 32;
    const int lane = threadIdx.x & 31, warp = Warps == 1 ? 0 : threadIdx.x >> 5;
    float top = -INFINITY, total = 0.0f, x[per] = {};
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, at(i)[D]);
    top = warp_max(top);
    for (int i0 = 32 * warp; i0 < parts; i0 += 32 * Warps) {
        float weight = 0.0f;
        if (i0 + lane < parts) {
            const float2 ml = *reinterpret_cast<const float2 *>(at(i0 + lane) + D);
            weight = ml.y == 0.0f ? 0.0f : ml.x == top ? 1.0f : exp2_fast(ml.x - top);
            total = fmaf(weight, ml.y, total);
        }
        // parts without a weight are not read
        for (unsigned left = __ballot_sync(0xffffffffu, weight != 0.0f); left;) {
            float v[4][per], w[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = left ? __ffs(left) - 1 : 0;
                w[u] = __shfl_sync(0xffffffffu, weight, i);
                if (!left) w[u] = 0.0f;
                const float *src = at(i0 + i) + per * lane;
#pragma unroll
                for (int e = 0; e < per; e += 2) {
                    float2 two = make_float2(0.0f, 0.0f);
                    if (left) two = *reinterpret_cast<const float2 *>(src + e);
                    v[u][e] = two.x, v[u][e + 1] = two.y;
                }
                left &= left - 1;
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int e = 0; e < per; e++) x[e] = fmaf(w[u], v[u][e], x[e]);
        }
    }
    total = warp_sum(total);
    if (Warps > 1) {
        __shared__ float merge[Warps][D + 1];
#pragma unroll
        for (int e = 0; e < per; e++) merge[warp][per * lane + e] = x[e];
        if (lane == 0) merge[warp][D] = total;
        __syncthreads();
        if (warp) return;
        total = 0.0f;
#pragma unroll
        for (int e = 0; e < per; e++) x[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < Warps; w++) {
            total += merge[w][D];
#pragma unroll
            for (int e = 0; e < per; e++) x[e] += merge[w][per * lane + e];
        }
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    T *dst = static_cast<T *>(p.out) + (size_t)row * p.out_stride + (size_t)head * D + per * lane;
#pragma unroll
    for (int e = 0; e < per; e++) dst[e] = from_float<T>(x[e] * inverse);
}

// The decode kernel's rows, [item][row of the tile]: 4 rows a block, a warp each, or,
// where items have many parts, one row a block of 8 warps.
template <int D, typename T, int Warps>
static __global__ void __launch_bounds__(Warps == 1 ? 128 : 32 * Warps) kv4_combine_kernel(Kv4AttnParams p, int tile_rows)
{
    const int at = Warps == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x, item = at / tile_rows;
    const int r0 = item % p.tiles * tile_rows, r = r0 + at % tile_rows;
    const int kvh = item / p.tiles % p.cache.heads, s = item / p.tiles / p.cache.heads;
    pdl_wait();
    pdl_launch_dependents();
    if (s >= p.rows.sequences) return;
    const Kv4Sequence q = kv4_sequence(p.rows, s);
    if (!q.ok || q.count * p.group > p.most || r >= q.count * p.group) return;
    const int token = r / p.group, head = kvh * p.group + r - token * p.group;
    int2 where = make_int2(0, -1);  // no keys: no parts
    if (q.length > 0) {
        where.x = p.items[item].x;
        if (where.x < 0) return;
        where.y = p.items[item].y;
    }
    // the first part, then the first of each warp up to the last
    const float *part = p.part + (size_t)(r - r0) * (D + 2);
    const int first_warp = where.x >> 1;
    kv4_combine<D, T, Warps>(
        p,
        [&](int i) { return part + (size_t)(i == 0 ? where.x : 2 * (first_warp + i)) * tile_rows * (D + 2); },
        where.y < 0 ? 0 : where.y - first_warp + 1, q.first + token, head);
}

}  // namespace lun
