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
// sequences), they merge first, through shared memory. Where that leaves a warp a page
// or less (one sequence, or short ones), time is what the steps wait for one another:
// then a cluster of 1 to 8 blocks takes an item, its warps shares of it in 16 keys, and
// merges it through distributed shared memory, in one launch (one sequence, 8 KV heads
// of 4 query heads, FP32, in a captured graph: 500 keys 7.5 us by clusters, 10.7 by the list; 2000
// keys 9.7 and 10.3; 4096 keys 12.3 and 10.8; 8192 keys 17.4 and 13.1). Clusters of 16 do not all
// find room at once. 4 blocks of 16 warps instead of 8 of 8: 8.8 us at 500 keys.
// Blocks of the list: 4 an SM, 3 slots a warp (3 of 4 slots: 127 us for 126 at four FP32 sequences of
// 131072 keys, 150 for 152 at those below). Four BF16 sequences of 131072 keys, 8 KV heads of 8, take
// 152 us with the combine in a captured graph, 4.0 TB/s; 64 FP32 sequences of up to 4352 keys, 8 KV
// heads of 4, 43 us, 37 of them in this kernel under a profiler, whose SMs are active for three
// quarters of it and issue in half of the slots: they wait for the chains of conversion, product and
// softmax.
//
// The products run on mma.sync m16n8k16 with FP16 operands and FP32 sums: a
// decode step has 1 to 16 query rows a KV head, so a tcgen05 tile of 128 rows would be
// mostly padding, while here the rows sit in the n = 8 side. FP32 rows of q and
// weights of the softmax enter as FP16 hi + lo parts in neighbouring columns
// (22 bits together), so one MMA serves 4 rows at FP32 grade. Up to 4
// rows of 16 bits go the same way. More of them have q in one FP16 (exact after a power-of-two
// scaling but for what lies below 2^-24 of the row's largest), 8 rows an MMA, and their weights in two
// FP16 all the same, in two MMAs (with one, off by 2^-12, FP16 outputs lost a fifth more than
// their own rounding does).
//   S = K Q^T     A: 16 keys x 16 dims of c - 8 (an AND and a subtraction); a group's sum, in FP32, is
//                 scaled by d after its two MMAs. Codes as they are, with -8 sum q to start a sum
//                 from, take as long and lose six times as much: the tensor core cuts sums to FP32
//                 towards zero, and those are larger.
//   O^T = V^T P^T A: 16 dims x 16 keys of d * (c - 8) * 2^-9. Four bits alone in a half's lowest eight
//                 are a subnormal, c * 2^-24 or c * 2^-20, that one AND leaves; one fused multiply-add
//                 follows, whose exact result FP16 holds while 2^-8 <= |d| < 2; a page with
//                 another d takes two more steps a code. B: the weights, moved from S's layout by
//                 movmatrix.
// The tensor core cuts what it adds up towards zero: over values of one sign, about 1.9e-7 of the
// sum so far each time, so that 443 pages in a row (64 FP32 sequences of 131072 keys) lost 1.7e-4.
// So the list's warps take O out every 4 pages (16-bit rows, which add up two products a step, every
// 12) and add those sums up to nearest: 1.4e-6 there, 0.9e-6 over 68 pages. Four FP32 sequences of
// 131072 keys take 126 us for 122, four BF16 ones with 8 rows 151 for 146. L2's own additions
// (red.add), which nothing waits for, take 132 and 156. A cluster's warps add up 4 units of 16
// keys at most.
#pragma once
#include "async.cuh"
#include "attention.cuh"
#include "kv4.cuh"

#include <cooperative_groups.h>
#include <type_traits>

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
    int ranks;     // decode kernel: blocks of an item's cluster
    int most;      // decode kernel: its sequences have at most so many rows a KV head
    int split_pages, splits;  // block kernel: pages of a split; splits, 1: the kernel writes the output itself
    bool wide;
    // unnormalised o, m, l, D + 2 floats a row: [2 warp + (0 the warp's first item, 1 its last)][row of
    // the tile] of the decode kernel, which keeps what it takes out of o there meanwhile, [row][query
    // head][split] of the block kernel
    float *part;
    int2 *items;     // decode kernel: an item's first part (-1: it is written out) and last warp
    int list_warps;  // and the warps of the list
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

// What this CTA has in flight once a wait gave up: the abort word does not end this wait, half a
// millisecond does.
__device__ __forceinline__ bool kv4_landed(uint64_t *bar, unsigned parity)
{
    for (unsigned spin = 0; spin < 1024; spin++) {
        if (mbar_test_wait(bar, parity)) return true;
        __nanosleep(500);
    }
    return false;
}

// The softmax's weights are taken times 2^14, and l with them: the largest is
// 16384, and the FP16 parts of a weight keep 22 bits down to 2^-28 of it, where a
// largest weight of 1 would leave small ones on the 2^-24 grid of FP16's
// subnormals. Where V is not times 2^-9, they are 2^9 smaller.
constexpr float kWeightShift = 14.0f, kValueShift = 9.0f, kValueScale = 512.0f;

constexpr int kListWarps = 4, kListSlots = 3, kListCtas = 4;  // of a block; of a warp; of an SM
constexpr int kClusterWarps = 8, kClusterSlots = 4, kClusterRanks = 8;  // of a block; of a warp; blocks at most

template <int D, typename T, int NT, int W, bool S> struct Kv4Decode {
    static constexpr bool split = S;                 // hi and lo columns
    static constexpr int lane_rows = split ? 1 : 2;  // query rows of a lane and n tile
    static constexpr int rows = 4 * NT * lane_rows;  // query rows of a tile
    static constexpr int keys = W > kListWarps ? 16 : 64;  // of a unit
    static constexpr int slots = W > kListWarps ? kClusterSlots : kListSlots;
    static constexpr int drain = sizeof(T) == 4 ? 4 : 12;  // pages that the list sums up on the tensor cores
    static constexpr int codes = keys * D / 2;
    static constexpr int half = codes + keys * 2 * (D / 32);  // K or V of a unit, laid out as in a page
    static constexpr int ring = W * slots * half;
    static constexpr int merge = (W + 1) * rows * (D + 2) * 4;  // the warps' parts, the block's
    static constexpr int bars = (ring > merge ? ring : merge);
    static constexpr int prefix = bars + W * slots * 8;  // an int a thread, one a warp
    static constexpr int smem = prefix + 33 * W * 4 + 16;
};

__device__ __forceinline__ float exp2_fast(float x)  // 2 ulp; 0 below 2^-126
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Four codes in the bytes' low and high nibbles of both halves -> c - 8 in FP16:
// a = (nibble 0, nibble 4), b = (nibble 1, nibble 5) of a word. The step is a published one of 4-bit
// weights: a nibble put under the exponent of 1024 is 1024 + c, or 1024 + 16 c from the
// upper one, and one exact operation takes the 1024 off.
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
// The nibbles alone: c * 2^-24 and c * 2^-20 as FP16 subnormals.
__device__ __forceinline__ uint32_t kv4_code(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t kv4_code16(uint32_t w) { return w & 0x00f000f0u; }
__device__ __forceinline__ uint32_t kv4_fma(uint32_t v, __half2 x, __half2 y)
{
    const __half2 h = __hfma2(*reinterpret_cast<__half2 *>(&v), x, y);
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

// 2^-e with 2^e the power of two at or below x, e within +-120; 1 for zero. Of an infinity a NaN,
// which the whole row becomes: scores that are all -infinity would look like masked ones.
__device__ __forceinline__ float power_scale(float x, float &back)
{
    int e = (int)(__float_as_uint(x) >> 23 & 255) - 127;
    const bool infinite = e == 128;
    if (x == 0.0f || infinite) e = 0;
    e = max(-120, min(120, e));
    back = __uint_as_float((uint32_t)(127 + e) << 23);
    return infinite ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(127 - e) << 23);
}


// What the decode kernel does of a sequence: units of KT * 16 keys an item, items.
struct Kv4Share {
    int units, tiles, all;  // `all`: units of all its items; the caller bounds their sum by 2^31
};
template <int KT, int ROWS>
__device__ __forceinline__ Kv4Share kv4_share(const Kv4AttnParams &p, const Kv4Sequence &q)
{
    Kv4Share w = {0, 0, 0};
    const int rows = q.count * p.group;
    if (!q.ok || rows == 0 || rows > p.most) return w;
    w.units = (q.length + 16 * KT - 1) / (16 * KT);
    w.tiles = (rows + ROWS - 1) / ROWS;
    w.all = w.units * p.cache.heads * w.tiles;
    return w;
}

// Items [sequence][KV head][row tile of p.tiles]. W = kListWarps: any number of blocks
// share the list. W = kClusterWarps: a cluster per item.
template <int D, typename T, int NT, int W, bool S>
static __global__ void __launch_bounds__(32 * W, W > kListWarps ? 1 : NT == 1 ? kListCtas : 2)
    kv4_decode_kernel(Kv4AttnParams p)
{
    namespace cg = cooperative_groups;
    using L = Kv4Layout<D>;
    using K = Kv4Decode<D, T, NT, W, S>;
    constexpr int G = L::groups, MT = D / 16, RP = K::lane_rows, SLOTS = K::slots, KT = K::keys / 16;
    constexpr bool cluster = W > kListWarps;
    constexpr int row_bytes = D / 2;
    extern __shared__ __align__(128) uint8_t kv4_smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(kv4_smem + K::bars);
    int *prefix = reinterpret_cast<int *>(kv4_smem + K::prefix);  // of a warp's 32 runs of sequences; warps' totals
    volatile int *abort_word = reinterpret_cast<volatile int *>(prefix + 33 * W);
    volatile int *merged_word = abort_word + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint64_t *bar = bars + warp * SLOTS;
    if (threadIdx.x == 0) *abort_word = 0;
    if (lane < SLOTS) mbar_init(&bar[lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_wait();
    pdl_launch_dependents();

    // ---- this warp's units [u0, u1): of the cluster's item, or of the list
    int s = 0, base = 0, u0 = 0, u1 = 0, me = 0, cluster_item = 0;
    bool shared_item = cluster;  // whether the block's warps share one item
    const int ranks = cluster ? p.ranks : 1, rank = cluster ? (int)blockIdx.x % ranks : 0;
    if constexpr (cluster) {
        cluster_item = blockIdx.x / ranks;
        s = cluster_item / p.tiles / p.cache.heads;
        const Kv4Sequence q = kv4_sequence(p.rows, s);
        const Kv4Share w = kv4_share<KT, K::rows>(p, q);
        if (!q.ok && threadIdx.x == 0) kv4_report(p.status, kKv4BadRows);
        if (cluster_item % p.tiles >= w.tiles) return;  // the whole cluster
        const int warps = ranks * W;
        me = rank * W + warp;
        u0 = w.units / warps * me + w.units % warps * me / warps;
        u1 = w.units / warps * (me + 1) + w.units % warps * (me + 1) / warps;
        __syncthreads();
    } else {
        const int run = (p.rows.sequences + 32 * W - 1) / (32 * W);  // sequences of a thread
        int total = 0, before = 0;
        {
            int sum = 0;
            for (int i = 0; i < run; i++) {
                const int s = threadIdx.x * run + i;
                if (s >= p.rows.sequences) break;
                const Kv4Sequence q = kv4_sequence(p.rows, s);
                if (!q.ok && blockIdx.x == 0) kv4_report(p.status, kKv4BadRows);
                sum += kv4_share<KT, K::rows>(p, q).all;
            }
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += other;
            }
            prefix[threadIdx.x] = upto - sum;
            if (lane == 31) prefix[32 * W + warp] = upto;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; w++) total += prefix[32 * W + w];
        }
        const int warps = min((int)gridDim.x * W, total);
        me = blockIdx.x * W + warp;
        if ((int)blockIdx.x * W >= warps) return;
        const int each = total / warps, more = total % warps;
        auto share_of = [&](int i) { return i >= warps ? total : each * i + more * i / warps; };
        u0 = share_of(me);
        u1 = share_of(me + 1);
        // the sequence of u0 and its first unit
        if (u1 > u0) {
            int k = 0;
#pragma unroll
            for (int w = 0; w < W; w++) {  // the warp's runs that u0 lies in, then the run
                const int all = prefix[32 * W + w];
                if (u0 >= before && u0 < before + all) {
                    k = 32 * w + 31 - __clz(__ballot_sync(0xffffffffu, before + prefix[32 * w + lane] <= u0));
                    base = before + prefix[k];
                }
                before += all;
            }
            s = k * run;
            for (;;) {
                const int all = kv4_share<KT, K::rows>(p, kv4_sequence(p.rows, s)).all;
                if (u0 < base + all) break;
                base += all;
                s++;
            }
        }
        // the block's warps share an item if the first one's reaches to the last one's end
        if (warp == 0 && (int)blockIdx.x * W + W <= warps) {
            const Kv4Share w = kv4_share<KT, K::rows>(p, kv4_sequence(p.rows, s));
            const int left = w.units - (u0 - base) % w.units;
            if (lane == 0) *merged_word = u0 + left >= share_of(me + W);
        } else if (threadIdx.x == 0) {
            *merged_word = 0;
        }
        __syncthreads();
        shared_item = *merged_word != 0;
    }
    const int n = u1 - u0;
    const bool merged = shared_item;
    // unit base_i + lane of the list: its block in the layer (or none) and its item
    auto map = [&](int i, uint32_t &block, int &item, int &unit) {
        block = 0xffffffffu;
        item = -1;
        unit = 0;
        const int u = u0 + i;
        if (u >= u1) return;
        if constexpr (cluster) {
            const int kvh = cluster_item / p.tiles % p.cache.heads;
            unit = u;
            item = cluster_item;
            const int id = p.rows.page_tables[s * p.rows.table_stride + (KT == 4 ? unit : unit >> 2)];
            if ((unsigned)id < (unsigned)p.cache.pages) block = (uint32_t)id * (uint32_t)p.cache.heads + kvh;
            else kv4_report(p.status, kKv4BadPage);
            return;
        }
        Kv4Share w;
        for (;;) {
            w = kv4_share<KT, K::rows>(p, kv4_sequence(p.rows, s));
            if (u < base + w.all) break;
            base += w.all;
            s++;
        }
        const int rest = u - base, of = rest / w.units, kvh = of / w.tiles;
        unit = rest - of * w.units;
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
        const uint8_t *src = p.cache.layer + (size_t)id * L::block + (h & 1 ? L::block / 2 : 0);
        uint8_t *dst = buffers + slot * K::half;
        if (KT == 4) {
            mbar_expect_tx(&bar[slot], K::half);
            bulk_g2s(dst, src, K::half, &bar[slot]);
        } else {
            constexpr int codes = 16 * row_bytes, scales = 32 * G;
            mbar_expect_tx(&bar[slot], codes + scales);
            bulk_g2s(dst, src + quarter * codes, codes, &bar[slot]);
            bulk_g2s(dst + codes, src + L::codes + quarter * scales, scales, &bar[slot]);
        }
    };
#pragma unroll
    for (int h = 0; h < SLOTS; h++)
        if (h < 2 * n) issue(h, h);
    // byte offsets of the lane's first reads in a half block; 16 keys on are 16 rows on, the swizzle the same
    const int k_at = g * row_bytes + 4 * G * t, ks_at = L::k_scale(g, 0) - L::codes + K::codes;
    const int v_even = L::v_word(2 * t, g * (MT / 4)) - L::block / 2, v_odd = v_even ^ row_bytes;
    const int vs_at = L::v_scale(2 * t, g * (D / 8) / 32) - L::block / 2 - L::codes + K::codes;
    bool ok = true, ends = false;
    unsigned phases = 0;  // parity of each slot's next wait
    int slot = 0;
    auto next = [&](int h) {  // done with half h: every lane has read it; refill its slot
        __syncwarp();
        if (h + SLOTS < 2 * n) issue(h + SLOTS, slot);
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
    };
    float m[NT][RP], l[NT][RP], o[NT][MT][4];
    float since[NT][RP];  // the list: what has scaled o since it was taken out last
    int item = 0, begin = 0, r0 = 0, kvh = 0;
    Kv4Sequence q = {0, 0, 0, false};
    if (cluster) {  // a warp without units has a part too
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int e = 0; e < RP; e++) m[nt][e] = -INFINITY, l[nt][e] = 0.0f;
#pragma unroll
            for (int j = 0; j < MT; j++) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.0f;
        }
        item = cluster_item;
        r0 = item % p.tiles * K::rows;
        kvh = item / p.tiles % p.cache.heads;
        q = kv4_sequence(p.rows, s);
    }
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
        float back[NT][RP];      // what a score is multiplied with, of the lane's rows 4 nt + t or 8 nt + 2 t + (0, 1)
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
                since[nt][e] = 1.0f;
            }
#pragma unroll
            for (int j = 0; j < MT; j++) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.0f;
        }
        const int all_see = q.length - q.count + r0 / p.group;  // every row of the tile sees keys up to here
        // The list takes o out every K::drain pages, into the place of the part that it would leave, a lane
        // its own values (an FP32 row's two columns as one): sum * since + o.
        float4 *sums = nullptr;
        if constexpr (!cluster)
            sums = reinterpret_cast<float4 *>(p.part + (size_t)(2 * me + (first_item ? 0 : 1)) * K::rows * (D + 2)) + lane;
        auto drain = [&](bool has, bool last) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < MT; j += K::split ? 2 : 1) {
                    float (&a)[4] = o[nt][j], (&b)[4] = o[nt][K::split ? j + 1 : j];
                    float4 *at = sums + 32 * (nt * MT + j) / (K::split ? 2 : 1);
                    float4 v = K::split ? make_float4(a[0] + a[1], a[2] + a[3], b[0] + b[1], b[2] + b[3])
                                        : make_float4(a[0], a[1], a[2], a[3]);
                    if (has) {
                        const float4 before = *at;
                        const float s0 = since[nt][0], s1 = K::split ? s0 : since[nt][RP - 1];
                        v.x = fmaf(before.x, s0, v.x), v.y = fmaf(before.y, s1, v.y);
                        v.z = fmaf(before.z, s0, v.z), v.w = fmaf(before.w, s1, v.w);
                    }
                    if (!last) {
                        *at = v;
                        v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                    if constexpr (K::split) {
                        a[0] = v.x, a[2] = v.y, b[0] = v.z, b[2] = v.w;
                        a[1] = a[3] = b[1] = b[3] = 0.0f;
                    } else {
                        a[0] = v.x, a[1] = v.y, a[2] = v.z, a[3] = v.w;
                    }
                }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < RP; e++) since[nt][e] = 1.0f;
        };
        do {
            if (!cluster && unit != begin && (unit - begin) % K::drain == 0) drain(unit - begin > K::drain, false);
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
            const int p0 = unit * 16 * KT;
            const uint8_t *block = buffers + slot * K::half;
            float sc[KT][NT][2][RP];
#pragma unroll
            for (int tile = 0; tile < KT; tile++) {
                float acc[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
                uint32_t ka[G], kb[G], da[G / 2], db[G / 2];
                const uint8_t *row = block + k_at + 16 * tile * row_bytes, *scale = block + ks_at + 32 * G * tile;
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
                        float c[4] = {};
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
            if (!(ok = kv4_warp_wait(&bar[slot], phases >> slot & 1, abort_word))) break;
            phases ^= 1u << slot;
            uint8_t *vblock = buffers + slot * K::half;
            uint8_t *vscales = vblock + K::codes;  // [position / 2][group][position % 2]
            bool small = true;  // every scale is 0 or 2^-8 <= |d| < 2
            {
                constexpr int words = KT * 8 * G, each = (words + 31) / 32;
                uint32_t *mine = reinterpret_cast<uint32_t *>(vscales) + each * lane, d[each] = {};
                const bool has = words % 32 == 0 || lane < words;
                const int valid = q.length - p0;
                if constexpr (each == 4) *reinterpret_cast<uint4 *>(d) = *reinterpret_cast<const uint4 *>(mine);
                else if constexpr (each == 2) *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(mine);
                else if (has) d[0] = *mine;
                const __half2 least = __half2half2(__ushort_as_half(0x1c00)), most = __half2half2(__ushort_as_half(0x3fff));
                // quick: zeros are odd too; exact: they are not
                auto odd = [&](bool exact) {
                    __half2 high = __habs2(*reinterpret_cast<__half2 *>(&d[0])), low = high;
                    uint32_t bad = 0;
#pragma unroll
                    for (int e = 0; e < each; e++) {
                        const __half2 x = __habs2(*reinterpret_cast<__half2 *>(&d[e]));
                        high = __hmax2_nan(high, x);
                        low = __hmin2(low, x);
                        if (exact) bad |= __hlt2_mask(x, least) & __hne2_mask(x, __half2half2(__ushort_as_half(0)));
                    }
                    bad |= __hgtu2_mask(high, most) | (exact ? 0u : __hlt2_mask(low, least));
                    return __any_sync(0xffffffffu, has && bad != 0);
                };
                if (valid < 16 * KT || odd(false)) {
                    // scales behind the last position (whatever those slots hold) and NaNs become zeros
                    // before the MMAs, in which a weight of zero would not keep a NaN away from a row
                    // that does not see its position; the rows that do see a NaN take it here
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
                        const int key = (each * lane + e) / G * 2;
                        if (key >= valid) d[e] = 0;
                        else if (key + 1 >= valid) d[e] &= 0xffffu;
                        if (has) mine[e] = d[e];
                    }
                    fence_proxy_async_smem();  // before the slot's next bulk copy
                    __syncwarp();
                    small = !odd(true);
                }
            }
            const float shift = small ? kWeightShift : kWeightShift - kValueShift, count = small ? 1.0f : kValueScale;
            uint32_t pb[KT][NT][2], pl[KT][NT][2];  // pl: 16-bit rows' lo parts
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
                        if (!cluster) since[nt][e] *= corr[e];
                    }
#pragma unroll
                    for (int j = 0; j < MT; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[nt][j][e] *= corr[K::split ? 0 : e & 1];
                }
                // a row without any key yet: exp2(-inf - 0) = 0
#pragma unroll
                for (int e = 0; e < RP; e++) zero[e] = m[nt][e] == -INFINITY ? 0.0f : m[nt][e] - shift;
#pragma unroll
                for (int tile = 0; tile < KT; tile++)
#pragma unroll
                    for (int k8 = 0; k8 < 2; k8++) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < RP; e++) {
                            w[e] = exp2_fast(sc[tile][nt][k8][e] - zero[e]);
                            l[nt][e] = fmaf(w[e], count, l[nt][e]);
                        }
                        __half2 two;
                        if constexpr (K::split) {
                            const __half h = __float2half_rn(w[0]);
                            two = __halves2half2(h, __float2half_rn(w[0] - __half2float(h)));
                        } else {
                            two = __floats2half2_rn(w[0], w[1]);
                            const __half2 rest = __floats2half2_rn(w[0] - __low2float(two), w[1] - __high2float(two));
                            pl[tile][nt][k8] = movmatrix_trans(*reinterpret_cast<const uint32_t *>(&rest));
                        }
                        pb[tile][nt][k8] = movmatrix_trans(*reinterpret_cast<const uint32_t *>(&two));
                    }
            }
            auto values = [&](auto fused) {
#pragma unroll
                for (int tile = 0; tile < KT; tile++) {
                    uint32_t d2[2], v[4][MT / 4];
                    const uint8_t *rows16 = vblock + 16 * tile * row_bytes;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        d2[e] = *reinterpret_cast<const uint32_t *>(vblock + vs_at + (16 * tile + 8 * e) * 2 * G);
#pragma unroll
                        for (int odd = 0; odd < 2; odd++) {
                            const uint8_t *at = rows16 + (odd ? v_odd : v_even) + 8 * e * row_bytes;
                            if constexpr (MT == 8) *reinterpret_cast<uint2 *>(v[2 * e + odd]) = *reinterpret_cast<const uint2 *>(at);
                            else v[2 * e + odd][0] = *reinterpret_cast<const uint32_t *>(at);
                        }
                    }
                    // c 2^-24 (d 2^15) - d 2^-6 = d (c - 8) 2^-9, of a high nibble from c 2^-20
                    __half2 x[2], x16[2], y[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const __half2 d = *reinterpret_cast<__half2 *>(&d2[e]);
                        x[e] = __hmul2(d, __half2half2(__ushort_as_half(0x7800)));    // 2^15
                        x16[e] = __hmul2(d, __half2half2(__ushort_as_half(0x6800)));  // 2^11
                        y[e] = __hmul2(d, __half2half2(__ushort_as_half(0xa400)));    // -2^-6
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
                                uint32_t a[4];
                                if constexpr (decltype(fused)::value) {
                                    a[0] = kv4_fma(kv4_code(y0), x[0], y[0]);
                                    a[1] = kv4_fma(kv4_code16(y0), x16[0], y[0]);
                                    a[2] = kv4_fma(kv4_code(y1), x[1], y[1]);
                                    a[3] = kv4_fma(kv4_code16(y1), x16[1], y[1]);
                                } else {
                                    a[0] = kv4_times(kv4_low(y0), d2[0]);
                                    a[1] = kv4_times(kv4_high(y0), d2[0]);
                                    a[2] = kv4_times(kv4_low(y1), d2[1]);
                                    a[3] = kv4_times(kv4_high(y1), d2[1]);
                                }
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) {
                                    float (&sum)[4] = o[nt][4 * w + 2 * half + two];
                                    if constexpr (!K::split) mma_16816(sum, a, pl[tile][nt][0], pl[tile][nt][1]);
                                    mma_16816(sum, a, pb[tile][nt][0], pb[tile][nt][1]);
                                }
                            }
                        }
                }
            };
            if (small) values(std::true_type());
            else values(std::false_type());
            next(2 * i + 1);
        } while (unit++, ++i < n && item_at(i) == item);
        ends = unit == units;
        if (!cluster && ok && unit - begin > K::drain) {
            drain(true, true);
            __syncwarp();  // the part's place is written by other lanes from here on
        }
        if (ok && !merged) {
            // the item's end in this warp: the output where all of it was, else a part
            const bool whole = begin == 0 && ends;
            const int at = 2 * me + (first_item ? 0 : 1);
            if (lane == 0) {
                if (begin == 0) p.items[item].x = whole ? -1 : at;
                if (ends && !whole) p.items[item].y = me;
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
                    const float inverse = !whole ? kValueScale : sum == 0.0f ? 0.0f : kValueScale / sum;
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
        for (int i = 0; i < SLOTS; i++) kv4_landed(&bar[i], phases >> i & 1);
    }
    __syncthreads();
    if (*abort_word && threadIdx.x == 0) kv4_report(p.status, kKv4Timeout);
    if (!cluster && (*abort_word || !merged)) return;  // a cluster goes on together
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
                    K::split ? make_float2((o[nt][i][0] + o[nt][i][1]) * kValueScale, (o[nt][i][2] + o[nt][i][3]) * kValueScale)
                             : make_float2(o[nt][i][e] * kValueScale, o[nt][i][2 + e] * kValueScale);
            if (g == 0) {
                ml[2 * r] = m[nt][e];
                ml[2 * r + 1] = sum;
            }
        }
    bool starts_here = false, ends_here = false;
    int at = 0;
    const int n_rows = q.count * p.group;
    if constexpr (cluster) {
        __syncthreads();
    } else {
        // whether the item begins here (the first warp knows) and ends here (the last one does)
        if (threadIdx.x == 0) *merged_word = begin == 0 ? 2 : 1;
        __syncthreads();
        if (threadIdx.x == 32 * (W - 1) && ends) *abort_word = 1;
        __syncthreads();
        starts_here = *merged_word == 2;
        ends_here = *abort_word != 0;
        at = 2 * blockIdx.x * W;
        if (threadIdx.x == 0) {
            if (starts_here) p.items[item].x = ends_here ? -1 : at;
            if (ends_here && !starts_here) p.items[item].y = blockIdx.x * W + W - 1;
        }
        if (!(starts_here && ends_here))  // the other warps' parts are empty
            for (int i = threadIdx.x; i < (W - 1) * K::rows; i += 32 * W)
                *reinterpret_cast<float2 *>(p.part + ((size_t)(at + 2 * (1 + i / K::rows)) * K::rows + i % K::rows) * (D + 2) + D) =
                    make_float2(-INFINITY, 0.0f);
    }
    const bool whole = cluster ? ranks == 1 : starts_here && ends_here;
    float *block_part = ml + 2 * W * K::rows;  // a cluster's: [row][D + 2]
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
            float *part = cluster ? block_part + r * (D + 2) : p.part + ((size_t)at * K::rows + r) * (D + 2);
#pragma unroll
            for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2 *>(part + d + e) = make_float2(x[e], x[e + 1]);
            if (d == 0) *reinterpret_cast<float2 *>(part + D) = make_float2(top, sum);
        }
    }
    if constexpr (cluster) {
        if (ranks == 1) return;
        // the blocks' parts in rank order: each block finishes a share of the rows' dims
        const cg::cluster_group group = cg::this_cluster();
        group.sync();
        for (int i = rank * 32 * W + threadIdx.x; i < K::rows * per; i += ranks * 32 * W) {
            const int r = i / per, d = i % per * 8;
            if (r0 + r >= n_rows) continue;
            float top = -INFINITY, sum = 0.0f, x[8] = {};
            for (int k = 0; k < ranks; k++) top = fmaxf(top, group.map_shared_rank(block_part, k)[r * (D + 2) + D]);
#pragma unroll 4
            for (int k = 0; k < ranks; k++) {
                const float *part = group.map_shared_rank(block_part, k) + r * (D + 2);
                const float2 ml2 = *reinterpret_cast<const float2 *>(part + D);
                const float weight = ml2.y == 0.0f ? 0.0f : ml2.x == top ? 1.0f : exp2_fast(ml2.x - top);
                sum = fmaf(weight, ml2.y, sum);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float2 v = *reinterpret_cast<const float2 *>(part + d + e);
                    x[e] = fmaf(weight, v.x, x[e]);
                    x[e + 1] = fmaf(weight, v.y, x[e + 1]);
                }
            }
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] *= inverse;
            const int token = (r0 + r) / p.group, head = kvh * p.group + (r0 + r) - token * p.group;
            store8(static_cast<T *>(p.out) + (size_t)(q.first + token) * p.out_stride + (size_t)head * D + d, p.wide, x);
        }
        group.sync();  // no block's shared memory goes while another reads it
    }
}

// `Warps` warps: the parts of an item's row, in a fixed order, to a row's head. at(i) is
// part i's D + 2 floats. Every thread of the block calls it. What it costs is trips to
// L2 one after the other, so a warp's parts are fetched eight at a time, the rows
// together with their maxima and sums.
template <int D, typename T, int Warps, typename At>
__device__ __forceinline__ void kv4_combine(const Kv4AttnParams &p, At &&at, int parts, int row, int head)
{
    constexpr int per = D / 32, batch = 8;
    const int lane = threadIdx.x & 31, warp = Warps == 1 ? 0 : threadIdx.x >> 5;
    float top = -INFINITY, total = 0.0f, x[per] = {};
    // a part without keys has l = 0, whatever else it holds
    auto weigh = [&](float m, float l) { return l == 0.0f ? 0.0f : m == top ? 1.0f : exp2_fast(m - top); };
    for (int i0 = warp; i0 < parts; i0 += batch * Warps) {
        float2 ml[batch], v[batch][per / 2];
#pragma unroll
        for (int u = 0; u < batch; u++) {
            ml[u] = make_float2(-INFINITY, 0.0f);
            if (i0 + u * Warps >= parts) continue;
            const float *src = at(i0 + u * Warps);
            ml[u] = *reinterpret_cast<const float2 *>(src + D);
#pragma unroll
            for (int e = 0; e < per / 2; e++) v[u][e] = *reinterpret_cast<const float2 *>(src + per * lane + 2 * e);
        }
        float high = top;
#pragma unroll
        for (int u = 0; u < batch; u++) high = fmaxf(high, ml[u].x);
        const float corr = high == top ? 1.0f : exp2_fast(top - high);
        top = high;
        total *= corr;
#pragma unroll
        for (int e = 0; e < per; e++) x[e] *= corr;
#pragma unroll
        for (int u = 0; u < batch; u++) {
            const float w = weigh(ml[u].x, ml[u].y);
            if (w == 0.0f && ml[u].y == 0.0f) continue;
            total = fmaf(w, ml[u].y, total);
#pragma unroll
            for (int e = 0; e < per; e += 2) {
                x[e] = fmaf(w, v[u][e / 2].x, x[e]);
                x[e + 1] = fmaf(w, v[u][e / 2].y, x[e + 1]);
            }
        }
    }
    if (Warps > 1) {
        __shared__ float merge[Warps][D + 2];
#pragma unroll
        for (int e = 0; e < per; e++) merge[warp][per * lane + e] = x[e];
        if (lane == 0) {
            merge[warp][D] = top;
            merge[warp][D + 1] = total;
        }
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int w = 1; w < Warps; w++) top = fmaxf(top, merge[w][D]);
        total = 0.0f;
#pragma unroll
        for (int e = 0; e < per; e++) x[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < Warps; w++) {
            const float weight = weigh(merge[w][D], merge[w][D + 1]);
            total = fmaf(weight, merge[w][D + 1], total);
#pragma unroll
            for (int e = 0; e < per; e++) x[e] = fmaf(weight, merge[w][per * lane + e], x[e]);
        }
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    T *dst = static_cast<T *>(p.out) + (size_t)row * p.out_stride + (size_t)head * D + per * lane;
#pragma unroll
    for (int e = 0; e < per; e++) dst[e] = from_float<T>(x[e] * inverse);
}

// Whether an item's record names parts of the list's warps. A warp that gave up a wait leaves its items'
// records as the workspace had them, which is no content at all.
__host__ __device__ inline bool kv4_valid_record(int first_part, int last_warp, int list_warps)
{
    return first_part >= 0 && last_warp < list_warps && last_warp >= first_part >> 1;
}

// The decode kernel's rows, [item][row of the tile], a block each, of 4 warps, or 8 where
// items have many parts (64 sequences of up to 4352 keys, decode and combine together: 42.2
// us, with 2 warps 43.4, with 1 45.0; 4 of 8000 keys: 24.0 with 8, 26.5 by one warp that
// fetched a part at a time).
template <int D, typename T, int Warps>
static __global__ void __launch_bounds__(32 * Warps) kv4_combine_kernel(Kv4AttnParams p, int tile_rows)
{
    const int at = blockIdx.x, item = at / tile_rows;
    const int r0 = item % p.tiles * tile_rows, r = r0 + at % tile_rows;
    const int kvh = item / p.tiles % p.cache.heads, s = item / p.tiles / p.cache.heads;
    pdl_wait();
    pdl_launch_dependents();
    if (s >= p.rows.sequences) return;
    int2 where = p.items[item];
    const Kv4Sequence q = kv4_sequence(p.rows, s);
    if (!q.ok || q.count * p.group > p.most || r >= q.count * p.group) return;
    const int token = r / p.group, head = kvh * p.group + r - token * p.group;
    if (q.length <= 0) {
        where = make_int2(0, -1);  // no keys: no parts
    } else if (where.x == -1) {
        return;
    } else if (!kv4_valid_record(where.x, where.y, p.list_warps)) {
        if (threadIdx.x == 0) kv4_report(p.status, kKv4Timeout);
        return;
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
