// Causal attention over the paged 4-bit KV cache for few query rows: decode
// steps over many sequences, and short runs of tokens.
//
// HBM-bound by design: a block of the cache (one page of one KV head, 9216 bytes for
// 128 dims) is copied once into shared memory, K with its scales and V with its
// scales by one bulk copy each, and serves all the query rows of its KV head. Each
// warp walks pages of its own with its own ring of half blocks, so nothing waits for
// another warp until the last merge; keys split over warps, CTAs (splits) and, in
// the combine kernel, back together in a fixed order.
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
    int group;        // query heads per KV head
    float scale2;     // scale * log2 e
    int split_pages;  // pages of a split
    int splits;       // 1: the kernel writes the output itself
    int tiles;        // row tiles of a (sequence, KV head)
    int most;         // the decode kernel's sequences have at most so many rows a KV head
    bool wide;
    // unnormalised o, m, l, D + 2 floats: [sequence][KV head][row of the tiles][split]
    // of the decode kernel, [row][query head][split] of the block kernel
    float *part;
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

#ifndef KV4_WARPS
#define KV4_WARPS 4
#define KV4_SLOTS 3
#define KV4_CTAS 4
#endif
constexpr int kDecodeWarps = KV4_WARPS, kDecodeSlots = KV4_SLOTS, kDecodeCtas = KV4_CTAS;

template <int D, typename T, int NT> struct Kv4Decode {
    static constexpr bool split = sizeof(T) == 4;    // hi and lo columns
    static constexpr int lane_rows = split ? 1 : 2;  // query rows of a lane and n tile
    static constexpr int rows = 4 * NT * lane_rows;  // query rows of a tile
    static constexpr int half = Kv4Layout<D>::block / 2;
    static constexpr int ring = kDecodeWarps * kDecodeSlots * half;
    static constexpr int merge = kDecodeWarps * rows * (D + 2) * 4;
    static constexpr int bars = (ring > merge ? ring : merge);
    static constexpr int smem = bars + kDecodeWarps * kDecodeSlots * 8 + 16;
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

// A block per (sequence, KV head, row tile, split), the split fastest.
template <int D, typename T, int NT>
static __global__ void __launch_bounds__(32 * kDecodeWarps, NT == 1 ? kDecodeCtas : 2) kv4_decode_kernel(Kv4AttnParams p)
{
    using L = Kv4Layout<D>;
    using K = Kv4Decode<D, T, NT>;
    constexpr int G = L::groups, MT = D / 16, RP = K::lane_rows, W = kDecodeWarps, SLOTS = kDecodeSlots;
    constexpr int row_bytes = D / 2;
    extern __shared__ __align__(128) uint8_t kv4_smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(kv4_smem + K::bars);
    volatile int *abort_word = reinterpret_cast<volatile int *>(bars + W * SLOTS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % p.splits, tile_of = blockIdx.x / p.splits, r0 = tile_of % p.tiles * K::rows;
    const int kvh = tile_of / p.tiles % p.cache.heads, s = tile_of / p.tiles / p.cache.heads;
    uint64_t *bar = bars + warp * SLOTS;
    if (threadIdx.x == 0) *abort_word = 0;
    if (lane < SLOTS) mbar_init(&bar[lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_wait();
    pdl_launch_dependents();
    const Kv4Sequence q = kv4_sequence(p.rows, s);
    if (!q.ok) {
        if (threadIdx.x == 0) kv4_report(p.status, kKv4BadRows);
        return;
    }
    const int n_rows = q.count * p.group;
    if (r0 >= n_rows || n_rows > p.most) return;
    const int pages = (q.length + kPage - 1) / kPage, first = split * p.split_pages;
    const int last = min(first + p.split_pages, pages);  // this split's pages [first, last)
    if (first >= last && p.splits > 1) return;           // the combine knows how many splits have pages
    __syncthreads();

    // the warp's pages are first + warp + W i; their ids, 32 at a time, one a lane
    const int *table = p.rows.page_tables + s * p.rows.table_stride;
    const int mine = last - first - warp > 0 ? (last - first - warp + W - 1) / W : 0;
    uint8_t *buffers = kv4_smem + warp * SLOTS * K::half;
    int ids = lane < mine ? table[first + warp + lane * W] : 0;
    int next_ids = 0;
    auto id_of = [&](int i) { return __shfl_sync(0xffffffffu, (i & 32) ? next_ids : ids, i & 31); };
    // half h of the walk: K (even) or V (odd) of the warp's page h / 2
    auto issue = [&](int h, int slot) {
        const uint8_t *block = kv4_block<D>(p.cache, id_of(h >> 1), kvh);
        if (lane == 0 && block) {
            mbar_expect_tx(&bar[slot], K::half);
            bulk_g2s(buffers + slot * K::half, block + (h & 1 ? K::half : 0), K::half, &bar[slot]);
        }
    };
#pragma unroll
    for (int h = 0; h < SLOTS; h++)
        if (h < 2 * mine) issue(h, h);
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
        }
    }
    const int all_see = q.length - q.count + r0 / p.group;  // every row of the tile sees keys up to here
    float m[NT][RP], l[NT][RP], o[NT][MT][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < RP; e++) {
            m[nt][e] = -INFINITY;
            l[nt][e] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < MT; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
    }
    // byte offsets of the lane's first reads in a half block; 16 keys on are 16 rows on, the swizzle the same
    const int k_at = g * row_bytes + 4 * G * t, ks_at = L::k_scale(g, 0);
    const int v_even = L::v_word(2 * t, g * (MT / 4)) - K::half, v_odd = v_even ^ row_bytes;
    const int vs_at = L::v_scale(2 * t, g * (D / 8) / 32) - K::half;
    bool ok = true;
    unsigned phases = 0;  // parity of each slot's next wait
    int slot = 0;
    auto next = [&](int h) {  // done with half h: every lane has read it; refill its slot
        __syncwarp();
        if (h + SLOTS < 2 * mine) issue(h + SLOTS, slot);
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
    };
    for (int i = 0; i < mine; i++) {
        if ((i & 31) == 0 && i + 32 < mine) {  // the other half of the ids, long before it is asked for
            const int fetched = i + 32 + lane < mine ? table[first + warp + (i + 32 + lane) * W] : 0;
            if (i & 32) ids = fetched;
            else next_ids = fetched;
        }
        if ((unsigned)id_of(i) >= (unsigned)p.cache.pages) {
            if (lane == 0) kv4_report(p.status, kKv4BadPage);
            next(2 * i);
            next(2 * i + 1);
            continue;
        }
        if (!(ok = kv4_warp_wait(&bar[slot], phases >> slot & 1, abort_word))) break;
        phases ^= 1u << slot;
        const uint8_t *block = buffers + slot * K::half;
        const int p0 = (first + warp + i * W) * kPage;
        float sc[4][NT][2][RP];
#pragma unroll
        for (int tile = 0; tile < 4; tile++) {
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
        if (p0 + kPage - 1 > all_see) {
#pragma unroll
            for (int tile = 0; tile < 4; tile++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int k8 = 0; k8 < 2; k8++)
#pragma unroll
                        for (int e = 0; e < RP; e++)
                            if (p0 + 16 * tile + 8 * k8 + g > limit[nt][e]) sc[tile][nt][k8][e] = -INFINITY;
        }
        uint32_t pb[4][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float corr[RP], base[RP];
            bool raised = false;
#pragma unroll
            for (int e = 0; e < RP; e++) {
                float mx = m[nt][e];
#pragma unroll
                for (int tile = 0; tile < 4; tile++) mx = fmaxf(mx, fmaxf(sc[tile][nt][0][e], sc[tile][nt][1][e]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                raised = raised || mx != m[nt][e];
                corr[e] = mx == m[nt][e] ? 1.0f : exp2_fast(m[nt][e] - mx);
                m[nt][e] = mx;
                // a row without any key yet: exp2(-inf - 0) = 0
                base[e] = mx == -INFINITY ? 0.0f : mx - kWeightShift;
                l[nt][e] *= corr[e];
            }
#pragma unroll
            for (int tile = 0; tile < 4; tile++)
#pragma unroll
                for (int k8 = 0; k8 < 2; k8++) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < RP; e++) {
                        w[e] = exp2_fast(sc[tile][nt][k8][e] - base[e]);
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
            if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
                for (int i2 = 0; i2 < MT; i2++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[nt][i2][e] *= corr[K::split ? 0 : e & 1];
            }
        }
        if (!(ok = kv4_warp_wait(&bar[slot], phases >> slot & 1, abort_word))) break;
        phases ^= 1u << slot;
        uint8_t *vblock = buffers + slot * K::half;
        {
            // scales behind the last position (whatever those slots hold) and NaNs become zeros
            // before the MMAs, in which a weight of zero would not keep a NaN away from a row
            // that does not see its position; the rows that do see a NaN take it here
            constexpr int own = kPage * G / 32;  // scales of a lane, [position / 2][group][position % 2]
            uint8_t *mine_at = vblock + L::v_scale(0, 0) - K::half + 2 * own * lane;
            uint32_t d[own / 2];
            if constexpr (own == 8) *reinterpret_cast<uint4 *>(d) = *reinterpret_cast<const uint4 *>(mine_at);
            else *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(mine_at);
            const int valid = q.length - p0;
            uint32_t nan = 0;
#pragma unroll
            for (int e = 0; e < own / 2; e++) nan |= __hneu2_mask(*reinterpret_cast<__half2 *>(&d[e]), *reinterpret_cast<__half2 *>(&d[e]));
            if (valid < kPage || __any_sync(0xffffffffu, nan != 0)) {
                for (int key = 0; key < min(valid, kPage); key++) {
                    const float x = __half2float(*reinterpret_cast<const __half *>(vblock + L::v_scale(key, g * (D / 8) / 32) - K::half));
                    if (x != x)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int e = 0; e < RP; e++)
                                if (p0 + key <= limit[nt][e])
#pragma unroll
                                    for (int i2 = 0; i2 < MT; i2++) o[nt][i2][e] = o[nt][i2][2 + e] = x;
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < own / 2; e++) {
                    d[e] &= ~__hneu2_mask(*reinterpret_cast<__half2 *>(&d[e]), *reinterpret_cast<__half2 *>(&d[e]));
                    const int key = (own * lane / (2 * G) + e / G) * 2;
                    if (key >= valid) d[e] = 0;
                    else if (key + 1 >= valid) d[e] &= 0xffffu;
                    reinterpret_cast<uint32_t *>(mine_at)[e] = d[e];
                }
                fence_proxy_async_smem();  // before the slot's next bulk copy
                __syncwarp();
            }
        }
#pragma unroll
        for (int tile = 0; tile < 4; tile++) {
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
    // merge the warps' parts, in warp order
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
    __syncthreads();
    constexpr int per = D / 8;  // threads of a row, 8 dims each
    for (int item = threadIdx.x; item < K::rows * per; item += 32 * W) {
        const int r = item / per, d = item % per * 8;
        if (r0 + r >= n_rows) continue;
        float top = -INFINITY, total = 0.0f, x[8] = {};
#pragma unroll
        for (int w = 0; w < W; w++) top = fmaxf(top, ml[2 * (w * K::rows + r)]);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const int at = w * K::rows + r;
            // a part without keys has l = 0; one whose scores are NaN has l = NaN and stays
            const float weight = ml[2 * at + 1] == 0.0f ? 0.0f : ml[2 * at] == top ? 1.0f : exp2_fast(ml[2 * at] - top);
            total = fmaf(weight, ml[2 * at + 1], total);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = fmaf(weight, mo[at * D + d + e], x[e]);
        }
        if (p.splits == 1) {
            const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] *= inverse;
            const int token = (r0 + r) / p.group, head = kvh * p.group + (r0 + r) - token * p.group;
            store8(static_cast<T *>(p.out) + (size_t)(q.first + token) * p.out_stride + (size_t)head * D + d, p.wide, x);
        } else {
            const size_t slot_of =
                (((size_t)s * p.cache.heads + kvh) * p.tiles * K::rows + r0 + r) * p.splits + split;
            float *part = p.part + slot_of * (D + 2);
#pragma unroll
            for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2 *>(part + d + e) = make_float2(x[e], x[e + 1]);
            if (d == 0) *reinterpret_cast<float2 *>(part + D) = make_float2(top, total);
        }
    }
}

// One warp: the parts of `splits` splits, in split order, to a row's head.
template <int D, typename T>
__device__ __forceinline__ void kv4_combine(const Kv4AttnParams &p, const float *part, int splits, int row, int head)
{
    constexpr int per = D / 32;
    const int lane = threadIdx.x & 31;
    float top = -INFINITY, total = 0.0f, x[per] = {};
    for (int i = lane; i < splits; i += 32) top = fmaxf(top, part[(size_t)i * (D + 2) + D]);
    top = warp_max(top);
    for (int i0 = 0; i0 < splits; i0 += 32) {
        float weight = 0.0f;
        if (i0 + lane < splits) {
            const float2 ml = *reinterpret_cast<const float2 *>(part + (size_t)(i0 + lane) * (D + 2) + D);
            weight = ml.y == 0.0f ? 0.0f : ml.x == top ? 1.0f : exp2_fast(ml.x - top);
            total = fmaf(weight, ml.y, total);
        }
        const int n = min(32, splits - i0);
#pragma unroll 4
        for (int i = 0; i < n; i++) {
            const float w = __shfl_sync(0xffffffffu, weight, i);
            const float *src = part + (size_t)(i0 + i) * (D + 2) + per * lane;
#pragma unroll
            for (int e = 0; e < per; e += 2) {
                const float2 v = *reinterpret_cast<const float2 *>(src + e);
                x[e] = fmaf(w, v.x, x[e]);
                x[e + 1] = fmaf(w, v.y, x[e + 1]);
            }
        }
    }
    total = warp_sum(total);
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    T *dst = static_cast<T *>(p.out) + (size_t)row * p.out_stride + (size_t)head * D + per * lane;
#pragma unroll
    for (int e = 0; e < per; e++) dst[e] = from_float<T>(x[e] * inverse);
}

// One warp per row of a (sequence, KV head) of the decode kernel's. A block of 4
// warps takes 4 rows, the rows fastest.
template <int D, typename T>
static __global__ void __launch_bounds__(128) kv4_combine_kernel(Kv4AttnParams p, int tile_rows)
{
    const int fours = (tile_rows + 3) / 4, r = blockIdx.x % fours * 4 + (threadIdx.x >> 5);
    const int kvh = blockIdx.x / fours % p.cache.heads, s = blockIdx.x / fours / p.cache.heads;
    pdl_wait();
    pdl_launch_dependents();
    const Kv4Sequence q = kv4_sequence(p.rows, s);
    if (!q.ok || q.count * p.group > p.most || r >= q.count * p.group) return;
    const int pages = (q.length + kPage - 1) / kPage, splits = (pages + p.split_pages - 1) / p.split_pages;
    const int token = r / p.group;
    kv4_combine<D, T>(p, p.part + (((size_t)s * p.cache.heads + kvh) * tile_rows + r) * p.splits * (D + 2), splits,
                      q.first + token, kvh * p.group + r - token * p.group);
}

}  // namespace lun
