// Causal attention over the paged 4-bit KV cache for blocks of query tokens, on
// the tcgen05 tensor cores.
//
// One CTA owns 128 query rows (128 / group tokens with the query heads of one KV
// head) and a page-aligned range of keys, in tiles of 64 (one page):
//   warp 0      bulk copies of a tile's K half and V half (codes and scales, 4608
//               bytes each for 128 dims) into two rings of three;
//   warp 1      allocates tensor memory; one lane issues the MMAs: S = Q K^T into
//               one of two buffers, O += P V;
//   warps 2-3   K codes -> d * (c - 8) in FP16 (exact), K-major with the 128-byte
//               swizzle, two buffers;
//   warps 4-5   V codes -> the same, transposed, two buffers; values behind the last
//               position, of a page outside the pool and of NaN scales are zeros;
//   warps 6-9   a thread per query row: Q into tensor memory once; per tile the
//               row's 64 scores from tensor memory, causal mask, online softmax,
//               weights over the scores as the A operand of P V; at the end O / l or
//               the split's part.
// FP32 rows go in as FP16 hi + lo parts (two MMAs a product, 22 bits; the cache's
// side is exact in one part), 16-bit rows as one. Weights are times 2^11, and the
// running maximum is kept until a tile raises it by more than 2^4, so a weight is at most
// 2^15 and its parts keep their bits down to 2^-25 of the largest.
//
// A code pair leaves the conversion as dims (n, n + 4) of a word, so each 8 dims lie
// in the order 0 4 1 5 2 6 3 7 in K and, to match, in Q.
//
// Tensor memory (512 columns, one CTA an SM): Q hi [0, D / 2), Q lo [64, 64 + D / 2), S and P
// buffers [128, 192) and [192, 256), O [256, 256 + D).
#pragma once
#include "kv4_attention.cuh"
#include "tcgen05.cuh"

namespace lun {

constexpr int kBlockRows = 128, kBlockThreads = 320, kBlockStages = 3;
constexpr float kBlockShift = 11.0f, kBlockRaise = 4.0f;

template <int D> struct Kv4BlockLayout {
    static constexpr int half = Kv4Layout<D>::block / 2;
    static constexpr int tile = kPage * D * 2;                 // FP16 K tile, or V^T tile
    static constexpr int k_tiles = 0, v_tiles = 2 * tile;      // two buffers each, 1024-byte aligned
    static constexpr int k_ring = 4 * tile, v_ring = k_ring + kBlockStages * half;
    static constexpr int bars = v_ring + kBlockStages * half;  // multiple of 8
    // more than half of an SM's shared memory: a second CTA would wait for tensor memory
    static constexpr int smem = 1024 + bars + 512 > 118 * 1024 ? 1024 + bars + 512 : 118 * 1024;
};

// The row tile `index` of the sequences that the block kernel takes (more than
// `least` query rows a KV head): its sequence and its place there. A warp asks together.
__device__ __forceinline__ bool kv4_block_tile(const Kv4Rows &r, int group, int least, int index, int &s, int &place)
{
    const int lane = threadIdx.x & 31, tokens = kBlockRows / group;
    int before = 0;
    for (int s0 = 0; s0 < r.sequences; s0 += 32) {
        int tiles = 0;
        if (s0 + lane < r.sequences) {
            const Kv4Sequence q = kv4_sequence(r, s0 + lane);
            if (q.ok && q.count * group > least) tiles = (q.count + tokens - 1) / tokens;
        }
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        const unsigned here = __ballot_sync(0xffffffffu, index < before + upto);
        if (here) {
            const int who = __ffs(here) - 1;
            s = s0 + who;
            place = index - before - __shfl_sync(0xffffffffu, upto - tiles, who);
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// A CTA per (row tile, KV head, split), the row tile slowest. p.tiles bounds the row tiles.
template <int D, typename T>
static __global__ void __launch_bounds__(kBlockThreads, 1) kv4_block_kernel(Kv4AttnParams p, int least)
{
    using L = Kv4Layout<D>;
    using B = Kv4BlockLayout<D>;
    constexpr int G = L::groups, parts = sizeof(T) == 4 ? 2 : 1;
    constexpr uint32_t q_col = 0, s_col = 128, o_col = 256;
    extern __shared__ __align__(1024) uint8_t kv4_block_raw[];
    const uint32_t raw = smem_u32(kv4_block_raw);
    uint8_t *base = kv4_block_raw + (((raw + 1023u) & ~1023u) - raw);
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + B::bars);
    uint64_t *k_full = bars, *k_empty = bars + 3, *v_full = bars + 6, *v_empty = bars + 9;       // raw rings
    uint64_t *k_ready = bars + 12, *k_free = bars + 14, *v_ready = bars + 16, *v_free = bars + 18;  // FP16 tiles
    uint64_t *s_full = bars + 20, *p_ready = bars + 22, *o_done = bars + 24, *q_ready = bars + 25;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 26);
    volatile int *abort_word = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *where = reinterpret_cast<int *>(tmem_slot + 2);    // sequence, place
    int *poison = where + 2;                                // per group of dims: first position with a NaN value
    volatile int *bad = poison + 4;                         // of tile j % 16: its page lies outside the pool
    int *error = &kv4_error_sink;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.splits, kvh = blockIdx.x / p.splits % p.cache.heads;
    const int index = blockIdx.x / p.splits / p.cache.heads;

    pdl_wait();
    pdl_launch_dependents();
    if (warp == 0) {
        int s = -1, place = 0;
        if (!kv4_block_tile(p.rows, p.group, least, index, s, place)) s = -1;
        if (lane == 0) where[0] = s, where[1] = place;
    }
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.rows.sequences; i += kBlockThreads)
            if (!kv4_sequence(p.rows, i).ok) kv4_report(p.status, kKv4BadRows);
    __syncthreads();
    const int s = where[0];
    if (s < 0) return;
    const Kv4Sequence q = kv4_sequence(p.rows, s);
    const int tokens = kBlockRows / p.group, t0 = where[1] * tokens, first_position = q.length - q.count;
    const int k0 = split * p.split_pages * kPage;
    const int seen = min(first_position + min(t0 + tokens, q.count), k0 + p.split_pages * kPage);  // keys [k0, seen)
    const int tiles = seen > k0 ? (seen - k0 + kPage - 1) / kPage : 0;
    if (tiles == 0 && p.splits > 1) return;  // the combine knows which splits have keys

    if (threadIdx.x == 0) {
        for (int i = 0; i < 3; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 2);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 2);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_ready[i], 2);
            mbar_init(&k_free[i], 1);
            mbar_init(&v_ready[i], 2);
            mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], 4);
        }
        mbar_init(o_done, 1);
        mbar_init(q_ready, 4);
        *abort_word = 0;
        for (int i = 0; i < 4; i++) poison[i] = 0x7fffffff;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ---- loads: each ring's next slot as soon as its converters released it
        if (lane == 0) {
            const int *table = p.rows.page_tables + s * p.rows.table_stride + k0 / kPage;
            int ik = 0, iv = 0;
            unsigned idle = 0;
            const unsigned long long start = wait_clock_ns();
            unsigned long long last = start;
            while ((ik < tiles || iv < tiles) && !*abort_word) {
                bool progressed = false;
                if (ik < tiles && (ik < 3 || mbar_test_wait(&k_empty[ik % 3], (ik / 3 - 1) & 1))) {
                    const uint8_t *block = kv4_block<D>(p.cache, table[ik], kvh);
                    bad[ik & 15] = !block;
                    if (block) {
                        mbar_expect_tx(&k_full[ik % 3], B::half);
                        bulk_g2s(base + B::k_ring + ik % 3 * B::half, block, B::half, &k_full[ik % 3]);
                    } else {
                        kv4_report(p.status, kKv4BadPage);
                        mbar_arrive(&k_full[ik % 3]);
                    }
                    ik++;
                    progressed = true;
                }
                if (iv < ik && (iv < 3 || mbar_test_wait(&v_empty[iv % 3], (iv / 3 - 1) & 1))) {
                    const uint8_t *block = kv4_block<D>(p.cache, table[iv], kvh);
                    if (block) {
                        mbar_expect_tx(&v_full[iv % 3], B::half);
                        bulk_g2s(base + B::v_ring + iv % 3 * B::half, block + B::half, B::half, &v_full[iv % 3]);
                    } else {
                        mbar_arrive(&v_full[iv % 3]);
                    }
                    iv++;
                    progressed = true;
                }
                if (progressed) {
                    idle = 0;
                    last = wait_clock_ns();
                } else if ((++idle & 1023u) == 0 && wait_clock_ns() - last > kWaitLimitNs) {
                    *abort_word = 1;
                    atomicExch(error, 1);
                    break;
                }
            }
            // every copy issued has landed before the CTA ends
            for (int j = max(0, ik - 3); j < ik; j++)
                mbar_wait_bounded(&k_full[j % 3], (j / 3) & 1, abort_word, error, kWaitSpinLimit);
            for (int j = max(0, iv - 3); j < iv; j++)
                mbar_wait_bounded(&v_full[j % 3], (j / 3) & 1, abort_word, error, kWaitSpinLimit);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issue: S(j) as soon as K(j) is converted, then P V of tile j - 1
        if (lane == 0 && tiles > 0) {
            const uint32_t idesc_s = f16_idesc(128, kPage), idesc_o = f16_idesc(128, D);
            const uint32_t kt = smem_u32(base + B::k_tiles), vt = smem_u32(base + B::v_tiles);
            bool ok = mbar_wait_bounded(q_ready, 0, abort_word, error, kWaitSpinLimit);
            for (int j = 0; ok && j <= tiles; j++) {
                if (j < tiles) {
                    const int b = j & 1;
                    if (!(ok = mbar_wait_bounded(&k_ready[b], (j >> 1) & 1, abort_word, error, kWaitSpinLimit))) break;
                    tc_fence_after();
                    const uint32_t sd = tmem + s_col + 64u * (uint32_t)b, k = kt + (uint32_t)b * B::tile;
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
                        for (int part = 0; part < parts; part++)
                            tc_mma_f16_tmem_a(sd, tmem + q_col + 64u * part + 8u * ks,
                                              sw128_desc(k + (ks >> 2) * 8192 + (ks & 3) * 32), idesc_s, (ks | part) != 0);
                    tc_commit(&k_free[b]);
                    tc_commit(&s_full[b]);
                }
                if (j >= 1) {
                    const int i = j - 1, b = i & 1;
                    if (!(ok = mbar_wait_bounded(&p_ready[b], (i >> 1) & 1, abort_word, error, kWaitSpinLimit) &&
                               mbar_wait_bounded(&v_ready[b], (i >> 1) & 1, abort_word, error, kWaitSpinLimit)))
                        break;
                    tc_fence_after();
                    const uint32_t pa = tmem + s_col + 64u * (uint32_t)b, v = vt + (uint32_t)b * B::tile;
#pragma unroll
                    for (int ks = 0; ks < kPage / 16; ks++)
#pragma unroll
                        for (int part = 0; part < parts; part++)
                            tc_mma_f16_tmem_a(tmem + o_col, pa + 32u * part + 8u * ks, sw128_desc(v + ks * 32), idesc_o,
                                              (i | ks | part) != 0);
                    tc_commit(&v_free[b]);
                    tc_commit(o_done);
                }
            }
        }
        __syncwarp();
    } else if (warp < 4) {
        // ---- K: a unit is 16 (8 for 64 dims) bytes of a key's row, word j of them is word 4 j + t of the
        // row; keys k and k + 4 share a quarter warp, whose stores then hit every bank once
        const int ct = threadIdx.x - 64;  // 0..63
        for (int j = 0; j < tiles; j++) {
            if (!warp_wait(&k_full[j % 3], (j / 3) & 1, abort_word, error)) break;
            if (j >= 2 && !warp_wait(&k_free[j & 1], ((j >> 1) - 1) & 1, abort_word, error)) break;
            const uint8_t *src = base + B::k_ring + j % 3 * B::half;
            uint8_t *dst = base + B::k_tiles + (j & 1) * B::tile;
            if (!bad[j & 15]) {
#pragma unroll
                for (int it = 0; it < 4; it++) {
                    const int u = ct + 64 * it, t = u & 3, key = (u >> 5) * 8 + ((u >> 2) & 1) * 4 + ((u >> 3) & 3);
                    uint32_t w[G], d[G / 2];
                    if constexpr (G == 4) {
                        *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(src + key * (D / 2) + 16 * t);
                        *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(src + L::k_scale(key, 0));
                    } else {
                        *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(src + key * (D / 2) + 8 * t);
                        d[0] = *reinterpret_cast<const uint32_t *>(src + L::k_scale(key, 0));
                    }
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        const uint32_t d2 = __byte_perm(d[g >> 1], 0, g & 1 ? 0x3232 : 0x1010);
                        uint4 v;
                        v.x = kv4_times(kv4_low(w[g]), d2);
                        v.y = kv4_times(kv4_high(w[g]), d2);
                        v.z = kv4_times(kv4_low(w[g] >> 8), d2);
                        v.w = kv4_times(kv4_high(w[g] >> 8), d2);
                        const int at = 4 * g + t;  // word of the row
                        *reinterpret_cast<uint4 *>(dst + (at >> 3) * 8192 + sw128_offset(key, (at & 7) * 8)) = v;
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&k_ready[j & 1]);
                mbar_arrive(&k_empty[j % 3]);
            }
        }
    } else if (warp < 6) {
        // ---- V: a unit is word w of 8 keys, stored as 8 dims x 8 keys; lanes start at different
        // dims, so that a quarter warp's stores hit every bank once
        const int ct = threadIdx.x - 128;  // 0..63
        for (int j = 0; j < tiles; j++) {
            if (!warp_wait(&v_full[j % 3], (j / 3) & 1, abort_word, error)) break;
            if (j >= 2 && !warp_wait(&v_free[j & 1], ((j >> 1) - 1) & 1, abort_word, error)) break;
            const uint8_t *src = base + B::v_ring + j % 3 * B::half - B::half;  // v_word and v_scale count from the block
            uint8_t *dst = base + B::v_tiles + (j & 1) * B::tile;
            const int p0 = k0 + j * kPage, valid = bad[j & 15] ? 0 : seen - p0;
#pragma unroll 1
            for (int u = ct; u < L::words * 8; u += 64) {
                const int w = u % L::words, kg = u / L::words, group = w / 4;
                uint32_t v[8], d2[4];
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = *reinterpret_cast<const uint32_t *>(src + L::v_word(8 * kg + i, w));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int key = 8 * kg + 2 * i;
                    d2[i] = *reinterpret_cast<const uint32_t *>(src + L::v_scale(key, group));
                    if (key >= valid) d2[i] = 0;
                    else if (key + 1 >= valid) d2[i] &= 0xffffu;
                    // a NaN times a masked row's weight of zero must not reach that row: the rows that
                    // see the position take it at the end
                    const uint32_t nan = __hneu2_mask(*reinterpret_cast<__half2 *>(&d2[i]), *reinterpret_cast<__half2 *>(&d2[i]));
                    if (nan) atomicMin(&poison[group], p0 + key + !(nan & 0xffffu));
                    d2[i] &= ~nan;
                }
                uint32_t lo[4], hi[4];  // nibbles 0..3 and 4..7 of key pairs
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    lo[i] = __byte_perm(v[2 * i], v[2 * i + 1], 0x5410);
                    hi[i] = __byte_perm(v[2 * i], v[2 * i + 1], 0x7632);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int e = (i + w) & 7, shift = 4 * (e & 3);
                    uint4 x;
                    x.x = kv4_times(kv4_low((e & 4 ? hi[0] : lo[0]) >> shift), d2[0]);
                    x.y = kv4_times(kv4_low((e & 4 ? hi[1] : lo[1]) >> shift), d2[1]);
                    x.z = kv4_times(kv4_low((e & 4 ? hi[2] : lo[2]) >> shift), d2[2]);
                    x.w = kv4_times(kv4_low((e & 4 ? hi[3] : lo[3]) >> shift), d2[3]);
                    *reinterpret_cast<uint4 *>(dst + sw128_offset(8 * w + e, 8 * kg)) = x;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&v_ready[j & 1]);
                mbar_arrive(&v_empty[j % 3]);
            }
        }
        asm volatile("bar.sync 1, 192;" ::: "memory");  // poison[] is complete
    } else {
        // ---- softmax: a thread is a query row
        const int row = 32 * (warp & 3) + lane, token = row / p.group, head = kvh * p.group + row - token * p.group;
        const bool live = token < tokens && t0 + token < q.count;
        const int limit = live ? first_position + t0 + token : -1;  // last key position this row sees
        const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const size_t tensor_row = (size_t)(q.first + t0 + (live ? token : 0));
        float back;
        {
            const T *src = static_cast<const T *>(p.q) + tensor_row * p.q_stride + (size_t)(live ? head : 0) * D;
            float top = 0.0f;
#pragma unroll 4
            for (int d = 0; d < D; d += 8) {
                float x[8];
                load8(src + d, p.wide, x);
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
            }
            float undo;
            const float f = live ? power_scale(top, undo) : 0.0f;
            if (!live) undo = 0.0f;
            back = undo * p.scale2;
#pragma unroll
            for (int d0 = 0; d0 < D; d0 += 64) {
                uint32_t hi[32], lo[32];
#pragma unroll
                for (int w = 0; w < 8; w++) {
                    float x[8];
                    load8(src + d0 + 8 * w, p.wide, x);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float a = live ? x[e] * f : 0.0f, b = live ? x[e + 4] * f : 0.0f;
                        split_half2(a, b, hi[4 * w + e], lo[4 * w + e]);
                    }
                }
                tmem_st32(lane_base + q_col + d0 / 2, hi);
                if (parts == 2) tmem_st32(lane_base + q_col + 64u + d0 / 2, lo);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
        }
        const int all_see = first_position + t0;  // every live row sees keys up to here
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < tiles; j++) {
            if (!(ok = warp_wait(&s_full[j & 1], (j >> 1) & 1, abort_word, error))) break;
            tc_fence_after();
            const uint32_t sb = s_col + 64u * (uint32_t)(j & 1);
            uint32_t raw_s[64];
            tmem_ld32(lane_base + sb, *reinterpret_cast<uint32_t(*)[32]>(&raw_s[0]));
            tmem_ld32(lane_base + sb + 32u, *reinterpret_cast<uint32_t(*)[32]>(&raw_s[32]));
            const int p0 = k0 + j * kPage;
            float x[64], mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 64; c++) x[c] = __uint_as_float(raw_s[c]) * back;
            if (bad[j & 15] || p0 + kPage - 1 > all_see) {
                const int last = bad[j & 15] ? -1 : limit;
#pragma unroll
                for (int c = 0; c < 64; c++) x[c] = p0 + c <= last ? x[c] : -INFINITY;
            }
#pragma unroll
            for (int c = 0; c < 64; c++) mx = fmaxf(mx, x[c]);
            // a row without any key yet has O = 0 and l = 0 and just takes the tile's maximum
            const bool raise = m != -INFINITY && mx > m + kBlockRaise;
            const float corr = raise ? exp2_fast(m - mx) : 1.0f;
            if (m == -INFINITY || raise) m = mx;
            if (__any_sync(0xffffffffu, raise)) {
                // O's row *= corr once P V of the tile before has landed
                if (!(ok = warp_wait(o_done, (j - 1) & 1, abort_word, error))) break;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(lane_base + o_col + c, o);
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                    tmem_st32(lane_base + o_col + c, o);
                }
            }
            l *= corr;
            const float zero = m == -INFINITY ? 0.0f : m - kBlockShift;
            float sum0 = 0.0f, sum1 = 0.0f;
            uint32_t ph[32], pl[32];
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const float a = exp2_fast(x[2 * i] - zero), b = exp2_fast(x[2 * i + 1] - zero);
                sum0 += a;
                sum1 += b;
                if (parts == 2) {
                    split_half2(a, b, ph[i], pl[i]);
                } else {
                    const __half2 h = __floats2half2_rn(a, b);
                    ph[i] = *reinterpret_cast<const uint32_t *>(&h);
                }
            }
            l += sum0 + sum1;
            tmem_st32(lane_base + sb, ph);
            if (parts == 2) tmem_st32(lane_base + sb + 32u, pl);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[j & 1]);
        }
        if (ok && tiles > 0) ok = warp_wait(o_done, (tiles - 1) & 1, abort_word, error);
        asm volatile("bar.sync 1, 192;" ::: "memory");
        if (__all_sync(0xffffffffu, ok && !*abort_word)) {
            tc_fence_after();
            const bool whole = p.splits == 1;
            const float inverse = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
            T *out = static_cast<T *>(p.out) + tensor_row * p.out_stride + (size_t)(live ? head : 0) * D;
            const int query_heads = p.cache.heads * p.group;
            float *part = p.part + ((tensor_row * query_heads + (live ? head : 0)) * p.splits + split) * (D + 2);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {  // the loads are warp-wide: every lane runs them
                uint32_t o[32];
                if (tiles > 0) {
                    tmem_ld32(lane_base + o_col + c, o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = 0u;
                }
                if (!live) continue;
                const bool nan = limit >= poison[c / kKv4Group];
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        x[e] = nan ? __uint_as_float(0x7fc00000u) : __uint_as_float(o[i + e]) * inverse;
                    if (whole) {
                        store8(out + c + i, p.wide, x);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e += 2)
                            *reinterpret_cast<float2 *>(part + c + i + e) = make_float2(x[e], x[e + 1]);
                    }
                }
            }
            if (!whole && live) *reinterpret_cast<float2 *>(part + D) = make_float2(m, l);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_word && threadIdx.x == 0) kv4_report(p.status, kKv4Timeout);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// One warp per (row, query head) of the block kernel's sequences: the splits' parts
// in split order. A block of 4 warps takes 4 heads of a row, the heads fastest.
template <int D, typename T>
static __global__ void __launch_bounds__(128) kv4_block_combine_kernel(Kv4AttnParams p, int least)
{
    const int heads = p.cache.heads * p.group, fours = (heads + 3) / 4;
    const int row = blockIdx.x / fours, head = blockIdx.x % fours * 4 + (threadIdx.x >> 5);
    pdl_wait();
    pdl_launch_dependents();
    const Kv4Sequence q = kv4_sequence(p.rows, kv4_sequence_of_row(p.rows, row));
    if (!q.ok || row < q.first || row >= q.first + q.count || q.count * p.group <= least || head >= heads) return;
    const int keys = q.length - q.count + (row - q.first) + 1, width = p.split_pages * kPage;
    const int splits = keys > 0 ? (keys + width - 1) / width : 0;
    kv4_combine<D, T>(p, p.part + ((size_t)row * heads + head) * p.splits * (D + 2), splits, row, head);
}

}  // namespace lun
