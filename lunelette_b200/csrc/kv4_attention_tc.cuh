// Causal attention over the paged 4-bit KV cache for blocks of query tokens, on
// the tcgen05 tensor cores.
//
// One CTA owns 128 query rows (128 / group tokens with the query heads of one KV
// head) and a page-aligned range of keys, in tiles of 64 (one page):
//   warp 0      bulk copies of a tile's K half and V half (codes and scales, 4608
//               bytes each for 128 dims) into two rings of six, which covers HBM's latency;
//   warp 1      allocates tensor memory; one lane issues the MMAs: S = Q K^T for two
//               tiles at once into one of two buffers (with 64 keys an MMA takes as
//               long as with 128: it waits for Q from tensor memory), O += P V a tile;
//   warps 2-5   K codes -> d * (c - 8) in FP16 (exact), [key][dim] with the 128-byte
//               swizzle, two buffers;
//   warps 6-9   V codes -> the same (P V takes them as an N-major operand, so nothing is
//               transposed); values behind the last position, of a page outside the
//               pool and of NaN scales are zeros;
//   warps 10-13 a thread per query row: Q into tensor memory once; per tile the
//               row's 64 scores from tensor memory, causal mask, online softmax,
//               weights over the scores as the A operand of P V; at the end O / l or
//               the split's part.
// FP32 rows of q go in as FP16 hi + lo parts (two MMAs a product, 22 bits; the cache's
// side is exact in one part), 16-bit rows as one, and the weights of either in two. Weights are times 2^7, and the
// running maximum is kept until a tile raises it by more than 2^8 (a raise waits for
// P V and rescales O, up to 2000 cycles; with 2^4 half the tiles had one), so a weight is at
// most 2^15, and its parts end at 2^-32 of the largest.
// The tensor core cuts what it adds up towards zero, over values of one sign about 1.7e-7 of the sum
// so far each time. So the softmax takes O out every 4 tiles, 32 products (16-bit rows: every 8,
// their own rounding is far larger), and sums those in shared memory, rounded to nearest, after the
// tile's weights, when P V of the tile before has mostly landed: 2.7e-6 over 500 or 2048 tiles of one
// sign, 0.9e-6 around zero. l is summed up with what its additions round off: 2048 tiles that
// repeat a few sums lost 5e-6 without.
//
// 256 FP32 tokens at 4352 keys, 8 KV heads of 4 query heads, with the combine: 55 us, 320 TFLOP/s
// of the definition's products and twice that issued; 34 tiles in 75000 cycles of a CTA, the tensor
// cores busy for 39 % of them: bound by the softmax warps' arithmetic between two products, on 128 of
// 148 SMs. 256 BF16 tokens take 51 us.
//
// A code pair leaves the conversion as dims (n, n + 4) of a word, so each 8 dims lie
// in the order 0 4 1 5 2 6 3 7 in K and V and, to match, in Q and O.
//
// Tensor memory (512 columns, one CTA an SM): Q hi [0, D / 2), Q lo [64, 64 + D / 2), S and P
// buffers of two tiles [128, 256) and [256, 384), O [384, 384 + D).
#pragma once
#include "kv4_attention.cuh"
#include "tcgen05.cuh"

namespace lun {

constexpr int kBlockRows = 128, kBlockThreads = 448, kBlockStages = 6;
constexpr float kBlockShift = 7.0f, kBlockRaise = 8.0f;

template <int D> struct Kv4BlockLayout {
    static constexpr int half = Kv4Layout<D>::block / 2;
    static constexpr int drain(int parts) { return parts == 2 ? 4 : 8; }  // tiles that O sums up on the tensor cores
    static constexpr int tile = kPage * D * 2;                 // 64 keys of K, or of V, in FP16
    static constexpr int k_tiles = 0, v_tiles = 4 * tile;      // two buffers of two tiles, and of one
    static constexpr int k_ring = 6 * tile, v_ring = k_ring + kBlockStages * half;
    static constexpr int q_stride = D * 4 + 16;  // bytes of a staged row of q, padded against bank conflicts
    static constexpr int q_rows = v_ring + kBlockStages * half;
    static constexpr int bars = q_rows + kBlockRows * q_stride;  // multiple of 8
    // more than half of an SM's shared memory: a second CTA would wait for tensor memory
    static constexpr int smem = 1024 + bars + 512 > 118 * 1024 ? 1024 + bars + 512 : 118 * 1024;
};

// Shared-memory descriptor of an N-major operand with the 128-byte swizzle: rows of
// 64 elements of N, 8 of them (K) an atom of 1024 bytes, atoms of K 1024 bytes apart
// (stride byte offset), the next 64 elements of N 8192 bytes on (leading byte offset).
__device__ __forceinline__ uint64_t sw128_desc_n(uint32_t saddr)
{
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
constexpr uint32_t kIdescNMajorB = 1u << 16;
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Whole warp: 8 consecutive 32-bit columns of this warp's 32 TMEM lanes; tmem_st_wait
// once for all.
__device__ __forceinline__ void tmem_st8_async(uint32_t taddr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Two FP32 operations in one instruction, on register pairs.
__device__ __forceinline__ uint64_t pack2(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t p, float &a, float &b)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

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
    constexpr uint32_t q_col = 0, s_col = 128, o_col = 384;
    extern __shared__ __align__(1024) uint8_t kv4_block_raw[];
    const uint32_t raw = smem_u32(kv4_block_raw);
    uint8_t *base = kv4_block_raw + (((raw + 1023u) & ~1023u) - raw);
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + B::bars);
    constexpr int N = kBlockStages;
    uint64_t *k_full = bars, *k_empty = bars + N, *v_full = bars + 2 * N, *v_empty = bars + 3 * N;  // raw rings
    uint64_t *tiles_at = bars + 4 * N;
    uint64_t *k_ready = tiles_at, *k_free = tiles_at + 2, *v_ready = tiles_at + 4, *v_free = tiles_at + 6;  // FP16 tiles
    uint64_t *s_full = tiles_at + 8, *p_ready = tiles_at + 10, *o_done = tiles_at + 12, *q_ready = tiles_at + 14;
    uint64_t *q_full = tiles_at + 15;  // rows of q staged, a barrier a warp
    uint64_t *products_done = tiles_at + 19;  // all of them
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tiles_at + 20);
    volatile int *abort_word = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *where = reinterpret_cast<int *>(tmem_slot + 2);    // sequence, place
    int *poison = where + 2;                                // per group of dims: first position with a NaN value
    volatile int *bad = poison + 4;                         // of tile j % 16: its page lies outside the pool
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
        for (int i = 0; i < N; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 4);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 4);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_ready[i], 4);
            mbar_init(&k_free[i], 1);
            mbar_init(&v_ready[i], 4);
            mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(q_ready, 4);
        for (int i = 0; i < 4; i++) mbar_init(&q_full[i], 1);
        mbar_init(products_done, 1);
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
        // ---- loads: each ring's next slot as soon as its converters released it. The warp holds
        // the ids of 64 tiles, so that no copy waits for the page table
        const int *table = p.rows.page_tables + s * p.rows.table_stride + k0 / kPage;
        int ids = lane < tiles ? table[lane] : 0, more = lane + 32 < tiles ? table[lane + 32] : 0;
        int ik = 0, iv = 0;
        unsigned idle = 0;
        unsigned long long last = wait_clock_ns();
        // one half of tile i into slot i % N of a ring
        auto issue = [&](int i, int offset, uint8_t *ring, uint64_t *full) {
            const int id = __shfl_sync(0xffffffffu, i & 32 ? more : ids, i & 31);
            if (lane) return;
            const uint8_t *block = kv4_block<D>(p.cache, id, kvh);
            bad[i & 15] = !block;
            if (block) {
                mbar_expect_tx(&full[i % N], B::half);
                bulk_g2s(ring + i % N * B::half, block + offset, B::half, &full[i % N]);
            } else {
                kv4_report(p.status, kKv4BadPage);
                mbar_arrive(&full[i % N]);
            }
        };
        auto released = [&](int i, uint64_t *empty) {
            return i < N || __any_sync(0xffffffffu, mbar_test_wait(&empty[i % N], (i / N - 1) & 1));
        };
        while (iv < tiles && !__any_sync(0xffffffffu, *abort_word)) {
            bool progressed = false;
            if (ik < tiles && released(ik, k_empty)) {
                issue(ik, 0, base + B::k_ring, k_full);
                ik++;
                progressed = true;
            }
            if (iv < ik && released(iv, v_empty)) {
                issue(iv, B::half, base + B::v_ring, v_full);
                iv++;
                progressed = true;
                if ((iv & 31) == 0 && iv + 32 < tiles) {  // 32 ids are used up: K is at most a few tiles ahead
                    const int fetched = iv + 32 + lane < tiles ? table[iv + 32 + lane] : 0;
                    if (iv & 32) ids = fetched;
                    else more = fetched;
                }
            }
            if (progressed) {
                idle = 0;
                last = wait_clock_ns();
            } else if ((++idle & 1023u) == 0 && __any_sync(0xffffffffu, wait_clock_ns() - last > kWaitLimitNs)) {
                *abort_word = 1;
                break;
            }
        }
        // every copy issued has landed before the CTA ends
        if (lane == 0) {
            for (int j = max(0, ik - N); j < ik; j++)
                if (!kv4_wait(&k_full[j % N], (j / N) & 1, abort_word)) kv4_landed(&k_full[j % N], (j / N) & 1);
            for (int j = max(0, iv - N); j < iv; j++)
                if (!kv4_wait(&v_full[j % N], (j / N) & 1, abort_word)) kv4_landed(&v_full[j % N], (j / N) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issue: S of the next two tiles ahead of P V of these. The warp runs
        // the loop together and one lane issues, so that descriptors stay in uniform registers
        const uint32_t idesc_o = f16_idesc(128, D) | kIdescNMajorB;
        const uint64_t k_desc = sw128_desc(smem_u32(base + B::k_tiles));
        const uint64_t v_desc = sw128_desc_n(smem_u32(base + B::v_tiles));
        const bool leader = elect_one();
        const int pairs = (tiles + 1) / 2;
        bool ok = tiles > 0 && kv4_warp_wait(q_ready, 0, abort_word);
        auto scores = [&](int i) {  // S of tiles 2 i and 2 i + 1
            const int b = i & 1;
            if (!kv4_warp_wait(&k_ready[b], (i >> 1) & 1, abort_word)) return false;
            tc_fence_after();
            if (leader) {
                const uint32_t idesc = 2 * i + 1 < tiles ? f16_idesc(128, 2 * kPage) : f16_idesc(128, kPage);
                const uint32_t sd = tmem + s_col + 128u * (uint32_t)b;
                const uint64_t k = k_desc + (uint32_t)b * (2 * B::tile >> 4);
#pragma unroll
                for (int part = parts - 1; part >= 0; part--)  // the small sums first
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++)
                        tc_mma_f16_tmem_a(sd, tmem + q_col + 64u * part + 8u * ks,
                                          k + (((ks >> 2) * 16384 + (ks & 3) * 32) >> 4), idesc,
                                          ks != 0 || part != parts - 1);
                tc_commit(&k_free[b]);
                tc_commit(&s_full[b]);
            }
            __syncwarp();
            return true;
        };
        ok = ok && scores(0);
        for (int j = 0; ok && j < tiles; j++) {
            if ((j & 1) == 0 && j / 2 + 1 < pairs && !(ok = scores(j / 2 + 1))) break;
            const int b = j & 1;
            if (!(ok = kv4_warp_wait(&p_ready[b], (j >> 1) & 1, abort_word) &&
                       kv4_warp_wait(&v_ready[b], (j >> 1) & 1, abort_word)))
                break;
            tc_fence_after();
            if (leader) {
                const uint32_t pa = tmem + s_col + 128u * (uint32_t)(j >> 1 & 1) + 64u * (uint32_t)b;
                const uint64_t v = v_desc + (uint32_t)b * (B::tile >> 4);
#pragma unroll
                for (int ks = 0; ks < kPage / 16; ks++)
#pragma unroll
                    for (int part = 0; part < 2; part++)
                        tc_mma_f16_tmem_a(tmem + o_col, pa + 32u * part + 8u * ks, v + (ks * 2048 >> 4), idesc_o,
                                          ks || part || j % B::drain(parts) != 0);
                tc_commit(&v_free[b]);
                tc_commit(&o_done[b]);
            }
            __syncwarp();
        }
        // every product issued has ended before tensor memory and the tiles go
        if (leader) tc_commit(products_done);
        __syncwarp();
        if (!kv4_warp_wait(products_done, 0, abort_word)) kv4_landed(products_done, 0);
    } else if (warp < 6) {
        // ---- K: a unit is 16 (8 for 64 dims) bytes of a key's row, word j of them is word 4 j + t of the
        // row; keys k and k + 4 share a quarter warp, whose stores then hit every bank once
        const int ct = threadIdx.x - 64;  // 0..127
        for (int j = 0; j < tiles; j++) {
            const int pair = j >> 1, b = pair & 1;
            if (!kv4_warp_wait(&k_full[j % N], (j / N) & 1, abort_word)) break;
            if ((j & 1) == 0 && pair >= 2 && !kv4_warp_wait(&k_free[b], ((pair >> 1) - 1) & 1, abort_word)) break;
            const uint8_t *src = base + B::k_ring + j % N * B::half;
            uint8_t *dst = base + B::k_tiles + b * 2 * B::tile;
            if (!bad[j & 15]) {
#pragma unroll
                for (int it = 0; it < 2; it++) {
                    const int u = ct + 128 * it, t = u & 3, key = (u >> 5) * 8 + ((u >> 2) & 1) * 4 + ((u >> 3) & 3);
                    uint32_t w[G], d[G / 2];
                    if constexpr (G == 4) {
                        *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(src + key * (D / 2) + 16 * t);
                        *reinterpret_cast<uint2 *>(d) = *reinterpret_cast<const uint2 *>(src + L::k_scale(key, 0));
                    } else {
                        *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(src + key * (D / 2) + 8 * t);
                        d[0] = *reinterpret_cast<const uint32_t *>(src + L::k_scale(key, 0));
                    }
                    const int row = 64 * (j & 1) + key;
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        const uint32_t d2 = __byte_perm(d[g >> 1], 0, g & 1 ? 0x3232 : 0x1010);
                        uint4 v;
                        v.x = kv4_times(kv4_low(w[g]), d2);
                        v.y = kv4_times(kv4_high(w[g]), d2);
                        v.z = kv4_times(kv4_low(w[g] >> 8), d2);
                        v.w = kv4_times(kv4_high(w[g] >> 8), d2);
                        const int at = 4 * g + t;  // word of the row
                        *reinterpret_cast<uint4 *>(dst + (at >> 3) * 16384 + sw128_offset(row, (at & 7) * 8)) = v;
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&k_empty[j % N]);
                if ((j & 1) || j == tiles - 1) mbar_arrive(&k_ready[b]);
            }
        }
    } else if (warp < 10) {
        // ---- V: a unit is the 4 words of a group of dims of one key; a quarter warp takes 8 keys, whose
        // stores then hit every bank once
        const int ct = threadIdx.x - 192;  // 0..127
        for (int j = 0; j < tiles; j++) {
            if (!kv4_warp_wait(&v_full[j % N], (j / N) & 1, abort_word)) break;
            if (j >= 2 && !kv4_warp_wait(&v_free[j & 1], ((j >> 1) - 1) & 1, abort_word)) break;
            const uint8_t *src = base + B::v_ring + j % N * B::half - B::half;  // v_word and v_scale count from the block
            uint8_t *dst = base + B::v_tiles + (j & 1) * B::tile;
            const int p0 = k0 + j * kPage, valid = bad[j & 15] ? 0 : seen - p0;
#pragma unroll
            for (int it = 0; it < G / 2; it++) {
                const int u = ct + 128 * it, key = u & 63, g = u >> 6;
                const uint4 w4 = *reinterpret_cast<const uint4 *>(src + L::v_word(key, 4 * g));
                const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
                uint32_t d = *reinterpret_cast<const uint16_t *>(src + L::v_scale(key, g));
                if (key >= valid) d = 0;
                if ((d & 0x7fffu) > 0x7c00u) {
                    // a NaN times a masked row's weight of zero must not reach that row: the rows that
                    // see the position take it at the end
                    atomicMin(&poison[g], p0 + key);
                    d = 0;
                }
                const uint32_t d2 = d * 0x10001u;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint4 v;
                    v.x = kv4_times(kv4_low(w[i]), d2);
                    v.y = kv4_times(kv4_high(w[i]), d2);
                    v.z = kv4_times(kv4_low(w[i] >> 8), d2);
                    v.w = kv4_times(kv4_high(w[i] >> 8), d2);
                    const int at = 4 * g + i;
                    *reinterpret_cast<uint4 *>(dst + (at >> 3) * 8192 + sw128_offset(key, (at & 7) * 8)) = v;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&v_ready[j & 1]);
                mbar_arrive(&v_empty[j % N]);
            }
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");  // poison[] is complete
    } else {
        // ---- softmax: a thread is a query row
        const int row = 32 * (warp & 3) + lane, token = row / p.group, head = kvh * p.group + row - token * p.group;
        const bool live = token < tokens && t0 + token < q.count;
        const int limit = live ? first_position + t0 + token : -1;  // last key position this row sees
        const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const size_t tensor_row = (size_t)(q.first + t0 + (live ? token : 0));
        float back;
        {
            // the warp's rows of q, one bulk copy a row, into shared memory (read directly, a lane's row
            // a lane, they take 7 us; by 16-byte asynchronous copies, 3.5)
            uint8_t *mine = base + B::q_rows + 32 * (warp & 3) * B::q_stride;
            const T *src = static_cast<const T *>(p.q) + tensor_row * p.q_stride + (size_t)(live ? head : 0) * D;
            const unsigned rows_live = __popc(__ballot_sync(0xffffffffu, live));
            bool landed = true;
            if (p.wide) {
                uint64_t *full = &q_full[warp & 3];
                if (lane == 0) mbar_expect_tx(full, rows_live * (unsigned)(D * sizeof(T)));
                __syncwarp();
                if (live) bulk_g2s(mine + lane * B::q_stride, src, D * sizeof(T), full);
                if (!(landed = kv4_warp_wait(full, 0, abort_word))) kv4_landed(full, 0);
            } else {
                for (int d = 0; d < D; d++) reinterpret_cast<T *>(mine + lane * B::q_stride)[d] = src[d];
                __syncwarp();
            }
            const T *row_q = reinterpret_cast<const T *>(mine + lane * B::q_stride);
            float top = 0.0f;
#pragma unroll 4
            for (int d = 0; d < D; d += 8) {
                float x[8];
                load8(row_q + d, true, x);
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
            }
            if (!live || !landed) top = 0.0f;
            // a score is (raw sum) * back with back > 0: the scale's sign goes into q, and a
            // scale of zero becomes one that moves nothing
            float f = power_scale(top, back);
            if (p.scale2 < 0.0f) f = -f;
            back = fmaxf(back * fabsf(p.scale2), 1e-37f);
#pragma unroll 2
            for (int d = 0; d < D; d += 16) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    float x[8];
                    load8(row_q + d + 8 * w, true, x);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        split_half2(live ? x[e] * f : 0.0f, live ? x[e + 4] * f : 0.0f, hi[4 * w + e], lo[4 * w + e]);
                }
                tmem_st8_async(lane_base + q_col + d / 2, hi);
                if (parts == 2) tmem_st8_async(lane_base + q_col + 64u + d / 2, lo);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
        }
        const int all_see = first_position + t0;  // every live row sees keys up to here
        // l_rest: what the additions to l have rounded off, which would add up over thousands of tiles
        float m = -INFINITY, l = 0.0f, l_rest = 0.0f;
        // what O held every few tiles, and what has scaled it since; where q's row was
        float4 *drained = reinterpret_cast<float4 *>(base + B::q_rows + row * B::q_stride);
        float since = 1.0f;
        bool ok = true;
        for (int j = 0; j < tiles; j++) {
            if (!(ok = kv4_warp_wait(&s_full[j >> 1 & 1], (j >> 2) & 1, abort_word))) break;
            tc_fence_after();
            const uint32_t sb = s_col + 128u * (uint32_t)(j >> 1 & 1) + 64u * (uint32_t)(j & 1);
            uint32_t raw_s[64];
            tmem_ld32(lane_base + sb, *reinterpret_cast<uint32_t(*)[32]>(&raw_s[0]));
            tmem_ld32(lane_base + sb + 32u, *reinterpret_cast<uint32_t(*)[32]>(&raw_s[32]));
            const int p0 = k0 + j * kPage;
            float *x = reinterpret_cast<float *>(raw_s);
            if (bad[j & 15] || p0 + kPage - 1 > all_see) {
                const int last = bad[j & 15] ? -1 : limit;
#pragma unroll
                for (int c = 0; c < 64; c++) x[c] = p0 + c <= last ? x[c] : -INFINITY;
            }
            float top0 = x[0], top1 = x[1];
#pragma unroll
            for (int c = 2; c < 62; c += 4) {
                top0 = max3(top0, x[c], x[c + 1]);
                top1 = max3(top1, x[c + 2], x[c + 3]);
            }
            const float mx = max3(fmaxf(top0, top1), x[62], x[63]);
            // m and mx are raw sums, of which differences are scored, so that the largest weight is 2^0 times
            // the shift whatever its size. A row without any key yet has O = 0 and l = 0 and just
            // takes the tile's maximum
            const bool raise = m != -INFINITY && (mx - m) * back > kBlockRaise;
            const float corr = raise ? exp2_fast((m - mx) * back) : 1.0f;
            if (m == -INFINITY || raise) m = mx;
            l *= corr;
            l_rest *= corr;
            const float zero = m == -INFINITY ? 0.0f : -m;
            uint64_t sum = pack2(0.0f, 0.0f);
            const uint64_t back2 = pack2(back, back), zero2 = pack2(zero, zero), shift2 = pack2(kBlockShift, kBlockShift);
            uint32_t ph[32], pl[32];
#pragma unroll
            for (int i = 0; i < 32; i++) {
                float a, b;
                unpack2(fma_f32x2(add_f32x2(pack2(x[2 * i], x[2 * i + 1]), zero2), back2, shift2), a, b);
                a = exp2_fast(a);
                b = exp2_fast(b);
                const uint64_t ab = pack2(a, b);
                sum = add_f32x2(sum, ab);
                // hi: the 11 leading bits, lo: the rest
                const float ha = __uint_as_float(__float_as_uint(a) & 0xffffe000u);
                const float hb = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
                float la, lb;
                unpack2(add_f32x2(ab, pack2(-ha, -hb)), la, lb);
                ph[i] = half2_bits(ha, hb);
                pl[i] = half2_bits(la, lb);
            }
            float sum0, sum1;
            unpack2(sum, sum0, sum1);
            sum0 += sum1;
            const float l_next = l + sum0;
            l_rest += sum0 - (l_next - l);
            l = l_next;
            // with this tile's weights done, so that P V of the tile before has mostly landed
            if (j > 0 && j % B::drain(parts) == 0) {
                // P V of the tile before has landed, and P V of this one starts from zero
                if (!(ok = kv4_warp_wait(&o_done[(j - 1) & 1], (j - 1) >> 1 & 1, abort_word))) break;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(lane_base + o_col + c, o);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float4 sum = j == B::drain(parts) ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : drained[(c + i) / 4];
                        sum.x = fmaf(sum.x, since, __uint_as_float(o[i]));
                        sum.y = fmaf(sum.y, since, __uint_as_float(o[i + 1]));
                        sum.z = fmaf(sum.z, since, __uint_as_float(o[i + 2]));
                        sum.w = fmaf(sum.w, since, __uint_as_float(o[i + 3]));
                        drained[(c + i) / 4] = sum;
                    }
                }
                since = corr;
            } else if (__any_sync(0xffffffffu, raise)) {
                // O's row *= corr once P V of the tile before has landed
                if (!(ok = kv4_warp_wait(&o_done[(j - 1) & 1], (j - 1) >> 1 & 1, abort_word))) break;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(lane_base + o_col + c, o);
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                    tmem_st32(lane_base + o_col + c, o);
                }
                since *= corr;
            }
            tmem_st32(lane_base + sb, ph);
            tmem_st32(lane_base + sb + 32u, pl);
            tc_fence_before();
            // not more than two tiles ahead of P V: a barrier's parity tells only two
            // phases in a row apart, here of p_ready (whose last one the issuer has then seen) and of
            // o_done, which is otherwise asked only on a raise and at the end
            if (j >= 2 && !(ok = kv4_warp_wait(&o_done[j & 1], ((j >> 1) - 1) & 1, abort_word))) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[j & 1]);
        }
        if (ok && tiles > 0) ok = kv4_warp_wait(&o_done[(tiles - 1) & 1], (tiles - 1) >> 1 & 1, abort_word);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (__all_sync(0xffffffffu, ok && !*abort_word)) {
            tc_fence_after();
            l += l_rest;
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
                if (tiles > B::drain(parts)) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 sum = drained[(c + i) / 4];
                        o[i] = __float_as_uint(fmaf(sum.x, since, __uint_as_float(o[i])));
                        o[i + 1] = __float_as_uint(fmaf(sum.y, since, __uint_as_float(o[i + 1])));
                        o[i + 2] = __float_as_uint(fmaf(sum.z, since, __uint_as_float(o[i + 2])));
                        o[i + 3] = __float_as_uint(fmaf(sum.w, since, __uint_as_float(o[i + 3])));
                    }
                }
                const bool nan = limit >= poison[c / kKv4Group];
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++)  // columns 0 .. 7 are dims 0 4 1 5 2 6 3 7
                        x[e] = nan ? __uint_as_float(0x7fc00000u)
                                   : __uint_as_float(o[i + (e & 3) * 2 + (e >> 2)]) * inverse;
                    if (whole) {
                        store8(out + c + i, p.wide, x);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e += 2)
                            *reinterpret_cast<float2 *>(part + c + i + e) = make_float2(x[e], x[e + 1]);
                    }
                }
            }
            if (!whole && live) *reinterpret_cast<float2 *>(part + D) = make_float2(m * back, l);
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
    int s;
    const Kv4Sequence q = kv4_sequence_of_row(p.rows, row, s);
    if (!q.ok || row < q.first || row >= q.first + q.count || q.count * p.group <= least || head >= heads) return;
    const int keys = q.length - q.count + (row - q.first) + 1, width = p.split_pages * kPage;
    const int splits = keys > 0 ? (keys + width - 1) / width : 0;
    const float *part = p.part + ((size_t)row * heads + head) * p.splits * (D + 2);
    kv4_combine<D, T, 1>(p, [&](int i) { return part + (size_t)i * (D + 2); }, splits, row, head);
}

}  // namespace lun
