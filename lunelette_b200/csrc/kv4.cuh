// The paged 4-bit KV cache: its layout, the rows of a ragged call, and the
// kernels that append rows (rotation and quantisation on the way) and read them
// back. The format is stated in include/lunelette_cuda.h.
//
// Why these choices. d keeps 8 significant bits and |c - 8| <= 8 has at most 3
// below its leading power of two, so d * (c - 8) has at most 11: FP16 holds it
// exactly, and the attention kernels feed the tensor cores the stored values
// themselves, with one exact multiplication and no rounding of their own. A row
// of a position shares no byte with another position's, so an append never reads
// what it writes beside. The word orders are those in which the attention's
// fragments read 16 (K) or 8 (V) consecutive bytes a lane without shared-memory
// bank conflicts.
#pragma once
#include "common.cuh"

namespace lun {

constexpr int kKv4Group = 32;  // dims that share a scale

template <int D> struct Kv4Layout {
    static constexpr int words = D / 8;            // 32-bit words of a row
    static constexpr int groups = D / kKv4Group;
    static constexpr int codes = kPage * D / 2;    // bytes of K (or V) codes of a block
    static constexpr int scales = kPage * groups * 2;
    static constexpr int k_scales = codes, v_codes = codes + scales, v_scales = 2 * codes + scales;
    static constexpr int block = 2 * (codes + scales);  // bytes of one (layer, page, KV head)
    // byte offsets within a block
    __host__ __device__ static constexpr int k_word(int slot, int w)
    {
        return slot * (D / 2) + 4 * ((w & 3) * groups + (w >> 2));
    }
    __host__ __device__ static constexpr int v_word(int slot, int w)
    {
        const int n = slot * words + w;
        return v_codes + 4 * (n ^ (8 * ((n >> 5) & (D == 128 ? 3 : 1))));
    }
    __host__ __device__ static constexpr int k_scale(int slot, int g) { return k_scales + 2 * (slot * groups + g); }
    __host__ __device__ static constexpr int v_scale(int slot, int g)
    {
        return v_scales + 2 * (((slot >> 1) * groups + g) * 2 + (slot & 1));
    }
};

// Bits of the caller's status word.
constexpr int kKv4BadRows = 1, kKv4BadPage = 2;

struct Kv4Cache {
    uint8_t *layer;  // the layer's first block
    int pages, heads;
};

struct Kv4Rows {
    int rows, sequences;
    const int *offsets, *lengths, *page_tables;
    size_t table_stride;
    int max_count, max_length;
};

// One sequence's rows, checked against the launch's bounds.
struct Kv4Sequence {
    int first, count, length;
    bool ok;
};

__device__ __forceinline__ Kv4Sequence kv4_sequence(const Kv4Rows &r, int s)
{
    Kv4Sequence q;
    const int end = r.offsets[s + 1];
    q.first = r.offsets[s];
    q.length = r.lengths[s];
    q.count = (int)((unsigned)end - (unsigned)q.first);
    q.ok = q.first >= 0 && end >= q.first && end <= r.rows && q.count <= r.max_count && q.length >= 0 &&
           q.length <= r.max_length;
    return q;
}

// The last sequence whose first row is at or before `row` (a whole warp asks
// together): 32 probes a round, so 1024 sequences take two rounds of loads.
__device__ __forceinline__ int kv4_sequence_of_row(const Kv4Rows &r, int row)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, n = r.sequences;
    while (n > 1) {
        const int step = (n + 31) / 32, i = lane * step;
        const bool before = i < n && (i == 0 || r.offsets[lo + i] <= row);
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, before));
        lo += last * step;
        n = min(step, n - last * step);
    }
    return lo;
}

// The block of (page, head), or nullptr for a page outside the pool.
template <int D>
__device__ __forceinline__ uint8_t *kv4_block(const Kv4Cache &c, int page, int head)
{
    if ((unsigned)page >= (unsigned)c.pages) return nullptr;
    return c.layer + ((size_t)page * c.heads + head) * Kv4Layout<D>::block;
}

__device__ __forceinline__ void kv4_report(int *status, int bit)
{
    if (status) atomicOr(status, bit);
}

// ---- element types ------------------------------------------------------------------
// Eight consecutive elements <-> FP32. `wide` says that the address is a multiple
// of 16 bytes (32 for FP32 is not needed: two loads).
template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T>
__device__ __forceinline__ void load8(const T *p, bool wide, float (&x)[8])
{
    constexpr int vectors = sizeof(T) / 2;
    if (wide) {
        uint4 u[vectors];
#pragma unroll
        for (int i = 0; i < vectors; i++) u[i] = reinterpret_cast<const uint4 *>(p)[i];
        const T *e = reinterpret_cast<const T *>(u);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_float(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_float(p[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, bool wide, const float (&x)[8])
{
    constexpr int vectors = sizeof(T) / 2;
    if (wide) {
        uint4 u[vectors];
        T *e = reinterpret_cast<T *>(u);
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = from_float<T>(x[i]);
#pragma unroll
        for (int i = 0; i < vectors; i++) reinterpret_cast<uint4 *>(p)[i] = u[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = from_float<T>(x[i]);
    }
}

// ---- append -------------------------------------------------------------------------
struct Kv4AppendParams {
    Kv4Cache cache;
    Kv4Rows rows;
    const void *k, *v, *q;
    size_t k_stride, v_stride, q_stride, q_out_stride;
    void *q_out;
    int query_heads;  // 0: no q
    const float *cosine, *sine;
    bool wide;  // every row of k, v, q and q_out starts on 16 bytes
    int *status;
};

// m / -8 rounded to 8 significant bits on the grid of 2^-24, at most 8160 in
// magnitude; NaN for a NaN or an infinity. One rounding, from 64 bits.
__device__ __forceinline__ double kv4_scale(double m)
{
    const double x = m * -0.125, a = fabs(x);
    if (!(a <= 1.7976931348623157e308)) return __longlong_as_double(0x7ff8000000000000ll);
    double d;
    if (a >= 0x1p-17) {
        long long bits = __double_as_longlong(x);
        bits += ((1ll << 44) - 1) + ((bits >> 45) & 1);
        d = __longlong_as_double(bits & ~((1ll << 45) - 1));
    } else {
        d = rint(x * 0x1p24) * 0x1p-24;
    }
    return fmin(fmax(d, -8160.0), 8160.0);
}

// Eight values of a lane -> their word of codes; the four lanes of an aligned
// quad hold the 32 values of a group. All lanes of the warp call it.
__device__ __forceinline__ uint32_t kv4_quantise(const double (&r)[8], __half &scale)
{
    double high = r[0], low = r[0];
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        high = fmax(high, r[e]);
        low = fmin(low, r[e]);
        finite = finite && fabs(r[e]) <= 1.7976931348623157e308;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        high = fmax(high, __shfl_xor_sync(0xffffffffu, high, o));
        low = fmin(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    const unsigned quad = 0xfu << (threadIdx.x & 28);
    finite = (__ballot_sync(0xffffffffu, finite) & quad) == quad;
    const double d = finite ? kv4_scale(high >= -low ? high : low) : kv4_scale(__longlong_as_double(0x7ff8000000000000ll));
    scale = __float2half_rn((float)d);
    uint32_t word = 0x88888888u;
    if (finite && d != 0.0) {
        word = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = (int)fmin(fmax(rint(r[e] / d), -8.0), 7.0) + 8;
            word |= (uint32_t)c << (4 * e);
        }
    }
    return word;
}

// One block per row; D / 16 lanes take one head's row, each 8 dims of the lower
// half and their 8 rotation partners.
template <int D, typename T>
static __global__ void __launch_bounds__(256) kv4_append_kernel(Kv4AppendParams p)
{
    using L = Kv4Layout<D>;
    constexpr int lanes = D / 16;
    const int row = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const int s = kv4_sequence_of_row(p.rows, row);
    const Kv4Sequence q = kv4_sequence(p.rows, s);
    if (!q.ok) {
        if (threadIdx.x == 0) kv4_report(p.status, kKv4BadRows);
        return;
    }
    if (row < q.first || row >= q.first + q.count) return;  // behind the last sequence
    const int position = q.length - q.count + (row - q.first);
    if (position < 0) return;
    const int page = p.rows.page_tables[s * p.rows.table_stride + position / kPage], slot = position % kPage;
    if ((unsigned)page >= (unsigned)p.cache.pages && threadIdx.x == 0) kv4_report(p.status, kKv4BadPage);
    const int heads = p.cache.heads, all = 2 * heads + p.query_heads;
    const int i = threadIdx.x % lanes;
    const float stretch = query_scale(position);
    for (int h0 = 0; h0 < all; h0 += blockDim.x / lanes) {
        const int h = h0 + threadIdx.x / lanes;  // K heads, V heads, query heads
        const bool live = h < all;
        const int kind = h < heads ? 0 : h < 2 * heads ? 1 : 2;
        const int head = live ? h - (kind == 0 ? 0 : kind == 1 ? heads : 2 * heads) : 0;
        const T *src = static_cast<const T *>(kind == 0 ? p.k : kind == 1 || !live ? p.v : p.q) +
                       (size_t)row * (kind == 0 ? p.k_stride : kind == 1 || !live ? p.v_stride : p.q_stride) +
                       (size_t)head * D + 8 * i;
        float lo[8], hi[8];
        load8(src, p.wide, lo);
        load8(src + D / 2, p.wide, hi);
        double a[8], b[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            a[e] = lo[e];
            b[e] = hi[e];
        }
        if (kind != 1 && p.cosine) {
            const float *c = p.cosine + (size_t)position * D + 8 * i, *sn = p.sine + (size_t)position * D + 8 * i;
            float cl[8], ch[8], sl[8], sh[8];
            load8(c, true, cl);
            load8(c + D / 2, true, ch);
            load8(sn, true, sl);
            load8(sn + D / 2, true, sh);
            // products of two 24-bit values are exact in 64 bits: one rounding in each sum
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const double x = a[e], y = b[e];
                a[e] = fma(x, (double)cl[e], -(y * (double)sl[e]));
                b[e] = fma(y, (double)ch[e], x * (double)sh[e]);
            }
        }
        __half da, db;
        const uint32_t wa = kv4_quantise(a, da), wb = kv4_quantise(b, db);
        if (!live) continue;
        if (kind == 2) {
            float x[8], y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[e] = (float)a[e] * stretch;
                y[e] = (float)b[e] * stretch;
            }
            T *dst = static_cast<T *>(p.q_out) + (size_t)row * p.q_out_stride + (size_t)head * D + 8 * i;
            store8(dst, p.wide, x);
            store8(dst + D / 2, p.wide, y);
        } else if (uint8_t *block = kv4_block<D>(p.cache, page, head)) {
            const int w = i, w2 = i + L::words / 2, g = i / 4, g2 = g + L::groups / 2;
            *reinterpret_cast<uint32_t *>(block + (kind ? L::v_word(slot, w) : L::k_word(slot, w))) = wa;
            *reinterpret_cast<uint32_t *>(block + (kind ? L::v_word(slot, w2) : L::k_word(slot, w2))) = wb;
            if ((i & 3) == 0) {
                *reinterpret_cast<__half *>(block + (kind ? L::v_scale(slot, g) : L::k_scale(slot, g))) = da;
                *reinterpret_cast<__half *>(block + (kind ? L::v_scale(slot, g2) : L::k_scale(slot, g2))) = db;
            }
        }
    }
}

// ---- read ---------------------------------------------------------------------------
struct Kv4ReadParams {
    Kv4Cache cache;
    Kv4Rows rows;
    void *k, *v;  // either may be nullptr
    size_t k_stride, v_stride;
    bool wide;
    int *status;
};

// One block per row; a thread takes one word of codes.
template <int D, typename T>
static __global__ void __launch_bounds__(256) kv4_read_kernel(Kv4ReadParams p)
{
    using L = Kv4Layout<D>;
    const int row = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const int s = kv4_sequence_of_row(p.rows, row);
    const Kv4Sequence q = kv4_sequence(p.rows, s);
    if (!q.ok) {
        if (threadIdx.x == 0) kv4_report(p.status, kKv4BadRows);
        return;
    }
    if (row < q.first || row >= q.first + q.count) return;
    const int position = q.length - q.count + (row - q.first);
    if (position < 0) return;
    const int page = p.rows.page_tables[s * p.rows.table_stride + position / kPage], slot = position % kPage;
    if ((unsigned)page >= (unsigned)p.cache.pages) {
        if (threadIdx.x == 0) kv4_report(p.status, kKv4BadPage);
        return;
    }
    const int heads = p.cache.heads;
    for (int item = threadIdx.x; item < 2 * heads * L::words; item += blockDim.x) {
        const int w = item % L::words, h = item / L::words;
        const bool is_v = h >= heads;
        const int head = is_v ? h - heads : h;
        T *dst = static_cast<T *>(is_v ? p.v : p.k);
        if (!dst) continue;
        const uint8_t *block = kv4_block<D>(p.cache, page, head);
        const uint32_t word = *reinterpret_cast<const uint32_t *>(block + (is_v ? L::v_word(slot, w) : L::k_word(slot, w)));
        const float d = __half2float(*reinterpret_cast<const __half *>(
            block + (is_v ? L::v_scale(slot, w / 4) : L::k_scale(slot, w / 4))));
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)((int)(word >> (4 * e) & 15u) - 8) * d;
        store8(dst + (size_t)row * (is_v ? p.v_stride : p.k_stride) + (size_t)head * D + 8 * w, p.wide, x);
    }
}

}  // namespace lun
