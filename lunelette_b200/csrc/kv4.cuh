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

__device__ __forceinline__ Kv4Sequence kv4_checked(const Kv4Rows &r, int first, int end, int length)
{
    Kv4Sequence q;
    q.first = first;
    q.length = length;
    q.count = (int)((unsigned)end - (unsigned)first);
    q.ok = first >= 0 && end >= first && end <= r.rows && q.count <= r.max_count && length >= 0 && length <= r.max_length;
    return q;
}
__device__ __forceinline__ Kv4Sequence kv4_sequence(const Kv4Rows &r, int s)
{
    return kv4_checked(r, r.offsets[s], r.offsets[s + 1], r.lengths[s]);
}

// The sequence of a row: the last whose first row is at or before it (a whole warp
// asks together). Up to 32 sequences are read a lane each, with their lengths, so that
// one round of loads finds the row's position; more take 32 probes a round first.
__device__ __forceinline__ Kv4Sequence kv4_sequence_of_row(const Kv4Rows &r, int row, int &s)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, n = r.sequences;
    while (n > 32) {
        const int step = (n + 31) / 32, i = lane * step;
        const bool before = i < n && (i == 0 || r.offsets[lo + i] <= row);
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, before));
        lo += last * step;
        n = min(step, n - last * step);
    }
    const bool in = lane < n;
    const int first = in ? r.offsets[lo + lane] : 0, end = in ? r.offsets[lo + lane + 1] : 0;
    const int length = in ? r.lengths[lo + lane] : 0;
    const int who = 31 - __clz(__ballot_sync(0xffffffffu, in && (lane == 0 || first <= row)));
    s = lo + who;
    return kv4_checked(r, __shfl_sync(0xffffffffu, first, who), __shfl_sync(0xffffffffu, end, who),
                       __shfl_sync(0xffffffffu, length, who));
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

// Where a row lives: a position of -1 where there is nothing to do (a row behind the
// last sequence, before position 0, of a sequence that breaks its bounds), a page
// outside the pool as it stands. A warp asks together.
constexpr int kKv4BlockRows = 8;
struct Kv4Place {
    int position, page;
};
__device__ __forceinline__ int kv4_position(const Kv4Rows &r, int row, const int *&table)
{
    int s;
    const Kv4Sequence q = kv4_sequence_of_row(r, row, s);
    table = r.page_tables + s * r.table_stride;
    const bool in = q.ok && row >= q.first && row < q.first + q.count;
    return in ? max(-1, q.length - q.count + (row - q.first)) : -1;
}
// The places of rows row0 .. row0 + n - 1 into shared memory, for the whole block. The pages are on
// their way when it returns: a barrier later they are there. A single row is looked up by
// every warp for itself and returned, without a barrier.
__device__ __forceinline__ Kv4Place kv4_places(const Kv4Rows &r, int pages, int row0, int n, Kv4Place *places, int *status)
{
    const int lane = threadIdx.x & 31;
    const int *table;
    if (n == 1) {
        Kv4Place place;
        place.position = kv4_position(r, row0, table);
        place.page = place.position >= 0 ? table[place.position / kPage] : 0;
        return place;
    }
    int mine = -1;
    const int *my_table = nullptr;
    for (int i = threadIdx.x >> 5; i < n; i += blockDim.x >> 5) {
        const int position = kv4_position(r, row0 + i, table);
        if (lane == 0) places[i].position = position;
        if (lane == i / (blockDim.x >> 5)) mine = position, my_table = table;
    }
    __syncthreads();
    if (mine >= 0) {
        const int i = (threadIdx.x >> 5) + lane * (blockDim.x >> 5), page = my_table[mine / kPage];
        places[i].page = page;
        if ((unsigned)page >= (unsigned)pages) kv4_report(status, kKv4BadPage);
    }
    return places[0];
}
// The blocks behind those of the rows look at every sequence, for no row falls in one whose offsets
// descend, or in an empty one. True in such a block, which is done then.
__device__ __forceinline__ bool kv4_check_sequences(const Kv4Rows &r, int block_rows, int *status)
{
    const int row_blocks = (r.rows + block_rows - 1) / block_rows, check = (int)blockIdx.x - row_blocks;
    if (check < 0) return false;
    for (int s = check * blockDim.x + threadIdx.x; s < r.sequences; s += ((int)gridDim.x - row_blocks) * blockDim.x)
        if (!kv4_sequence(r, s).ok) kv4_report(status, kKv4BadRows);
    return true;
}
__device__ __forceinline__ void kv4_check_page(const Kv4Place &place, int pages, int *status)
{
    if (threadIdx.x == 0 && place.position >= 0 && (unsigned)place.page >= (unsigned)pages) kv4_report(status, kKv4BadPage);
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

// Eight elements as they are, loaded now and converted later.
template <typename T> struct Raw8 {
    static constexpr int vectors = sizeof(T) / 2;
    uint4 u[vectors];
    __device__ __forceinline__ void load(const T *p, bool wide)
    {
        if (wide) {
#pragma unroll
            for (int i = 0; i < vectors; i++) u[i] = reinterpret_cast<const uint4 *>(p)[i];
        } else {
            T *e = reinterpret_cast<T *>(u);
#pragma unroll
            for (int i = 0; i < 8; i++) e[i] = p[i];
        }
    }
    __device__ __forceinline__ void get(float (&x)[8]) const
    {
        const T *e = reinterpret_cast<const T *>(u);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_float(e[i]);
    }
};

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
    int block_rows;  // rows of a block
    bool wide;       // every row of k, v, q and q_out starts on 16 bytes
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

// Eight values of a lane in 64 bits -> their word of codes; the four lanes of an
// aligned quad hold the 32 values of a group. All lanes of the warp call it.
__device__ __noinline__ uint32_t kv4_quantise_exactly(const double (&r)[8], float &scale)
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
    const double d = kv4_scale(finite ? (high >= -low ? high : low) : __longlong_as_double(0x7ff8000000000000ll));
    scale = (float)d;
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

// x c - y s and y c + x s with one rounding of the products' sum and one of the
// second product's error: off by 2^-23 of the result at most, whatever cancels. An infinite
// product has no error to take off.
__device__ __forceinline__ float kv4_turn(float x, float c, float y, float s)
{
    const float t = y * s, error = fmaf(y, s, -t);
    return fmaf(x, c, -t) - (error == error ? error : 0.0f);
}

// Eight values of a lane in FP32 -> their word of codes as in 64 bits. Values that are
// `exact` decide everything: a scale is rounded on their bits, and a quotient next to a
// tie is divided with one rounding, which cannot reach a tie that it is not (d has 8
// bits, so r / d is off a tie by more than half an ulp or not at all). Values within 2^-22 of
// themselves leave the group `unsure` where the scale's rounding, its sign or a quotient lies
// that near a border, about 1 group in 1000. So does, of all, a value that is not finite or
// a scale on the grid of FP16's smallest steps or past the clamp. The quad's lanes hold a
// group and agree on its scale.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&r)[8], bool exact, float &scale, bool &unsure)
{
    float high = r[0], low = r[0];
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        high = fmaxf(high, r[e]);
        low = fminf(low, r[e]);
        nan = nan || r[e] != r[e];
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    const float m = high >= -low ? high : low, top = fabsf(m);
    const uint32_t bits = __float_as_uint(m), rest = bits & 0xffffu;
    // 2^-14 keeps d = m / -8 off the grid of 2^-24, 60000 off the clamp
    unsure = nan || !(top >= 0x1p-14f && top <= 60000.0f) ||
             (!exact && (fabsf(high + low) <= top * 0x1p-20f || (rest >= 0x8000u - 8u && rest <= 0x8000u + 8u)));
    const float d = __uint_as_float((bits + 0x7fffu + (bits >> 16 & 1u)) & 0xffff0000u) * -0.125f;
    scale = d;
    const float inverse = __frcp_rn(d);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float q = r[e] * inverse;
        float c = rintf(q);
        if (fabsf(q - c) > 0.4999f) {
            const float quotient = __fdiv_rn(r[e], d);
            c = rintf(quotient);
            unsure = unsure || (!exact && fabsf(quotient - c) > 0.49999f);
        }
        word |= (uint32_t)((int)fminf(fmaxf(c, -8.0f), 7.0f) + 8) << (4 * e);
    }
    return word;
}

// A block takes block_rows rows one after the other, with its places and rotations
// looked up at once and the next values in flight: one row a block waits four round
// trips to L2 for each (4401 rows of 40 heads of 64 dims: 19 us, of 4 rows 12). D / 16 lanes
// take one head's row, each 8 dims of the lower half and their 8 rotation partners.
// Everything is decided as in 64 bits, in FP32 but for the few values next to a border: with
// FP64 throughout (its conversions run at an eighth of FP32's rate) those rows took 55 us.
template <int D, typename T>
static __global__ void __launch_bounds__(512, 2) kv4_append_kernel(Kv4AppendParams p)
{
    using L = Kv4Layout<D>;
    constexpr int lanes = D / 16;
    __shared__ Kv4Place places[kKv4BlockRows];
    __shared__ __align__(16) float turns[kKv4BlockRows][2][D];  // the positions' cosines and sines
    const int i = threadIdx.x % lanes, heads = p.cache.heads, all = 2 * heads + p.query_heads, step = blockDim.x / lanes;
    const int row0 = blockIdx.x * p.block_rows, n = min(p.block_rows, p.rows.rows - row0);
    pdl_wait();
    pdl_launch_dependents();
    if (kv4_check_sequences(p.rows, p.block_rows, p.status)) return;
    // K heads, V heads, query heads: a thread's values are h = its first head, h + step, ..., row after row
    Raw8<T> raw_lo, raw_hi;
    auto values = [&](int r, int h) {
        const int kind = h < heads ? 0 : h < 2 * heads ? 1 : 2;
        const T *src = static_cast<const T *>(kind == 0 ? p.k : kind == 1 ? p.v : p.q) +
                       (size_t)(row0 + r) * (kind == 0 ? p.k_stride : kind == 1 ? p.v_stride : p.q_stride) +
                       (size_t)(h - min(kind, 2) * heads) * D + 8 * i;
        return src;
    };
    auto fetch = [&](int r, int h) {
        const T *src = values(r, h);
        raw_lo.load(src, p.wide);
        raw_hi.load(src + D / 2, p.wide);
    };
    const int h_first = min((int)threadIdx.x / lanes, all - 1);
    fetch(0, h_first);
    const Kv4Place first = kv4_places(p.rows, p.cache.pages, row0, n, places, p.status);
    if (p.cosine) {
        for (int e = threadIdx.x; e < n * (D / 2); e += blockDim.x) {  // both tables, 4 floats at once
            const int r = e / (D / 2), d = e % (D / 2), position = r ? places[r].position : first.position;
            if (position >= 0)
                reinterpret_cast<float4 *>(turns[r])[d] = reinterpret_cast<const float4 *>(
                    (d < D / 4 ? p.cosine : p.sine) + (size_t)position * D)[d % (D / 4)];
        }
    }
    __syncthreads();
    for (int r = 0; r < n; r++) {
        const Kv4Place place = n == 1 ? first : places[r];
        const int position = place.position, slot = position % kPage;
        for (int h0 = 0; h0 < all; h0 += step) {
            const int h = h0 + (int)threadIdx.x / lanes;
            float lo[8], hi[8], a[8], b[8];
            raw_lo.get(lo);
            raw_hi.get(hi);
            if (h0 + step < all) fetch(r, min(h + step, all - 1));
            else if (r + 1 < n) fetch(r + 1, h_first);
            if (position < 0) continue;
            const bool live = h < all, turn = p.cosine && (h < heads || h >= 2 * heads);
            const float *cl = &turns[r][0][8 * i], *ch = cl + D / 2, *sl = &turns[r][1][8 * i], *sh = sl + D / 2;
            if (turn) {
                float c[8], sn[8];
                load8(cl, true, c);
                load8(sl, true, sn);
#pragma unroll
                for (int e = 0; e < 8; e++) a[e] = kv4_turn(lo[e], c[e], hi[e], sn[e]);
                load8(ch, true, c);
                load8(sh, true, sn);
#pragma unroll
                for (int e = 0; e < 8; e++) b[e] = kv4_turn(hi[e], c[e], -lo[e], sn[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) a[e] = lo[e], b[e] = hi[e];
            }
            if (live && h >= 2 * heads) {
                const float stretch = query_scale(position);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    a[e] *= stretch;
                    b[e] *= stretch;
                }
                T *dst = static_cast<T *>(p.q_out) + (size_t)(row0 + r) * p.q_out_stride + (size_t)(h - 2 * heads) * D + 8 * i;
                store8(dst, p.wide, a);
                store8(dst + D / 2, p.wide, b);
            }
            const bool cached = h < 2 * heads;
            if (!__any_sync(0xffffffffu, cached)) continue;
            if (n == 1) kv4_check_page(place, p.cache.pages, p.status);
            float da, db;
            bool unsure_a, unsure_b;
            uint32_t wa = kv4_quantise(a, !turn, da, unsure_a), wb = kv4_quantise(b, !turn, db, unsure_b);
            // a group with an unsure value is done again in 64 bits: products of two 24-bit values are exact
            // there, and each sum has one rounding
            const unsigned quad = 0xfu << (threadIdx.x & 28);
            const unsigned again_a = __ballot_sync(0xffffffffu, cached && unsure_a);
            const unsigned again_b = __ballot_sync(0xffffffffu, cached && unsure_b);
            if (again_a | again_b) {
                const T *src = values(r, min(h, all - 1));
                for (int part = 0; part < 2; part++) {
                    if (!(part ? again_b : again_a)) continue;
                    double x64[8];
                    for (int e = 0; e < 8; e++) {
                        const double x = to_float(src[e]), y = to_float(src[D / 2 + e]);
                        if (part == 0) x64[e] = turn ? fma(x, (double)cl[e], -(y * (double)sl[e])) : x;
                        else x64[e] = turn ? fma(y, (double)ch[e], x * (double)sh[e]) : y;
                    }
                    float d;
                    const uint32_t word = kv4_quantise_exactly(x64, d);
                    if ((part ? again_b : again_a) & quad) {
                        if (part) wb = word, db = d;
                        else wa = word, da = d;
                    }
                }
            }
            if (!cached) continue;
            const int v = h >= heads;
            uint8_t *block = kv4_block<D>(p.cache, place.page, v ? h - heads : h);
            if (!block) continue;
            const int w = i, w2 = i + L::words / 2, g = i / 4, g2 = g + L::groups / 2;
            *reinterpret_cast<uint32_t *>(block + (v ? L::v_word(slot, w) : L::k_word(slot, w))) = wa;
            *reinterpret_cast<uint32_t *>(block + (v ? L::v_word(slot, w2) : L::k_word(slot, w2))) = wb;
            if ((i & 3) == 0) {
                *reinterpret_cast<__half *>(block + (v ? L::v_scale(slot, g) : L::k_scale(slot, g))) = __float2half_rn(da);
                *reinterpret_cast<__half *>(block + (v ? L::v_scale(slot, g2) : L::k_scale(slot, g2))) = __float2half_rn(db);
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
    int block_rows;
    bool wide;
    int *status;
};

// A block takes block_rows rows, a thread one word of codes at a time. Bound by the trips to
// rows' places and pages, then by the bytes written (append and read of 4401 FP16 rows of 32 + 4
// heads of 64 dims: 24 us together, 2 TB/s).
template <int D, typename T>
static __global__ void __launch_bounds__(256) kv4_read_kernel(Kv4ReadParams p)
{
    using L = Kv4Layout<D>;
    __shared__ Kv4Place places[kKv4BlockRows];
    const int heads = p.cache.heads, per = 2 * heads * L::words;
    const int row0 = blockIdx.x * p.block_rows, n = min(p.block_rows, p.rows.rows - row0);
    pdl_wait();
    pdl_launch_dependents();
    if (kv4_check_sequences(p.rows, p.block_rows, p.status)) return;
    const Kv4Place first = kv4_places(p.rows, p.cache.pages, row0, n, places, p.status);
    if (n == 1) kv4_check_page(first, p.cache.pages, p.status);
    else __syncthreads();
    for (int item = threadIdx.x; item < n * per; item += blockDim.x) {
        const int r = item / per, rest = item - r * per, w = rest % L::words, h = rest / L::words;
        const bool is_v = h >= heads;
        T *dst = static_cast<T *>(is_v ? p.v : p.k);
        const Kv4Place place = n == 1 ? first : places[r];
        const int position = place.position, slot = position % kPage, head = is_v ? h - heads : h;
        const uint8_t *block = kv4_block<D>(p.cache, place.page, head);
        if (position < 0 || !block || !dst) continue;
        const uint32_t word = *reinterpret_cast<const uint32_t *>(block + (is_v ? L::v_word(slot, w) : L::k_word(slot, w)));
        const float d = __half2float(*reinterpret_cast<const __half *>(
            block + (is_v ? L::v_scale(slot, w / 4) : L::k_scale(slot, w / 4))));
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)((int)(word >> (4 * e) & 15u) - 8) * d;
        store8(dst + (size_t)(row0 + r) * (is_v ? p.v_stride : p.k_stride) + (size_t)head * D + 8 * w, p.wide, x);
    }
}

}  // namespace lun
