// C-ABI of the 4-bit KV cache (include/lunelette_cuda.h): argument checks and launches.
#include "kv4_attention_tc.cuh"
#include "launch.h"

#include "lunelette_cuda.h"

#include <limits.h>
#include <string.h>

#define LUN_API extern "C" __attribute__((visibility("default")))

using namespace lun;

namespace {

constexpr size_t kMaxRows = 1 << 24, kMaxLength = 1 << 28;

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

size_t element_size(int type) { return type == LUNELETTE_CUDA_FLOAT32 ? 4 : 2; }

bool valid_type(int type)
{
    return type == LUNELETTE_CUDA_FLOAT32 || type == LUNELETTE_CUDA_BFLOAT16 || type == LUNELETTE_CUDA_FLOAT16;
}

size_t block_bytes(size_t head_dim) { return head_dim == 128 ? Kv4Layout<128>::block : Kv4Layout<64>::block; }

bool valid_sizes(size_t layers, size_t pages, size_t kv_heads, size_t head_dim)
{
    return layers && layers <= 4096 && pages && pages <= INT_MAX / 64 && kv_heads && kv_heads <= 256 &&
           pages * kv_heads < 0xffffffffu && (head_dim == 64 || head_dim == 128);
}

bool valid_cache(const lunelette_cuda_kv4 *c, size_t layer)
{
    return c && c->pool && aligned(c->pool, 16) && valid_sizes(c->layers, c->pages, c->kv_heads, c->head_dim) &&
           layer < c->layers;
}

// The sizes of a call; `empty` when there is nothing to do.
bool valid_rows(const lunelette_cuda_rows *r, bool *empty)
{
    if (!r) return false;
    *empty = !r->rows || !r->sequences || !r->max_count;
    if (r->rows > kMaxRows || r->sequences > kMaxRows || r->max_count > kMaxRows || r->max_length > kMaxLength)
        return false;
    if (r->table_stride > kMaxLength || r->max_length > r->table_stride * kPage || !aligned(r->offsets, 4) ||
        !aligned(r->lengths, 4) || !aligned(r->page_tables, 4))
        return false;
    return *empty || (r->offsets && r->lengths && r->page_tables);
}

Kv4Cache cache_of(const lunelette_cuda_kv4 *c, size_t layer)
{
    Kv4Cache k;
    k.layer = static_cast<uint8_t *>(c->pool) + layer * c->pages * c->kv_heads * block_bytes(c->head_dim);
    k.pages = (int)c->pages;
    k.heads = (int)c->kv_heads;
    return k;
}

Kv4Rows rows_of(const lunelette_cuda_rows *r)
{
    Kv4Rows k;
    k.rows = (int)r->rows;
    k.sequences = (int)r->sequences;
    k.offsets = r->offsets;
    k.lengths = r->lengths;
    k.page_tables = r->page_tables;
    k.table_stride = r->table_stride;
    k.max_count = (int)r->max_count;
    k.max_length = (int)r->max_length;
    return k;
}

// Rows of `width` elements at a base, `stride` elements apart: element-aligned,
// and *wide is cleared unless each starts on 16 bytes. A call without rows needs
// no base.
bool valid_tensor(const void *base, size_t stride, size_t width, int type, bool empty, bool *wide)
{
    const size_t size = element_size(type);
    if (!base) return empty;
    if (!aligned(base, size) || stride < width || stride > (size_t)1 << 32) return false;
    if (!aligned(base, 16) || stride * size % 16) *wide = false;
    return true;
}

template <typename F> cudaError_t by_type(int type, F &&f)
{
    switch (type) {
    case LUNELETTE_CUDA_FLOAT32: return f((float)0);
    case LUNELETTE_CUDA_BFLOAT16: return f(__nv_bfloat16());
    default: return f(__half());
    }
}

// Rows of a block: as few as one wave of blocks holds, at 64 registers a thread.
int block_rows_for(size_t rows, unsigned threads)
{
    const size_t slots = 148 * (size_t)(threads > 512 ? 1 : 1024 / threads < 32 ? 1024 / threads : 32);
    const size_t n = (rows + slots - 1) / slots;
    return (int)(n < kKv4BlockRows ? n : kKv4BlockRows);
}

unsigned threads_for(size_t work, size_t most) { return (unsigned)(work < most ? (work + 31) / 32 * 32 : most); }

// Blocks of a call over rows: for the rows, and with a status word to look at the sequences.
dim3 grid_for(const lunelette_cuda_rows *rows, int block_rows, unsigned threads, const int *status)
{
    const size_t checks = status ? (rows->sequences + threads - 1) / threads : 0;
    return dim3((unsigned)((rows->rows + block_rows - 1) / block_rows + (checks < 148 ? checks : 148)));
}

int ok(cudaError_t e) { return e == cudaSuccess ? 0 : -1; }

}  // namespace

LUN_API size_t lunelette_cuda_kv4_bytes(size_t layers, size_t pages, size_t kv_heads, size_t head_dim)
{
    return valid_sizes(layers, pages, kv_heads, head_dim) ? layers * pages * kv_heads * block_bytes(head_dim) : 0;
}

LUN_API int lunelette_cuda_kv4_append(const lunelette_cuda_kv4 *cache, size_t layer, const lunelette_cuda_rows *rows,
                                      int type, const void *k, size_t k_stride, const void *v, size_t v_stride,
                                      const void *q, size_t q_stride, size_t query_heads, void *q_out,
                                      size_t q_out_stride, const float *rope_cos, const float *rope_sin,
                                      size_t rope_positions, int *status, void *stream)
{
    bool empty = false, wide = true;
    if (!valid_cache(cache, layer) || !valid_rows(rows, &empty) || !valid_type(type)) return -1;
    const size_t width = cache->kv_heads * cache->head_dim, q_width = query_heads * cache->head_dim;
    if (!q != !q_out || !rope_cos != !rope_sin || (q && (!query_heads || query_heads > 4096))) return -1;
    if (rope_cos && (!aligned(rope_cos, 16) || !aligned(rope_sin, 16) || rows->max_length > rope_positions)) return -1;
    if (!valid_tensor(k, k_stride, width, type, empty, &wide) || !valid_tensor(v, v_stride, width, type, empty, &wide))
        return -1;
    if (q && (!valid_tensor(q, q_stride, q_width, type, empty, &wide) ||
              !valid_tensor(q_out, q_out_stride, q_width, type, empty, &wide)))
        return -1;
    if (!aligned(status, 4)) return -1;
    if (empty) return 0;
    Kv4AppendParams p;
    memset(&p, 0, sizeof p);
    p.cache = cache_of(cache, layer);
    p.rows = rows_of(rows);
    p.k = k;
    p.v = v;
    p.q = q;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_stride = q_stride;
    p.q_out = q_out;
    p.q_out_stride = q_out_stride;
    p.query_heads = q ? (int)query_heads : 0;
    p.cosine = rope_cos;
    p.sine = rope_sin;
    p.wide = wide;
    p.status = status;
    // a thread for every 16 dims of a row, up to 512
    const unsigned threads = threads_for((2 * cache->kv_heads + p.query_heads) * (cache->head_dim / 16), 512);
    p.block_rows = block_rows_for(rows->rows, threads);
    return ok(by_type(type, [&](auto t) {
        using T = decltype(t);
        auto kernel = cache->head_dim == 128 ? kv4_append_kernel<128, T> : kv4_append_kernel<64, T>;
        return launch(kernel, grid_for(rows, p.block_rows, threads, status), dim3(threads), 0, (cudaStream_t)stream, p);
    }));
}

LUN_API int lunelette_cuda_kv4_read(const lunelette_cuda_kv4 *cache, size_t layer, const lunelette_cuda_rows *rows,
                                    int type, void *k, size_t k_stride, void *v, size_t v_stride, int *status,
                                    void *stream)
{
    bool empty = false, wide = true;
    if (!valid_cache(cache, layer) || !valid_rows(rows, &empty) || !valid_type(type)) return -1;
    const size_t width = cache->kv_heads * cache->head_dim;
    if (!valid_tensor(k, k_stride, width, type, true, &wide) || !valid_tensor(v, v_stride, width, type, true, &wide) ||
        !aligned(status, 4))
        return -1;
    if (empty || (!k && !v)) return 0;
    Kv4ReadParams p;
    memset(&p, 0, sizeof p);
    p.cache = cache_of(cache, layer);
    p.rows = rows_of(rows);
    p.k = k;
    p.v = v;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.block_rows = block_rows_for(rows->rows, 128);
    p.wide = wide;
    p.status = status;
    const unsigned threads = threads_for(p.block_rows * 2 * cache->kv_heads * (cache->head_dim / 8), 256);  // one a word
    return ok(by_type(type, [&](auto t) {
        using T = decltype(t);
        auto kernel = cache->head_dim == 128 ? kv4_read_kernel<128, T> : kv4_read_kernel<64, T>;
        return launch(kernel, grid_for(rows, p.block_rows, threads, status), dim3(threads), 0, (cudaStream_t)stream, p);
    }));
}

// Sequences with more query rows a KV head than this take the block kernel, where
// there are any and the group fits its tiles.
constexpr size_t kBlockLeast = 16;

// How a call's keys and rows are split over the GPU.
struct AttnPlan {
    bool decode, block;  // which kernels run
    bool split;          // decode kernel: hi and lo columns
    // decode kernel: n tiles and rows of a row tile, row tiles of a sequence's KV head, tiles of 16 keys in
    // a unit, blocks, whether items can have many parts
    int nt, tile_rows, tiles, ctas;
    int ranks;  // blocks of an item's cluster; 0: the list
    bool many_parts;
    size_t items, items_offset;
    // block kernel
    int least, block_tiles, block_split_pages, block_splits;
    size_t block_ctas, block_combines;
    size_t part_bytes;
    bool fits;  // all grids and the list's count of pages
};

static AttnPlan plan_attention(const lunelette_cuda_kv4 *cache, const lunelette_cuda_rows *rows, size_t query_heads,
                               int type)
{
    AttnPlan a;
    memset(&a, 0, sizeof a);
    a.fits = true;
    const size_t group = query_heads / cache->kv_heads, part = (cache->head_dim + 2) * sizeof(float);
    const size_t pages = (rows->max_length + kPage - 1) / kPage;
    size_t most = rows->max_count * group;
    a.block = most > kBlockLeast && group <= kBlockRows;
    // a few sequences are not worth the second kernel
    a.decode = !a.block || rows->sequences > 4;
    a.least = a.decode ? (int)kBlockLeast : 0;
    if (a.decode) {
        if (a.block) most = kBlockLeast;
        // rows of an n tile: hi and lo columns for each of 4, or one for each of 8 16-bit rows, whose weights then take
        // two products (4 FP16 sequences of 131072 keys, 8 KV heads of 4: 125 us for 150)
        a.split = type == LUNELETTE_CUDA_FLOAT32 || most <= 4;
        const int lane = a.split ? 4 : 8;
        a.nt = most <= (size_t)lane ? 1 : 2;
        a.tile_rows = lane * a.nt;
        a.tiles = (int)((most + a.tile_rows - 1) / a.tile_rows);
        a.items = rows->sequences * cache->kv_heads * a.tiles;
        const size_t tiles16 = (rows->max_length + 15) / 16;  // of an item
        // a cluster an item, of as many blocks as there are SMs and 16 keys a warp, where a
        // warp's share is a page or less (both sides measured at the kernel). A GPC's SMs hold one
        // or two clusters of 8: 15 of those ran at once (15 KV heads of 2000 keys 10.3 us, 16
        // of them 18.9 in two waves, 11.9 by clusters of 4), and one less is counted on.
        const size_t kClusters8 = 14;
        size_t ranks = 1;
        while (ranks < (size_t)kClusterRanks && a.items * ranks * 2 <= (ranks < 4 ? 148 : 8 * kClusters8) &&
               tiles16 > ranks * kClusterWarps)
            ranks *= 2;
        if (tiles16 <= 4 * ranks * kClusterWarps && a.items * ranks <= 2 * 148) {
            a.ranks = (int)ranks;
        } else {
            const size_t slots = 148 * (a.nt == 1 ? kListCtas : 2), units = pages * a.items;
            const size_t blocks = (units + kListWarps - 1) / kListWarps;
            a.ctas = (int)(blocks < slots ? blocks ? blocks : 1 : slots);
            a.many_parts = (size_t)a.ctas > 4 * a.items;
            a.items_offset = 2 * (size_t)a.ctas * kListWarps * a.tile_rows * part;
            a.part_bytes = a.items_offset + a.items * sizeof(int2);
            a.fits = a.items <= INT_MAX / 64 && a.items * (rows->max_length / kPage + 1) <= INT_MAX;
        }
    }
    if (a.block) {
        const size_t tokens = kBlockRows / group, each = (rows->max_count + tokens - 1) / tokens * rows->sequences;
        const size_t packed = (rows->rows + rows->sequences * (tokens - 1)) / tokens;
        a.block_tiles = (int)(each < packed ? each : packed);
        // the splits whose waves of CTAs take the fewest tiles of keys, a CTA's own
        // steps counted as kOwn of them
        const size_t ctas = a.block_tiles * cache->kv_heads;
        size_t best = ~(size_t)0;
        for (size_t splits = 1; splits <= 16 && splits <= (pages ? pages : 1); splits++) {
            const size_t kOwn = 6, per = (pages + splits - 1) / splits;
            const size_t cost = (ctas * splits + 147) / 148 * (per + kOwn) + (splits > 1 ? 3 : 0);
            if (cost < best) best = cost, a.block_split_pages = (int)per, a.block_splits = (int)splits;
        }
        if (a.block_split_pages < 1) a.block_split_pages = 1;
        if (a.block_splits > 1) a.block_splits = (int)((pages + a.block_split_pages - 1) / a.block_split_pages);
        a.block_ctas = ctas * a.block_splits;
        a.block_combines = a.block_splits > 1 ? rows->rows * ((query_heads + 3) / 4) : 0;
        a.fits = a.fits && a.block_ctas <= INT_MAX && a.block_combines <= INT_MAX;
        const size_t bytes = a.block_splits > 1 ? rows->rows * query_heads * a.block_splits * part : 0;
        if (bytes > a.part_bytes) a.part_bytes = bytes;  // the kernels run one after the other
    }
    return a;
}

static bool valid_heads(const lunelette_cuda_kv4 *cache, const lunelette_cuda_rows *rows, size_t query_heads)
{
    return query_heads && query_heads <= 4096 && query_heads % cache->kv_heads == 0 &&
           rows->max_count <= (size_t)(INT_MAX / 2) / (query_heads / cache->kv_heads);
}

LUN_API size_t lunelette_cuda_kv4_attention_workspace(const lunelette_cuda_kv4 *cache, const lunelette_cuda_rows *rows,
                                                      size_t query_heads)
{
    bool empty = false;
    if (!valid_cache(cache, 0) || !valid_rows(rows, &empty) || !valid_heads(cache, rows, query_heads) || empty) return 0;
    const size_t wide = plan_attention(cache, rows, query_heads, LUNELETTE_CUDA_FLOAT32).part_bytes;
    const size_t narrow = plan_attention(cache, rows, query_heads, LUNELETTE_CUDA_FLOAT16).part_bytes;
    return wide > narrow ? wide : narrow;
}

template <int D, typename T, int NT, bool S>
static cudaError_t launch_decode(Kv4AttnParams p, const AttnPlan &a, cudaStream_t stream)
{
    p.tiles = a.tiles;
    p.most = a.block ? a.least : INT_MAX;
    if (a.ranks) {
        constexpr int smem = Kv4Decode<D, T, NT, kClusterWarps, S>::smem;
        const cudaError_t e = opt_in<kv4_decode_kernel<D, T, NT, kClusterWarps, S>>(smem);
        if (e != cudaSuccess) return e;
        p.ranks = a.ranks;
        return launch_cluster(kv4_decode_kernel<D, T, NT, kClusterWarps, S>, dim3((unsigned)(a.items * a.ranks)),
                              dim3(32 * kClusterWarps), smem, a.ranks, stream, p);
    }
    constexpr int smem = Kv4Decode<D, T, NT, kListWarps, S>::smem;
    cudaError_t e = opt_in<kv4_decode_kernel<D, T, NT, kListWarps, S>>(smem);
    if (e != cudaSuccess) return e;
    p.items = reinterpret_cast<int2 *>(reinterpret_cast<char *>(p.part) + a.items_offset);
    p.list_warps = a.ctas * kListWarps;
    e = launch(kv4_decode_kernel<D, T, NT, kListWarps, S>, dim3((unsigned)a.ctas), dim3(32 * kListWarps), smem, stream, p);
    if (e != cudaSuccess) return e;
    const unsigned rows = (unsigned)(a.items * a.tile_rows);
    if (a.many_parts) return launch(kv4_combine_kernel<D, T, 8>, dim3(rows), dim3(256), 0, stream, p, a.tile_rows);
    return launch(kv4_combine_kernel<D, T, 4>, dim3(rows), dim3(128), 0, stream, p, a.tile_rows);
}

template <int D, typename T>
static cudaError_t launch_block(Kv4AttnParams p, const AttnPlan &a, cudaStream_t stream)
{
    constexpr int smem = Kv4BlockLayout<D>::smem;
    auto kernel = kv4_block_kernel<D, T>;
    cudaError_t e = opt_in<kv4_block_kernel<D, T>>(smem);
    if (e != cudaSuccess) return e;
    p.split_pages = a.block_split_pages;
    p.splits = a.block_splits;
    p.tiles = a.block_tiles;
    e = launch(kernel, dim3((unsigned)a.block_ctas), dim3(kBlockThreads), smem, stream, p, a.least);
    if (e != cudaSuccess || a.block_splits == 1) return e;
    return launch(kv4_block_combine_kernel<D, T>, dim3((unsigned)a.block_combines), dim3(128), 0, stream, p, a.least);
}

template <int D, typename T>
static cudaError_t launch_attention(const Kv4AttnParams &p, const AttnPlan &a, cudaStream_t stream)
{
    cudaError_t e = cudaSuccess;
    constexpr bool wide = sizeof(T) == 4;
    if (a.decode && a.nt == 2) e = launch_decode<D, T, 2, wide>(p, a, stream);
    else if (a.decode && a.split) e = launch_decode<D, T, 1, true>(p, a, stream);
    else if (a.decode) e = launch_decode<D, T, 1, wide>(p, a, stream);
    if (e == cudaSuccess && a.block) e = launch_block<D, T>(p, a, stream);
    return e;
}

LUN_API int lunelette_cuda_kv4_attention(const lunelette_cuda_kv4 *cache, size_t layer,
                                         const lunelette_cuda_rows *rows, int type, const void *q, size_t q_stride,
                                         size_t query_heads, float scale, void *out, size_t out_stride,
                                         void *workspace, size_t workspace_bytes, int *status, void *stream)
{
    bool empty = false, wide = true;
    if (!valid_cache(cache, layer) || !valid_rows(rows, &empty) || !valid_type(type)) return -1;
    if (!valid_heads(cache, rows, query_heads) || !(scale - scale == 0.0f)) return -1;
    const size_t width = query_heads * cache->head_dim;
    if (!valid_tensor(q, q_stride, width, type, empty, &wide) ||
        !valid_tensor(out, out_stride, width, type, empty, &wide) || !aligned(status, 4) || !aligned(workspace, 16))
        return -1;
    if (empty) return 0;
    const AttnPlan a = plan_attention(cache, rows, query_heads, type);
    if (!a.fits || workspace_bytes < a.part_bytes || (a.part_bytes && !workspace)) return -1;
    Kv4AttnParams p;
    memset(&p, 0, sizeof p);
    p.cache = cache_of(cache, layer);
    p.rows = rows_of(rows);
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.group = (int)(query_heads / cache->kv_heads);
    p.scale2 = scale * 1.4426950408889634f;
    p.wide = wide;
    p.part = static_cast<float *>(workspace);
    p.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    return ok(by_type(type, [&](auto t) {
        using T = decltype(t);
        return cache->head_dim == 128 ? launch_attention<128, T>(p, a, st) : launch_attention<64, T>(p, a, st);
    }));
}
