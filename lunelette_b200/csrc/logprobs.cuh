// Log probabilities of given tokens, entropy and the most probable tokens, from
// rows of logits.
//
// One pass over the logits, which is all the traffic there is. A thread keeps a
// running maximum m, z = sum e^(x - m) and t = sum e^(x - m) (x - m); a raise of m
// by r turns them into z e^-r and (t - r z) e^-r. Then ln p(x) = x - m - ln z and the
// entropy is ln z - t / z. 16 logits a thread share the maximum's update, and
// pairs share their additions and multiplications (FP32x2). A row is read by a
// cluster of 1 to 16 CTAs, merged through distributed shared memory in rank order:
// one launch, no workspace. 256 rows of 131072 FP32 logits with 20 tokens each take
// 25.3 us (5.3 TB/s), one row 5.6 us, 1000 rows of 50001 BF16 logits 28.1 us: what
// is left of HBM's time is the rows' last steps and the second wave of CTAs.
//
// The top tokens come out of the same pass: each thread notes the maximum of
// every few logits that it reads (a record). The threads fall into 64 groups; the
// top-th largest of the groups' maxima is at most the top-th largest logit, so
// only the records that reach this bound, a few dozen, are read again, and the
// elements that reach it get a list, in which each counts the keys above its own:
// its place. Keys are 64 bits, the value's order and the falling id, so ties go to
// the lowest id. A row with more elements at the bound than the list holds
// (nearly all alike, say) or with a NaN is read twice more, by one CTA, with each thread's
// largest key for a bound. So is one of which a mask leaves tokens to fewer groups than `top` (the
// bound is -infinity then, and every logit reaches it): one such row of 131072 FP32 logits
// takes 100 us for 5.5, 256 of them 175 for 25, 1000 BF16 rows of 50001 304 for 30, 20 tokens each.
#pragma once
#include "common.cuh"

#include <cooperative_groups.h>

namespace lun {

constexpr int kMaxTop = 64;
constexpr int kLogprobList = 1024;    // keys, and records to read again
constexpr int kLogprobRecords = 16;   // of a thread

struct LogprobParams {
    const void *logits;
    int rows, vocab, top, parts;  // parts: CTAs of a row's cluster
    size_t stride;
    const int64_t *targets;
    float *logprobs, *entropy, *top_logprobs;
    int64_t *top_ids;
};

template <int THREADS> struct LogprobShared {
    unsigned long long list[kLogprobList], bound;
    float4 part, warps[16];  // m, z, t and whether there was a NaN: the CTA's, its warps'
    float m, log_z;
    uint32_t slots[64], all[64], least;  // orders of the groups' maxima, in the CTA and in the cluster
    int count, again_count, overflow;
    int again[kLogprobList];  // record * THREADS + thread
    float records[kLogprobRecords][THREADS];
};

// A logit's order as an unsigned number: NaN above all, both zeros equal.
__device__ __forceinline__ uint32_t logit_order(float x)
{
    if (x != x) return 0xffffffffu;
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return bits >> 31 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float logit_of_order(uint32_t k)
{
    if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long logit_key(float x, int id)
{
    return (unsigned long long)logit_order(x) << 32 | (0xffffffffu - (uint32_t)id);
}

__device__ __forceinline__ float max_nan(float a, float b, float c)  // NaN if one is
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
constexpr float kLog2e = 1.4426950408889634f, kExpClip = -200.0f;  // e^-200 is 0
__device__ __forceinline__ float exp2_approx(float d)     // 2 ulp; 0 below 2^-126
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}
__device__ __forceinline__ float exp_clipped(float d) { return exp2_approx(d * kLog2e); }

// Two FP32 values in a register pair, and two operations in one instruction.
typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t pair_of(float a, float b)
{
    pair_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(pair_t p, float &a, float &b)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b)
{
    pair_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b)
{
    pair_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c)
{
    pair_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// 16 bytes of logits -> pairs of FP32
template <typename T> struct LogitVector;
template <> struct LogitVector<float> {
    static constexpr int n = 4;
    static constexpr uint32_t lowest = 0xff800000u;  // -infinity
    static __device__ __forceinline__ void get(uint4 u, pair_t *x)
    {
        x[0] = pair_of(__uint_as_float(u.x), __uint_as_float(u.y));
        x[1] = pair_of(__uint_as_float(u.z), __uint_as_float(u.w));
    }
    static __device__ __forceinline__ float one(float v) { return v; }
};
template <> struct LogitVector<__nv_bfloat16> {
    static constexpr int n = 8;
    static constexpr uint32_t lowest = 0xff80ff80u;
    static __device__ __forceinline__ void get(uint4 u, pair_t *x)
    {
        x[0] = pair_of(bf16_lo(u.x), bf16_hi(u.x)), x[1] = pair_of(bf16_lo(u.y), bf16_hi(u.y));
        x[2] = pair_of(bf16_lo(u.z), bf16_hi(u.z)), x[3] = pair_of(bf16_lo(u.w), bf16_hi(u.w));
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <> struct LogitVector<__half> {
    static constexpr int n = 8;
    static constexpr uint32_t lowest = 0xfc00fc00u;
    static __device__ __forceinline__ void get(uint4 u, pair_t *x)
    {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[i] = pair_of(f.x, f.y);
        }
    }
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
};

// (m, z, t) += (m2, z2, t2)
__device__ __forceinline__ void logprob_merge(float &m, float &z, float &t, float m2, float z2, float t2)
{
    const float top = fmaxf(m, m2);
    const float da = fmaxf(m - top, kExpClip), db = fmaxf(m2 - top, kExpClip);  // also where both are -inf
    const float fa = exp_clipped(da), fb = exp_clipped(db);
    t = fmaf(z, da, t) * fa + fmaf(z2, db, t2) * fb;
    z = z * fa + z2 * fb;
    m = top;
}

template <typename T, int THREADS>
static __global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprobs_kernel(LogprobParams p)
{
    namespace cg = cooperative_groups;
    using V = LogitVector<T>;
    // 4 vectors a thread are in flight, 16 values share an update of m
    constexpr int kVectors = 4, kBatch = kVectors * V::n, kStep = 16 / V::n, kWarps = THREADS / 32;
    extern __shared__ __align__(16) uint8_t logprob_smem[];
    LogprobShared<THREADS> &sh = *reinterpret_cast<LogprobShared<THREADS> *>(logprob_smem);
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = p.parts, row = blockIdx.x / parts, part = blockIdx.x % parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) sh.count = sh.again_count = sh.overflow = 0;
    pdl_wait();
    pdl_launch_dependents();
    const T *x = static_cast<const T *>(p.logits) + (size_t)row * p.stride;
    // this CTA's ids [lo, hi), whole 16-byte vectors [a, b) and single elements around them
    const int chunk = ((p.vocab + parts - 1) / parts + 63) & ~63;
    const int lo = min(part * chunk, p.vocab), hi = min(lo + chunk, p.vocab);
    const int skew = (int)(((uintptr_t)(x + lo) & 15) / sizeof(T));
    const int a = min(lo + (skew ? V::n - skew : 0), hi), vectors = (hi - a) / V::n, b = a + vectors * V::n;
    const bool leader = part == 0;
    int64_t target = -1;
    float target_x = 0.0f;
    if (leader && tid == THREADS - 32 && p.targets) {  // the lane that writes the row's results
        target = p.targets[row];
        if (target >= 0 && target < p.vocab) target_x = V::one(x[target]);
    }

    float m = -INFINITY;
    pair_t zz = pair_of(0.0f, 0.0f), tt = zz;
    bool nan = false;
    auto raise = [&](float high) {  // m to high
        const float d = fmaxf(m - high, kExpClip), f = exp_clipped(d);
        const pair_t ff = pair_of(f, f);
        tt = mul2(fma2(zz, pair_of(d, d), tt), ff);
        zz = mul2(zz, ff);
        m = high;
    };
    // the elements around the vectors: at most 2 (V::n - 1), one a thread
    const int edge = tid < a - lo ? lo + tid : b + tid - (a - lo);
    const bool has_single = edge < hi;
    float single = -INFINITY;
    if (has_single) {
        single = V::one(x[edge]);
        if (single != single) nan = true;
        if (single > m) raise(single);
        const float d = fmaxf(single - m, kExpClip), e = exp_clipped(d);
        zz = add2(zz, pair_of(e, 0.0f));
        tt = fma2(pair_of(e, 0.0f), pair_of(d, 0.0f), tt);
    }
    constexpr int round_vectors = kVectors * THREADS;
    const int full = vectors / round_vectors, rounds = full + (vectors % round_vectors != 0);
    const int span = max(1, (rounds + kLogprobRecords - 1) / kLogprobRecords);  // rounds of a record
    float record = -INFINITY;
    int left = span, records = 0;
    const T *base = x + a + tid * V::n;
    auto fetch = [&](uint4 (&u)[kVectors], int r) {  // a round that every thread has whole
#pragma unroll
        for (int j = 0; j < kVectors; j++) u[j] = ld_stream(base + ((size_t)r * round_vectors + j * THREADS) * V::n);
    };
    auto sum = [&](const uint4 *u) {  // 16 values
        pair_t v[8];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kStep; j++) V::get(u[j], v + j * V::n / 2);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float x0, x1;
            unpair(v[i], x0, x1);
            top = max_nan(top, x0, x1);
        }
        if (top != top) {  // the row has no distribution: only its top ids matter from here on
            nan = true;
            top = m;
        }
        if (top > m) raise(top);
        const pair_t down = pair_of(-m, -m), log2e = pair_of(kLog2e, kLog2e);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // -inf, and the NaN of -inf - -inf, land on the clip: weight 0
            float d0, d1;
            unpair(add2(v[i], down), d0, d1);
            const pair_t d = pair_of(fmaxf(d0, kExpClip), fmaxf(d1, kExpClip));
            unpair(mul2(d, log2e), d0, d1);
            const pair_t w = pair_of(exp2_approx(d0), exp2_approx(d1));
            zz = add2(zz, w);
            tt = fma2(w, d, tt);
        }
        record = fmaxf(record, top);
    };
    auto note = [&](bool end) {
        if (--left == 0 || end) {
            sh.records[records++][tid] = record;
            record = -INFINITY;
            left = span;
        }
    };
    auto take = [&](const uint4 (&u)[kVectors], int r) {
#pragma unroll
        for (int j = 0; j < kVectors; j += kStep) sum(u + j);
        note(r == rounds - 1);
    };
    uint4 even[kVectors], odd[kVectors];  // one round is in flight while the other's values are summed
    if (full > 0) fetch(even, 0);
    for (int r = 0; r < full; r += 2) {
        if (r + 1 < full) fetch(odd, r + 1);
        take(even, r);
        if (r + 1 >= full) break;
        if (r + 2 < full) fetch(even, r + 2);
        take(odd, r + 1);
    }
    if (full < rounds) {
        const int v0 = full * round_vectors + tid;
#pragma unroll
        for (int j = 0; j < kVectors; j++) {
            even[j] = make_uint4(V::lowest, V::lowest, V::lowest, V::lowest);
            if (v0 + j * THREADS < vectors) even[j] = ld_stream(x + a + (size_t)(v0 + j * THREADS) * V::n);
        }
#pragma unroll
        for (int j = 0; j < kVectors; j += kStep)
            if (full * round_vectors + j * THREADS < vectors) sum(even + j);
        note(true);
    }
    float z, t, z1, t1;
    unpair(zz, z, z1);
    unpair(tt, t, t1);
    z += z1;
    t += t1;
    const float best = m;  // the thread's largest

    constexpr int each = THREADS / 64;  // threads of a group, which share its work too
    // the top-th largest of 64 orders; all threads call
    auto select = [&](const uint32_t *slots) {
        const uint32_t mine = slots[tid / each];
        int above = 0, equal = 0;
#pragma unroll
        for (int i = 0; i < 64 / each; i++) {
            const uint32_t other = slots[tid % each + i * each];
            above += other > mine;
            equal += other == mine;
        }
#pragma unroll
        for (int o = 1; o < each; o <<= 1) {
            above += __shfl_xor_sync(0xffffffffu, above, o);
            equal += __shfl_xor_sync(0xffffffffu, equal, o);
        }
        if (above < p.top && above + equal >= p.top) sh.least = mine;
        __syncthreads();
    };

    // (m, z, t) of the CTA, then of the cluster, each in a fixed order
    auto merge_lanes = [&] {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            logprob_merge(m, z, t, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, z, o),
                          __shfl_xor_sync(0xffffffffu, t, o));
    };
    auto take_part = [&](const float4 &f) {
        m = f.x, z = f.y, t = f.z, nan = f.w != 0.0f;
    };
    const float4 none = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    merge_lanes();
    nan = __any_sync(0xffffffffu, nan);
    if (lane == 0) sh.warps[warp] = make_float4(m, z, t, nan ? 1.0f : 0.0f);
    if (p.top) {
        // neighbouring lanes make a group
        uint32_t order = logit_order(best);
#pragma unroll
        for (int o = 1; o < each; o <<= 1) order = max(order, __shfl_xor_sync(0xffffffffu, order, o));
        if (tid % each == 0) sh.slots[tid / each] = order;
    }
    __syncthreads();
    if (warp == 0) {
        take_part(lane < kWarps ? sh.warps[lane] : none);
        merge_lanes();
        nan = __any_sync(0xffffffffu, nan);
        if (lane == 0) sh.part = make_float4(m, z, t, nan ? 1.0f : 0.0f);
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    LogprobShared<THREADS> &lead = parts > 1 ? *cluster.map_shared_rank(&sh, 0) : sh;
    if (p.top) {
        const uint32_t *slots = sh.slots;
        if (parts > 1) {
            uint32_t order = 0;
            for (int i = tid % each; i < parts; i += each)
                order = max(order, cluster.map_shared_rank(&sh, i)->slots[tid / each]);
#pragma unroll
            for (int o = 1; o < each; o <<= 1) order = max(order, __shfl_xor_sync(0xffffffffu, order, o));
            if (tid % each == 0) sh.all[tid / each] = order;
            slots = sh.all;
            __syncthreads();
        }
        select(slots);
        const float least = logit_of_order(sh.least);
        auto put_key = [&](float v, int id) {  // to the leader's list
            const int at = atomicAdd(&lead.count, 1);
            if (at < kLogprobList) lead.list[at] = logit_key(v, id);
        };
        if (has_single && single >= least) put_key(single, edge);
        for (int i = 0; i < records; i++)
            if (sh.records[i][tid] >= least) {
                const int at = atomicAdd(&sh.again_count, 1);
                if (at < kLogprobList) sh.again[at] = i * THREADS + tid;
            }
        __syncthreads();
        const int n = sh.again_count;
        if (tid == 0 && (n > kLogprobList || sh.part.w != 0.0f)) lead.overflow = 1;
        for (int i = warp; i < min(n, kLogprobList); i += kWarps) {  // a warp reads a record's logits again
            const int who = sh.again[i] % THREADS, first = sh.again[i] / THREADS * span * kBatch;
            for (int k = first + lane; k < min(first + span * kBatch, rounds * kBatch); k += 32) {
                const int vector = k / V::n * THREADS + who, id = a + vector * V::n + k % V::n;
                if (vector >= vectors) continue;
                const float v = V::one(x[id]);
                if (v >= least) put_key(v, id);
            }
        }
    }
    if (leader && warp == kWarps - 1) {
        take_part(lane < parts ? (parts > 1 ? cluster.map_shared_rank(&sh, lane) : &sh)->part : none);
        merge_lanes();
        nan = __any_sync(0xffffffffu, nan);
        if (lane == 0) {
            const float nothing = __uint_as_float(0x7fc00000u);
            const float log_z = nan || !(fabsf(m) < INFINITY) ? nothing : logf(z);
            sh.m = m;
            sh.log_z = log_z;
            if (p.entropy) p.entropy[row] = log_z - t / z;
            if (p.logprobs) p.logprobs[row] = target >= 0 && target < p.vocab ? target_x - m - log_z : nothing;
        }
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    if (!leader || !p.top) return;
    const float row_m = sh.m, log_z = sh.log_z;
    auto place_of = [&](unsigned long long key, int n) {
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) place += sh.list[j] > key;
        return place;
    };
    int n = sh.count;
    if (sh.overflow || n > kLogprobList) {
        // read the row for each thread's largest key, then for the keys from the top-th
        // largest of those on; while they are too many, from the top-th largest of a full list on
        unsigned long long mine = 0;
        for (int i = tid; i < p.vocab; i += THREADS) mine = max(mine, logit_key(V::one(x[i]), i));
        __syncthreads();
        sh.list[tid] = mine;
        if (tid == 0) sh.bound = 0;
        __syncthreads();
        for (n = THREADS;; n = kLogprobList) {
            for (int i = tid; i < n; i += THREADS)
                if (place_of(sh.list[i], n) == p.top - 1) sh.bound = sh.list[i];
            __syncthreads();
            const unsigned long long bound = sh.bound;
            if (tid == 0) sh.count = 0;
            __syncthreads();
            for (int i = tid; i < p.vocab; i += THREADS) {
                const unsigned long long key = logit_key(V::one(x[i]), i);
                if (key < bound) continue;
                const int at = atomicAdd(&sh.count, 1);
                if (at < kLogprobList) sh.list[at] = key;
            }
            __syncthreads();
            if (sh.count <= kLogprobList) break;
        }
        n = sh.count;
    }
    for (int i = tid; i < n; i += THREADS) {
        const unsigned long long key = sh.list[i];
        const int place = place_of(key, n);
        if (place >= p.top) continue;
        p.top_ids[(size_t)row * p.top + place] = 0xffffffffu - (uint32_t)key;
        p.top_logprobs[(size_t)row * p.top + place] = logit_of_order((uint32_t)(key >> 32)) - row_m - log_z;
    }
}

}  // namespace lun
