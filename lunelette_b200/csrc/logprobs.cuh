// Log probabilities of given tokens, entropy and the most probable tokens, from
// rows of logits.
#pragma once
#include "common.cuh"

namespace lun {

constexpr int kMaxTop = 64;

struct LogprobParams {
    const void *logits;
    int rows, vocab, top;
    size_t stride;
    const int64_t *targets;
    float *logprobs, *entropy, *top_logprobs;
    int64_t *top_ids;
};

template <typename T> __device__ __forceinline__ float logit(T v);
template <> __device__ __forceinline__ float logit<float>(float v) { return v; }
template <> __device__ __forceinline__ float logit<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float logit<__half>(__half v) { return __half2float(v); }

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

template <typename T>
static __global__ void __launch_bounds__(256) logprobs_kernel(LogprobParams p)
{
    __shared__ float scratch[32];
    __shared__ unsigned long long best[8];
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_launch_dependents();
    const T *x = static_cast<const T *>(p.logits) + (size_t)row * p.stride;
    float m = -INFINITY;
    bool nan = false;
    for (int i = threadIdx.x; i < p.vocab; i += 256) {
        const float v = logit(x[i]);
        m = fmaxf(m, v);
        nan = nan || v != v;
    }
    m = warp_max(m);
    if (lane == 0) scratch[warp] = m;
    nan = __syncthreads_or(nan);
    for (int w = 0; w < 8; w++) m = fmaxf(m, scratch[w]);
    float z = 0.0f, t = 0.0f;
    for (int i = threadIdx.x; i < p.vocab; i += 256) {
        const float d = logit(x[i]) - m, e = expf(d);
        z += e;
        if (e > 0.0f) t += e * d;
    }
    z = block_sum(z, scratch);
    t = block_sum(t, scratch);
    const float log_z = nan || !(fabsf(m) < INFINITY) ? __uint_as_float(0x7fc00000u) : logf(z);
    if (threadIdx.x == 0) {
        if (p.entropy) p.entropy[row] = log_z - t / z;
        if (p.logprobs) {
            const int64_t id = p.targets[row];
            p.logprobs[row] = id < 0 || id >= p.vocab ? __uint_as_float(0x7fc00000u) : logit(x[id]) - m - log_z;
        }
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; k++) {
        unsigned long long mine = 0;
        for (int i = threadIdx.x; i < p.vocab; i += 256) {
            const unsigned long long key = (unsigned long long)logit_order(logit(x[i])) << 32 | (0xffffffffu - i);
            if (key < last && key > mine) mine = key;
        }
        for (int o = 16; o; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
            mine = other > mine ? other : mine;
        }
        __syncthreads();
        if (lane == 0) best[warp] = mine;
        __syncthreads();
        for (int w = 0; w < 8; w++) mine = best[w] > mine ? best[w] : mine;
        last = mine;
        if (threadIdx.x == 0) {
            p.top_ids[(size_t)row * p.top + k] = 0xffffffffu - (uint32_t)mine;
            p.top_logprobs[(size_t)row * p.top + k] = logit_of_order((uint32_t)(mine >> 32)) - m - log_z;
        }
    }
}

}  // namespace lun
