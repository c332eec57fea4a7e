// C-ABI of the token log probabilities (include/lunelette_cuda.h).
#include "logprobs.cuh"
#include "launch.h"

#include "lunelette_cuda.h"

#include <limits.h>
#include <string.h>

#define LUN_API extern "C" __attribute__((visibility("default")))

using namespace lun;

namespace {

template <typename T, int THREADS> cudaError_t launch_clusters(LogprobParams p, cudaStream_t stream)
{
    auto kernel = logprobs_kernel<T, THREADS>;
    constexpr int smem = (int)sizeof(LogprobShared<THREADS>);
    const cudaError_t e = opt_in<logprobs_kernel<T, THREADS>>(smem, true);
    if (e != cudaSuccess) return e;
    return launch_cluster(kernel, dim3((unsigned)((size_t)p.rows * p.parts)), dim3(THREADS), smem, p.parts, stream, p);
}

// CTAs of a row: up to 16, while there are fewer than about one an SM and each
// thread keeps 16 logits.
int parts_of(const LogprobParams &p, int threads)
{
    int parts = 1;
    while (parts < 16 && (size_t)p.rows * parts < 150 && p.vocab / (2 * parts) >= threads * 16) parts *= 2;
    return parts;
}

// 512 threads where a CTA has 4 rounds of loads for them (256 x 131072 FP32: 25.3 us
// against 27.3 with 256), 256 where it has fewer (1000 x 50001 BF16: 28.1 against
// 34.4, one row 5.6 against 6.1), 128 for vocabularies that 256 threads read in two.
template <typename T> cudaError_t launch_rows(LogprobParams p, cudaStream_t stream)
{
    constexpr int round = 4 * LogitVector<T>::n;  // logits of a thread
    if (p.vocab <= 8192) {
        p.parts = parts_of(p, 128);
        return launch_clusters<T, 128>(p, stream);
    }
    p.parts = parts_of(p, 512);
    if (p.vocab / p.parts >= 4 * 512 * round) return launch_clusters<T, 512>(p, stream);
    p.parts = parts_of(p, 256);
    return launch_clusters<T, 256>(p, stream);
}

}  // namespace

LUN_API int lunelette_cuda_token_logprobs(const void *logits, int type, size_t rows, size_t vocab, size_t stride,
                                          const int64_t *targets, size_t top, float *logprobs, float *entropy,
                                          int64_t *top_ids, float *top_logprobs, void *stream)
{
    if (type != LUNELETTE_CUDA_FLOAT32 && type != LUNELETTE_CUDA_BFLOAT16 && type != LUNELETTE_CUDA_FLOAT16) return -1;
    if (rows > INT_MAX / 16 || !vocab || vocab > 1u << 30 || stride < vocab || stride > (size_t)1 << 32) return -1;
    if (!targets != !logprobs || !top != !top_ids || !top != !top_logprobs || top > (size_t)kMaxTop || top > vocab)
        return -1;
    const size_t size = type == LUNELETTE_CUDA_FLOAT32 ? 4 : 2;
    if ((uintptr_t)logits % size || ((uintptr_t)targets | (uintptr_t)top_ids) % 8 ||
        ((uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)top_logprobs) % 4)
        return -1;
    if (!rows) return 0;
    if (!logits) return -1;
    if (!logprobs && !entropy && !top) return 0;
    LogprobParams p;
    memset(&p, 0, sizeof p);
    p.logits = logits;
    p.rows = (int)rows;
    p.vocab = (int)vocab;
    p.stride = stride;
    p.targets = targets;
    p.top = (int)top;
    p.logprobs = logprobs;
    p.entropy = entropy;
    p.top_ids = top_ids;
    p.top_logprobs = top_logprobs;
    cudaStream_t st = (cudaStream_t)stream;
    const cudaError_t e = type == LUNELETTE_CUDA_FLOAT32    ? launch_rows<float>(p, st)
                          : type == LUNELETTE_CUDA_BFLOAT16 ? launch_rows<__nv_bfloat16>(p, st)
                                                            : launch_rows<__half>(p, st);
    return e == cudaSuccess ? 0 : -1;
}
