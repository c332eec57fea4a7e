// C-ABI of the token log probabilities (include/lunelette_cuda.h).
#include "logprobs.cuh"
#include "launch.h"

#include "lunelette_cuda.h"

#include <limits.h>
#include <string.h>

#define LUN_API extern "C" __attribute__((visibility("default")))

using namespace lun;

LUN_API int lunelette_cuda_token_logprobs(const void *logits, int type, size_t rows, size_t vocab, size_t stride,
                                          const int64_t *targets, size_t top, float *logprobs, float *entropy,
                                          int64_t *top_ids, float *top_logprobs, void *stream)
{
    if (type != LUNELETTE_CUDA_FLOAT32 && type != LUNELETTE_CUDA_BFLOAT16 && type != LUNELETTE_CUDA_FLOAT16) return -1;
    if (rows > INT_MAX || !vocab || vocab > 1u << 30 || stride < vocab || stride > (size_t)1 << 32) return -1;
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
    auto kernel = type == LUNELETTE_CUDA_FLOAT32    ? logprobs_kernel<float>
                  : type == LUNELETTE_CUDA_BFLOAT16 ? logprobs_kernel<__nv_bfloat16>
                                                    : logprobs_kernel<__half>;
    return launch(kernel, dim3((unsigned)rows), dim3(256), 0, (cudaStream_t)stream, p) == cudaSuccess ? 0 : -1;
}
