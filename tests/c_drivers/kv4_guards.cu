// What keeps the attention over the 4-bit cache inside its memory when a wait gives up, for the tests.
#include "kv4_attention_tc.cuh"

#define EXPORT extern "C" __attribute__((visibility("default")))

EXPORT int valid_record(int first_part, int last_warp, int list_warps)
{
    return lun::kv4_valid_record(first_part, last_warp, list_warps);
}

// One warp, two barriers: [0] that nothing ever completes, [1] of a copy in flight. `aborted` is what the
// abort word holds before. Of each step what it returned, and its nanoseconds.
struct Waits {
    int waited, landed, copied, abort_word;
    unsigned long long wait_ns, land_ns;
    int words_right;
};

static __global__ void waits_kernel(Waits *out, const int *src, int aborted)
{
    using namespace lun;
    __shared__ __align__(16) int copy[1024];
    __shared__ __align__(8) uint64_t bars[2];
    __shared__ volatile int abort_word;
    if (threadIdx.x == 0) {
        mbar_init(&bars[0], 1);
        mbar_init(&bars[1], 1);
        abort_word = aborted;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (threadIdx.x == 0) {
        mbar_expect_tx(&bars[1], sizeof copy);
        bulk_g2s(copy, src, sizeof copy, &bars[1]);
    }
    __syncwarp();
    const bool copied = kv4_landed(&bars[1], 0);
    int right = 0;
    for (int i = threadIdx.x; i < 1024; i += 32) right += copied && copy[i] == src[i];
    for (int o = 16; o; o >>= 1) right += __shfl_xor_sync(0xffffffffu, right, o);
    const unsigned long long t0 = wait_clock_ns();
    const bool waited = kv4_warp_wait(&bars[0], 0, &abort_word);
    const unsigned long long t1 = wait_clock_ns();
    const bool landed = kv4_landed(&bars[0], 0);
    const unsigned long long t2 = wait_clock_ns();
    if (threadIdx.x == 0) {
        out->waited = waited;
        out->landed = landed;
        out->copied = copied;
        out->abort_word = abort_word;
        out->wait_ns = t1 - t0;
        out->land_ns = t2 - t1;
        out->words_right = right;
    }
}

EXPORT int run_waits(Waits *out, const int *src, int aborted)
{
    waits_kernel<<<1, 32>>>(out, src, aborted);
    return cudaDeviceSynchronize() == cudaSuccess ? 0 : -1;
}
