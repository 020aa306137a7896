// Failed waits of the language-model operators.  A call has no context that
// could hold a status word, so there is one per device: the first failed wait
// (DevStatus) since vxb_operators_sync last read it.
#pragma once

#include "common.cuh"

namespace vxb {

static __device__ int g_op_status;

// The bounded wait of these operators.  One that runs out leaves its code in
// the block's abort flag, which ends the block's other waits; the block
// records it when it ends (record_abort), off the path of the waits: with the
// status word written in the wait itself a batch of 256 single tokens took 34.5
// us for 33.1.
__device__ __forceinline__ bool op_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int code) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer_ns();
    while (true) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort) return false;
        if (globaltimer_ns() - t0 > kWaitNs) {
            *abort = code;
            return false;
        }
    }
}

// After the block's last wait, behind a barrier of its threads: by one of them.
__device__ __forceinline__ void record_abort(volatile int* abort) {
    if (*abort) set_status(&g_op_status, *abort);
}

// One thread waits on a barrier that nothing arrives on, with a short limit.
static __global__ void op_wait_probe_kernel(unsigned long long limit_ns) {
    __shared__ uint64_t bar;
    __shared__ int abort_flag;
    if (threadIdx.x != 0) return;
    mbar_init(&bar, 1);
    abort_flag = 0;
    fence_barrier_init();
    mbar_wait_for(&bar, 0, &abort_flag, &g_op_status, kErrWaitFull, limit_ns);
}

}  // namespace vxb
