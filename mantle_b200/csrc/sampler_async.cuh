// The self-test of the bounded wait on an mbarrier (mbarrier.cuh).
// Part of the device-side logits sampler; included by sampler_kernels.cu, in this order, into one
// translation unit.
#pragma once

#include "mbarrier.cuh"

namespace {

// No kernel of the sampler waits on anything another CTA, copy engine or GPU completes -- the streaming
// kernel uses plain loads -- so the self-test is this unit's only user of the wait; the head projection
// (head_rows.cuh) feeds its tensor cores through it.

// Self-test of the bounded wait: waits on an mbarrier that nothing ever completes.  The wait
// must give up after limit_ns, report it in the status word and leave the context usable.
__global__ void bounded_wait_selftest_kernel(uint64_t limit_ns, int32_t* status) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        mbar_init(&bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const bool landed = mbar_wait(&bar, 0, limit_ns);
    if (!landed && threadIdx.x == 0) atomicOr(status, MANTLE_SAMPLE_STATUS_TIMEOUT);
}

}  // namespace
