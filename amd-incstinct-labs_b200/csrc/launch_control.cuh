// Cluster launch control of sm_100a (PTX clusterlaunchcontrol): a running CTA takes over the index of a CTA of its grid that has not
// started yet, so that a grid of one CTA per work item is drawn from like a queue, without a counter in memory.  For launches
// without clusters.  After a request that came back empty no other may be made.
#pragma once
#include "dme/dme_tma.cuh"

namespace b200p {

// Asks for an index; the 16-byte answer arrives in `answer` (shared memory, 16-byte aligned) as one phase of `bar` (one arrival).
__device__ __forceinline__ void request_cta(void* answer, uint64_t* bar) {
    dme::fence_proxy_async_smem();                         // the last answer has been read
    dme::mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 :: "r"(dme::smem_addr(answer)), "r"(dme::smem_addr(bar)) : "memory");
}
// The answer, once its phase has completed: blockIdx.x of the CTA taken over, or -1.
__device__ __forceinline__ int taken_cta(const void* answer) {
    uint32_t some, x;
    asm volatile("{\n\t.reg .b128 a;\n\t.reg .pred p;\n\tld.shared.b128 a, [%2];\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t}"
                 : "=r"(some), "=r"(x) : "r"(dme::smem_addr(answer)) : "memory");
    return some ? int(x) : -1;
}

} // namespace b200p
