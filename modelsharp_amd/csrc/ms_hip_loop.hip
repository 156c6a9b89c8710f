// ms_hip_loop.hip — the launches declared in serving_loop.h: what a server's loop needs around a
// serving step's attention.
#include "serving_loop.h"

#include <algorithm>

#include "paged_plan.h"
#include "sample.h"

namespace msnb {

// ---- a step's plan and its end -----------------------------------------------------------------
hipError_t launch_plan(const PlanArgs& p, int cus, hipStream_t s)
{
    // a token or a new page to a thread, as far as two workgroups to a CU go
    const int64_t items = std::max<int64_t>(p.tokens, p.requests);
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, 2 * cus));
    const unsigned lds = 2 * (p.requests + 1) * sizeof(uint32_t);
    if (lds > 63 * 1024)   // beside the kernel's own
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(paged_plan_kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds))
            return e;
    hipLaunchKernelGGL(paged_plan_kernel, dim3(grid), dim3(256), lds, s, p);
    return hipGetLastError();
}

hipError_t launch_commit(const CommitArgs& p, hipStream_t s)
{
    hipLaunchKernelGGL(paged_commit_kernel, dim3(1), dim3(1024), 0, s, p);
    return hipGetLastError();
}

// ---- sampling ----------------------------------------------------------------------------------
SamplePlan sample_plan(int, int, int) { return {}; }

hipError_t launch_sample(const SampleArgs& p, const SamplePlan&, void*, hipStream_t s)
{
    hipLaunchKernelGGL(sample_any_kernel, dim3(p.rows), dim3(kSampleThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace msnb
