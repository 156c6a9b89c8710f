// ms_hip_loop.hip — the launches declared in serving_loop.h: what a server's loop needs around a
// serving step's attention.
#include "serving_loop.h"

#include <algorithm>

#include "paged_attention.h"
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

// ---- attention behind shared prefixes ------------------------------------------------------------
SharedPlan shared_attention_plan(int64_t tokens, int requests, int64_t max_new, int groups, int64_t prefix, int64_t rest,
                                 int H, int kvH, int D, int f16, int cus)
{
    SharedPlan pl;
    if (groups <= 0) return pl;
    const int64_t grp = H / kvH, size = f16 ? 2 : 4;
    const bool fit = f16 || D <= 128;   // an fp32 block's three parts in LDS
    pl.few_rows = f16 ? 64 : 128;
    pl.prefix_blocks = fit && tokens * grp > (int64_t)pl.few_rows * groups;
    const int64_t far = pl.prefix_blocks ? tokens * grp / 128 + groups : tokens * grp / 16 + groups;
    const bool few = max_new * grp <= pl.few_rows || !fit;
    const int64_t blocks = few ? 0 : tokens * grp / 128 + std::min<int64_t>(requests, tokens * grp / (pl.few_rows + 1) + 1);
    const int64_t rows16 = tokens * grp / 16 + requests;
    const int64_t rows = few ? rows16 : std::min<int64_t>(rows16, (int64_t)requests * (pl.few_rows / 16));
    const int64_t near = few ? std::max<int64_t>(1, std::min(rows, (max_new * grp + 15) / 16 * requests))
                             : tokens * grp / 128 + 1 + std::min<int64_t>(requests, tokens);
    auto count = [&](int64_t tiles, int64_t keys, int64_t most) {
        const int64_t bytes = keys * D * size;
        return std::max<int64_t>(1, std::min<int64_t>({2 * (int64_t)cus / std::max<int64_t>(1, tiles * kvH), bytes >> 15, most}));
    };
    pl.prefix_splits = (int)count(far, prefix, 32);
    pl.splits = pl.prefix_splits + (int)count(near, rest, 16);
    pl.prefix_min = (int)((prefix + pl.prefix_splits - 1) / pl.prefix_splits);
    pl.split_min = (int)((rest + pl.splits - pl.prefix_splits - 1) / (pl.splits - pl.prefix_splits));
    pl.prefix_grid = far * pl.prefix_splits * kvH;
    pl.blocks_grid = blocks * (pl.splits - pl.prefix_splits) * kvH;
    pl.rows_grid = rows * (pl.splits - pl.prefix_splits) * kvH;
    pl.ws_bytes = pl.splits * tokens * H * (D + 2) * (int64_t)sizeof(float);
    return pl;
}

namespace {
template <typename T, bool WHOLE, PagedMode MODE>
void launch_shared(const SharedAttnArgs& p, unsigned grid, hipStream_t s)
{
    if (p.D <= 64)
        hipLaunchKernelGGL((shared_attention_kernel<T, 64, WHOLE, MODE>), dim3(grid), dim3(256), 0, s, p);
    else if (MODE != kPagedRows && p.D <= 96)
        hipLaunchKernelGGL((shared_attention_kernel<T, MODE == kPagedRows ? 64 : 96, WHOLE, MODE>), dim3(grid), dim3(256), 0, s, p);
    else if (p.D <= 128)
        hipLaunchKernelGGL((shared_attention_kernel<T, 128, WHOLE, MODE>), dim3(grid), dim3(256), 0, s, p);
    else if constexpr (sizeof(T) == 2 || MODE == kPagedRows)
        hipLaunchKernelGGL((shared_attention_kernel<T, 256, WHOLE, MODE>), dim3(grid), dim3(256), 0, s, p);
}
}  // namespace

hipError_t launch_shared_attention(const SharedAttnArgs& args, const SharedPlan& plan, hipStream_t s)
{
    SharedAttnArgs p = args;
    p.splits = plan.splits;
    p.split_min = plan.split_min;
    p.prefix_splits = plan.prefix_splits;
    p.prefix_min = plan.prefix_min;
    p.prefix_blocks = plan.prefix_blocks;
    p.prefix_grid = (int)plan.prefix_grid;
    p.blocks_grid = (int)plan.blocks_grid;
    p.few_rows = plan.few_rows;
    const unsigned grid = (unsigned)(plan.prefix_grid + plan.blocks_grid + plan.rows_grid);
    const bool whole = p.b.page.div % 16 == 0, both = plan.prefix_blocks || plan.blocks_grid;
    if (p.f16)
        (whole ? both ? launch_shared<_Float16, true, kPagedBoth> : launch_shared<_Float16, true, kPagedRows>
               : both ? launch_shared<_Float16, false, kPagedBoth> : launch_shared<_Float16, false, kPagedRows>)(p, grid, s);
    else
        (whole ? both ? launch_shared<float, true, kPagedBoth> : launch_shared<float, true, kPagedRows>
               : both ? launch_shared<float, false, kPagedBoth> : launch_shared<float, false, kPagedRows>)(p, grid, s);
    if (hipError_t e = hipGetLastError()) return e;
    const int64_t rows = (int64_t)p.b.tokens * p.H;
    hipLaunchKernelGGL(paged_merge_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, p);
    return hipGetLastError();
}

// ---- sampling ----------------------------------------------------------------------------------
namespace {
int64_t sample_row_bytes(int64_t chunks)
{
    return chunks * ((kSampleBins + kSampleListChunk + 3 * kSampleTiles + 1) * 8 + 24) + sizeof(SampleFound);
}
}  // namespace

SamplePlan sample_plan(int rows, int vocab, int cus)
{
    SamplePlan pl;
    pl.chunks = (vocab + 3 + kSampleChunk - 1) / kSampleChunk;   // (rows that begin up to 3 floats behind 16 bytes)
    pl.parts = (int64_t)rows * pl.chunks * 4 <= 2 * cus ? 4 : 1;
    // rows at a time: what fits 64 MB, and 64 at the least
    pl.batch = (int)std::min<int64_t>(rows, std::max<int64_t>(64, (64ll << 20) / sample_row_bytes(pl.chunks)));
    pl.ws_bytes = (pl.batch * sample_row_bytes(pl.chunks) + 15) / 16 * 16;
    return pl;
}

hipError_t launch_sample(const SampleArgs& p, const SamplePlan& plan, void* workspace, hipStream_t s)
{
    static_assert(kSampleChunk == kSampleTile * kSampleTiles && kSampleChunk < 1 << 15, "a chunk's counts have 15 bits");
    static_assert(sizeof(SampleFound) % 8 == 0, "the workspace's parts are aligned");
    SampleWs ws{};
    const int64_t n = plan.batch, c = n * plan.chunks;
    ws.chunks = plan.chunks;
    ws.parts = plan.parts;
    while ((1 << ws.index_bits) < p.vocab) ++ws.index_bits;
    ws.hist = static_cast<unsigned long long*>(workspace);
    ws.list = ws.hist + c * kSampleBins;
    ws.tiles = ws.list + c * kSampleListChunk;
    ws.sums = ws.tiles + c * kSampleTiles;
    ws.all = ws.sums + c * 2 * kSampleTiles;
    ws.found = reinterpret_cast<SampleFound*>(ws.all + c);
    ws.top = reinterpret_cast<float*>(ws.found + n);
    ws.first = reinterpret_cast<int32_t*>(ws.top + c);
    ws.listed = reinterpret_cast<uint32_t*>(ws.first + c);
    const int lds = (int)(sizeof(SampleLds) + plan.chunks * kSampleTiles * 8);
    if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(sample_draw_kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, lds))
        return e;
    for (; ws.row0 < p.rows; ws.row0 += plan.batch) {
        const int rows = std::min(plan.batch, p.rows - ws.row0);
        const dim3 grid(plan.chunks, rows), block(kSampleThreads);
        hipLaunchKernelGGL(sample_scan_kernel, grid, block, 0, s, p, ws);
        if (plan.parts == 1)
            hipLaunchKernelGGL(sample_sum_kernel<kSampleWaves>, grid, block, 0, s, p, ws);
        else
            hipLaunchKernelGGL(sample_sum_kernel<kSampleWaves / 4>, dim3(4 * plan.chunks, rows), dim3(kSampleThreads / 4), 0, s, p, ws);
        hipLaunchKernelGGL(sample_draw_kernel, dim3(rows), dim3(kDrawThreads), lds, s, p, ws);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace msnb
