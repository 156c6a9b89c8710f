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
    if (lds > 63 * 1024)   // beside the kernel's own; always the most there is, for calls of two threads
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(paged_plan_kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 2 * (kPlanRequests + 1) * 4))
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
    const int64_t grp = H / kvH, size = f16 ? 2 : 4, row_bytes = kvH * D * size * 2;
    // Shared where that leaves out 16 MB and more of keys and values (which lie in the caches all the same). us, alone
    // and shared: four requests behind 700 (1 MB) 9.8 and 10.9, eight tokens each behind 800 (5 MB) 11.4 and 11.6, two
    // chunks of 100 behind 8000 (16 MB) 76 and 72, four behind 3000 of 8 kv heads (37 MB) 15.1 and 12.8, 64 behind 500
    // (65 MB) 16.2 and 14.4, 64 behind 16000 (2 GB) 152 and 59.
    if (groups <= 0 || (double)(requests - groups) * prefix * row_bytes < 16 << 20) return pl;   // (bounds may be anything)
    const bool fit = f16 || D <= 128;   // an fp32 block's three parts in LDS
    pl.few_rows = f16 ? 64 : 128;
    // A prefix's rows by tiles of 128 or of 16, for all groups alike: a CU takes about 2400 rows by keys a us in the
    // larger, 1700 in the smaller, without 5 us of the larger ones' start. us, by 128 and by 16 at their best
    // splits: 32 single tokens of 28 / 4 heads behind 4000 26 and 21, 64 behind 16000 59 and 83, 64 of 16 / 2 heads of 256
    // behind 4000 46 and 43, four groups of 16 of 32 / 8 heads behind 8000 65 and 65, eight chunks of 64 behind 6000
    // 114 and 229. (fp32, page of 24: 24 and 27 for two groups of eight, 35 and 35 for 32 behind 4000.)
    const int64_t group_rows = (tokens * grp + groups - 1) / groups;
    const double work = (double)prefix * groups * kvH;
    const int64_t rows128 = (group_rows + 127) / 128 * 128, rows16 = (group_rows + 15) / 16 * 16;
    pl.prefix_blocks = fit && rows128 * work / 2400 + 5 * cus < rows16 * work / 1700;
    const int64_t far = tokens * grp / (pl.prefix_blocks ? 128 : 16) + groups;   // tiles at the most; likely
    const int64_t far_likely = groups * (pl.prefix_blocks ? rows128 / 128 : rows16 / 16);
    const bool few = max_new * grp <= pl.few_rows || !fit;
    const int64_t blocks = few ? 0 : tokens * grp / 128 + std::min<int64_t>(requests, tokens * grp / (pl.few_rows + 1) + 1);
    const int64_t tiles16 = tokens * grp / 16 + requests;
    const int64_t rows = few ? tiles16 : std::min<int64_t>(tiles16, (int64_t)requests * (pl.few_rows / 16));
    const int64_t near = few ? std::max<int64_t>(1, std::min(rows, (max_new * grp + 15) / 16 * requests))
                             : tokens * grp / 128 + 1 + std::min<int64_t>(requests, tokens);
    // A workgroup to a CU for tiles of 16 (32 tokens behind 4000 in 2, 4, 8 splits: 27, 21, 26 us), with 64 KB of keys
    // or more (four requests behind 3000 in 8, 12, 16: 14.1, 12.8, 15), and for the requests' own keys; 128 rows: two, or
    // one and a half beside single tokens (64 behind 16000 in 16, 24, 32: 68, 59, 69; chunks: in 2, 4, 8 147, 114, 128).
    auto count = [&](int64_t tiles, int64_t wgs, int64_t keys, int64_t bytes, int64_t most) {
        const int64_t n = std::max<int64_t>(1, tiles * kvH);
        return std::max<int64_t>(1, std::min<int64_t>({wgs / n, keys * D * size / bytes, most}));
    };
    pl.prefix_splits = (int)(pl.prefix_blocks ? count(far_likely, few ? 3 * cus / 2 : 2 * cus, prefix, 32 << 10, 48)
                                              : count(far_likely, cus, prefix, 64 << 10, 48));
    pl.splits = pl.prefix_splits + (int)count(near, cus, rest, 32 << 10, 16);
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
    // without tiles of 128 for the requests' own keys those of 16 take requests of any length (max_new may be too small)
    p.few_rows = plan.blocks_grid ? plan.few_rows : INT32_MAX;
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
    return chunks * ((kSampleBins + 3 * kSampleTiles + 1) * 8 + 8) + kSampleList * 8 + 8 + sizeof(SampleFound);
}
}  // namespace

SamplePlan sample_plan(int rows, int vocab)
{
    SamplePlan pl;
    pl.chunks = (vocab + 3 + kSampleChunk - 1) / kSampleChunk;   // (rows that begin up to 3 floats behind 16 bytes)
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
    while ((1 << ws.index_bits) < p.vocab) ++ws.index_bits;
    ws.hist = static_cast<unsigned long long*>(workspace);
    ws.list = ws.hist + c * kSampleBins;
    ws.tiles = ws.list + n * kSampleList;
    ws.sums = ws.tiles + c * kSampleTiles;
    ws.all = ws.sums + c * 2 * kSampleTiles;
    ws.found = reinterpret_cast<SampleFound*>(ws.all + c);
    ws.top = reinterpret_cast<float*>(ws.found + n);
    ws.first = reinterpret_cast<int32_t*>(ws.top + c);
    ws.listed = reinterpret_cast<uint32_t*>(ws.first + c);
    constexpr int kMostChunks = (kSampleVocab + 3 + kSampleChunk - 1) / kSampleChunk;
    constexpr int kMostLds = (int)sizeof(SampleLds) + kMostChunks * kSampleTiles * 8;
    static_assert(kMostLds <= 160 * 1024, "a CU's LDS");
    const int lds = (int)sizeof(SampleLds) + plan.chunks * kSampleTiles * 8;
    if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(sample_draw_kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds))
        return e;
    for (; ws.row0 < p.rows; ws.row0 += plan.batch) {
        const int rows = std::min(plan.batch, p.rows - ws.row0);
        const dim3 grid(plan.chunks, rows), block(kSampleThreads);
        hipLaunchKernelGGL(sample_scan_kernel, grid, block, 0, s, p, ws);
        const dim3 parts(kSampleParts * plan.chunks, rows);
        if (p.top_k || p.top_p) {
            hipLaunchKernelGGL(sample_find_kernel, dim3(rows), dim3(kFindThreads), 0, s, p, ws);
            hipLaunchKernelGGL(sample_sum_kernel<false>, parts, dim3(kSumWaves * kWave), 0, s, p, ws);
        } else {
            hipLaunchKernelGGL(sample_sum_kernel<true>, parts, dim3(kSumWaves * kWave), 0, s, p, ws);
        }
        hipLaunchKernelGGL(sample_draw_kernel, dim3(rows), dim3(kDrawThreads), lds, s, p, ws);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace msnb
