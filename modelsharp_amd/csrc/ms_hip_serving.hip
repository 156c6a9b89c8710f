// ms_hip_serving.hip — the launches declared in serving.h: a serving step's operators over many
// requests.
#include "serving.h"

#include <algorithm>

#include "lora.h"
#include "paged_append.h"
#include "paged_attention.h"

namespace msnb {

// ---- norms, rotation and append ----------------------------------------------------------------
hipError_t launch_append(const AppendArgs& p, hipStream_t s)
{
    const int slots = p.H + p.kvH * (p.b.cu ? 2 : 1), lanes = p.D / 8;
    if (p.vec && p.D % 8 == 0 && p.rot_half % 4 == 0 && lanes <= 64) {
        const int gs = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
        const dim3 grid(p.b.tokens, (slots + 256 / gs - 1) / (256 / gs));
        switch (gs) {
            case 8: hipLaunchKernelGGL(append_vec_kernel<8>, grid, dim3(256), 0, s, p); break;
            case 16: hipLaunchKernelGGL(append_vec_kernel<16>, grid, dim3(256), 0, s, p); break;
            case 32: hipLaunchKernelGGL(append_vec_kernel<32>, grid, dim3(256), 0, s, p); break;
            default: hipLaunchKernelGGL(append_vec_kernel<64>, grid, dim3(256), 0, s, p); break;
        }
    } else {
        hipLaunchKernelGGL(append_any_kernel, dim3(p.b.tokens, (slots + 3) / 4), dim3(256), 0, s, p);
    }
    return hipGetLastError();
}

// ---- attention over pages ----------------------------------------------------------------------
PagedAttnPlan paged_attention_plan(int64_t tokens, int requests, int64_t max_new, int64_t max_total, int H, int kvH,
                                   int D, int f16, int64_t ws_avail, int cus)
{
    PagedAttnPlan pl;
    const int grp = H / kvH;
    const int64_t tiles = tokens * grp / 16 + requests;
    const int64_t likely = std::max<int64_t>(1, std::min(tiles, (max_new * grp + 15) / 16 * (int64_t)requests)) * kvH;
    int64_t splits = std::max<int64_t>(1, 4 * (int64_t)cus / likely);
    splits = std::min<int64_t>({splits, std::max<int64_t>(1, max_total / 128), 64});
    const int64_t ws = splits > 1 ? splits * tokens * H * (D + 2) * (int64_t)sizeof(float) : 0;
    if (ws_avail >= 0 && ws > ws_avail) splits = 1;
    pl.splits = (int)splits;
    pl.ws_bytes = splits > 1 ? ws : 0;
    pl.grid = (int)std::min<int64_t>(tiles * splits * kvH, INT32_MAX);
    return pl;
}

namespace {
template <typename T>
void launch_rows(const PagedAttnArgs& p, int grid, hipStream_t s)
{
    if (p.D <= 64)
        hipLaunchKernelGGL((paged_rows_kernel<T, 64, 2>), dim3(grid), dim3(256), 0, s, p);
    else if (p.D <= 128)
        hipLaunchKernelGGL((paged_rows_kernel<T, 128, 2>), dim3(grid), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((paged_rows_kernel<T, 256, 1>), dim3(grid), dim3(256), 0, s, p);
}
}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& p, const PagedAttnPlan& plan, hipStream_t s)
{
    if (p.f16)
        launch_rows<_Float16>(p, plan.grid, s);
    else
        launch_rows<float>(p, plan.grid, s);
    if (hipError_t e = hipGetLastError()) return e;
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.b.tokens * p.H;
        hipLaunchKernelGGL(paged_merge_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, p);
    }
    return hipGetLastError();
}

// ---- low-rank adapters -------------------------------------------------------------------------
LoraPlan lora_plan(int T, int K, int N, int adapters, int rank, int cus)
{
    LoraPlan pl;
    const int tiles = (T + kLoraTokens - 1) / kLoraTokens;
    pl.slots = T <= 64 ? std::min(kLoraTokens, adapters + 1) : 1;
    pl.splits = std::max(1, std::min({2 * cus / (tiles * pl.slots), (K + 255) / 256, 16}));
    pl.ws_bytes = (int64_t)pl.splits * T * ((rank + 15) / 16 * 16) * (int64_t)sizeof(float);
    return pl;
}

namespace {
template <typename T>
void launch_lora_t(const LoraArgs& p, const LoraPlan& plan, hipStream_t s)
{
    const int tiles = (p.T + kLoraTokens - 1) / kLoraTokens;
    const dim3 shrink(tiles * plan.slots * plan.splits), expand(tiles * plan.slots * ((p.N + kLoraRows - 1) / kLoraRows));
    if (p.rank16 == 16)
        hipLaunchKernelGGL((lora_shrink_kernel<T, 1>), shrink, dim3(256), 0, s, p, plan.slots);
    else if (p.rank16 == 32)
        hipLaunchKernelGGL((lora_shrink_kernel<T, 2>), shrink, dim3(256), 0, s, p, plan.slots);
    else
        hipLaunchKernelGGL((lora_shrink_kernel<T, 4>), shrink, dim3(256), 0, s, p, plan.slots);
    hipLaunchKernelGGL(lora_expand_kernel<T>, expand, dim3(256), 0, s, p, plan.slots);
}
}  // namespace

hipError_t launch_lora(const LoraArgs& p, const LoraPlan& plan, hipStream_t s)
{
    if (p.f16)
        launch_lora_t<_Float16>(p, plan, s);
    else
        launch_lora_t<float>(p, plan, s);
    return hipGetLastError();
}

}  // namespace msnb
