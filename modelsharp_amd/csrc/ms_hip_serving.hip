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
namespace {
// Which cases paged_blocks() takes: an fp32 block's three parts fit LDS up to 128 channels.
bool blocks_fit(int D, int f16) { return f16 || D <= 128; }
}  // namespace

PagedAttnPlan paged_attention_plan(int64_t tokens, int requests, int64_t max_new, int64_t keys, int H, int kvH,
                                   int D, int f16, int64_t ws_avail, int cus)
{
    PagedAttnPlan pl;
    const int64_t grp = H / kvH;
    // Rows of a request up to which tiles of 16 rows take it, though each reads its keys. At 2000 cached
    // tokens of 28 / 4 heads of 128, fp16: 8 requests of 42 rows 19 us against 24 in tiles of 128, 32 of
    // 63 46 against 57; 32 of 126 80 against 64. An fp32 cache (32 / 8 heads), whose larger
    // tiles do six products a pair: 8 of 128 rows 72 against 94, 8 of 192 119 against 116. Where all tiles of
    // 16 leave CUs idle, further: one request of 126 rows 15.3 against 21.8, of 252 17.2 against 23.5.
    pl.few_rows = tokens * H <= 4 * (int64_t)cus ? 256 : f16 ? 64 : 128;
    const bool few = max_new * grp <= pl.few_rows || !blocks_fit(D, f16);   // as far as is known
    const bool one = requests == 1 && !few;
    // tiles at the most, and as many as the bounds make likely
    const int64_t blocks =
        few ? 0 : tokens * grp / 128 + std::min<int64_t>(requests, tokens * grp / (pl.few_rows + 1) + 1);
    const int64_t rows16 = tokens * grp / 16 + requests;
    const int64_t rows = one ? 0 : few ? rows16 : std::min<int64_t>(rows16, (int64_t)requests * (pl.few_rows / 16));
    const int64_t likely = few ? std::max<int64_t>(1, std::min(rows, (max_new * grp + 15) / 16 * requests))
                               : tokens * grp / 128 + 1 + (one ? 0 : std::min<int64_t>(requests, tokens));
    // Two workgroups to a CU, and as many splits of a tile's keys as pay for their join: of 32 KB of keys
    // up to 16, more only of 128 KB. One token of 28 / 4 heads of 128, fp16: 1000 cached ones in 7 splits
    // 10.8 us, in 3 12.1; 8000 in 16 13.0, in 31 13.6, in 62 15.8. fp32 (8 kv heads): 1000 in 15 12.5, in 7
    // 13.3; 4000 in 15 18.2, in 62 22.8; 64 tokens after 500 (96 channels) in 8 19.3, in 2 32.5. Up to 128 KB
    // a tile of 16 rows keeps its keys together, without the merge: 500 in one 9.8, in 3 10.8.
    const int64_t bytes = keys * D * (f16 ? 2 : 4);
    const int64_t most = few && bytes <= (128 << 10) ? 1 : std::max(std::min<int64_t>(bytes >> 15, 16), bytes >> 17);
    // (no more workgroups than a launch can have, should the bounds be far too small)
    const int64_t fit = ((1 << 24) - 1) / std::max<int64_t>(1, (rows + blocks) * kvH);
    int64_t splits = std::max<int64_t>(1, std::min<int64_t>({2 * (int64_t)cus / (likely * kvH), most, 64, fit}));
    const int64_t ws = splits > 1 ? splits * tokens * H * (D + 2) * (int64_t)sizeof(float) : 0;
    if (ws_avail >= 0 && ws > ws_avail) splits = 1;
    pl.splits = (int)splits;
    pl.split_min = (int)((keys + splits - 1) / splits);
    pl.ws_bytes = splits > 1 ? ws : 0;
    pl.rows_grid = rows * splits * kvH;
    pl.blocks_grid = blocks * splits * kvH;
    return pl;
}

namespace {
template <typename T, bool WHOLE, PagedMode MODE>
void launch_paged_t(const PagedAttnArgs& p, unsigned grid, hipStream_t s)
{
    constexpr bool kWide = sizeof(T) == 2 || MODE == kPagedRows;   // blocks_fit()
    if (p.D <= 64)
        hipLaunchKernelGGL((paged_attention_kernel<T, 64, WHOLE, MODE>), dim3(grid), dim3(256), 0, s, p);
    else if (MODE != kPagedRows && p.D <= 96)
        hipLaunchKernelGGL((paged_attention_kernel<T, MODE == kPagedRows ? 64 : 96, WHOLE, MODE>), dim3(grid), dim3(256), 0, s, p);
    else if (p.D <= 128)
        hipLaunchKernelGGL((paged_attention_kernel<T, 128, WHOLE, MODE>), dim3(grid), dim3(256), 0, s, p);
    else if constexpr (kWide)
        hipLaunchKernelGGL((paged_attention_kernel<T, 256, WHOLE, MODE>), dim3(grid), dim3(256), 0, s, p);
}

template <typename T, bool WHOLE>
void launch_paged(const PagedAttnArgs& p, const PagedAttnPlan& plan, hipStream_t s)
{
    const unsigned grid = (unsigned)(plan.blocks_grid + plan.rows_grid);
    if (!plan.blocks_grid)
        launch_paged_t<T, WHOLE, kPagedRows>(p, grid, s);
    else if (!plan.rows_grid)
        launch_paged_t<T, WHOLE, kPagedBlocks>(p, grid, s);
    else
        launch_paged_t<T, WHOLE, kPagedBoth>(p, grid, s);
}
}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& args, const PagedAttnPlan& plan, hipStream_t s)
{
    PagedAttnArgs p = args;
    p.blocks_grid = (int)plan.blocks_grid;
    p.few_rows = plan.few_rows;
    const bool whole = p.b.page.div % 16 == 0;
    const auto launch = p.f16 ? (whole ? launch_paged<_Float16, true> : launch_paged<_Float16, false>)
                              : (whole ? launch_paged<float, true> : launch_paged<float, false>);
    launch(p, plan, s);
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
    // Many tiles: x and A through LDS, a tile's classes and then K over workgroups only as long as CUs
    // would be idle, and as many tiles of tokens to an expand workgroup, which keeps B in registers across
    // them, as leave two workgroups to a CU. us, the other way first: K = N = 4096, 3 adapters of rank 16,
    // 200 tokens 14.4 against 11.3, 512 20.1 against 14.0, 1024 33 against 22; 16 of rank 16, a token each its
    // own, 64 tokens 15.7 against 18.0, 128 22.4 against 19.2, 512 65 against 36; 8 of rank 64 likewise, 64
    // 21.7 against 24.5, 128 28.9 against 32.2, 200 38 against 44.
    pl.many = tiles > cus / 32;
    if (pl.many) {
        const int nb = (N + kLoraRows - 1) / kLoraRows;
        while (pl.subs < tiles && (int64_t)((tiles + pl.subs - 1) / pl.subs) * nb > 2 * cus) ++pl.subs;
        const int groups = (rank + 31) / 32;
        pl.shrink_slots = std::max(1, std::min({kLoraTokens, adapters, cus / (tiles * groups)}));
        pl.splits = std::max(1, std::min({cus / (tiles * groups * pl.shrink_slots), (K + 511) / 512, 16}));
    } else {   // few: the classes side by side, and K over workgroups
        pl.slots = std::max(1, std::min({kLoraTokens, adapters + 1, 2 * cus / tiles}));
        pl.splits = std::max(1, std::min({2 * cus / (tiles * pl.slots), (K + 255) / 256, 16}));
        pl.shrink_slots = pl.slots;
    }
    pl.ws_bytes = (int64_t)pl.splits * T * ((rank + 15) / 16 * 16) * (int64_t)sizeof(float);
    return pl;
}

namespace {
template <typename T, int C, int CH, bool ONE>
void launch_expand(const LoraArgs& p, const LoraPlan& plan, hipStream_t s)
{
    const int tokens = kLoraTokens * plan.subs;
    const dim3 grid((p.T + tokens - 1) / tokens * plan.slots * ((p.N + kLoraRows - 1) / kLoraRows));
    const auto fn = !p.vec_y                  ? lora_expand_kernel<T, C, CH, ONE, 0>
                    : C == 16 || p.vec_y == 4 ? lora_expand_kernel<T, C, CH, ONE, 4>
                                              : lora_expand_kernel<T, C, CH, ONE, C == 16 ? 4 : 8>;
    hipLaunchKernelGGL(fn, grid, dim3(256), 0, s, p, plan.slots, plan.subs);
}

template <typename T, int RT, int WAVES, bool VEC>
void launch_shrink(const LoraArgs& p, const LoraPlan& plan, hipStream_t s)
{
    const int groups = (p.rank16 + 16 * RT - 1) / (16 * RT);
    const dim3 grid((p.T + kLoraTokens - 1) / kLoraTokens * groups * plan.shrink_slots * plan.splits);
    hipLaunchKernelGGL((lora_shrink_kernel<T, RT, WAVES, VEC>), grid, dim3(64 * WAVES), 0, s, p, plan.shrink_slots);
}

template <typename T, int RT>
hipError_t launch_shrink_lds(const LoraArgs& p, const LoraPlan& plan, hipStream_t s)
{
    constexpr int lds = lora_lds_bytes<T, RT>();
    const auto fn = lora_shrink_lds_kernel<T, RT>;
    if (lds > 64 * 1024)
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds))
            return e;
    const int groups = (p.rank16 + 16 * RT - 1) / (16 * RT);
    const dim3 grid((p.T + kLoraTokens - 1) / kLoraTokens * groups * plan.shrink_slots * plan.splits);
    hipLaunchKernelGGL(fn, grid, dim3(64 * kLoraLdsWaves), lds, s, p, plan.shrink_slots);
    return hipSuccess;
}

template <typename T, int C, int CH>
hipError_t launch_lora_c(const LoraArgs& p, const LoraPlan& plan, hipStream_t s)
{
    constexpr int RT = C / 16;
    if (!plan.many) {
        (p.vec_x ? launch_shrink<T, RT * CH, 4, true> : launch_shrink<T, RT * CH, 4, false>)(p, plan, s);
        launch_expand<T, C, CH, false>(p, plan, s);
        return hipGetLastError();
    }
    if (!p.vec_x)
        launch_shrink<T, RT, 16, false>(p, plan, s);
    else if (hipError_t e = launch_shrink_lds<T, RT>(p, plan, s))
        return e;
    (plan.splits == 1 ? launch_expand<T, C, CH, true> : launch_expand<T, C, CH, false>)(p, plan, s);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_lora_t(const LoraArgs& p, const LoraPlan& plan, hipStream_t s)
{
    const auto launch = p.rank16 == 16   ? launch_lora_c<T, 16, 1>
                        : p.rank16 == 32 ? launch_lora_c<T, 32, 1>
                                         : launch_lora_c<T, 32, 2>;
    return launch(p, plan, s);
}
}  // namespace

hipError_t launch_lora(const LoraArgs& p, const LoraPlan& plan, hipStream_t s)
{
    return p.f16 ? launch_lora_t<_Float16>(p, plan, s) : launch_lora_t<float>(p, plan, s);
}

}  // namespace msnb
