// serving.h — the operators of a serving step over many requests, kernels of a code object of
// their own (ms_hip_serving.hip; formats.h says why they are apart from the decode kernels):
//
//   paged_append.h      norms of queries and keys per head, rotation, append to a paged cache
//   paged_attention.h   attention of each request's new tokens over its pages
//   lora.h              low-rank adapters of many requests beside a shared projection
#pragma once
#include "formats.h"
#include "nbits_device.h"

namespace msnb {

// An fp32 value as two fp16 halves, the low one times 2^12 with a sum of its own: a half ulp of a
// high half below 2^15 becomes at most 2^15, and what is left of a value so small that its high
// half is subnormal keeps its bits.
constexpr int kLowExp = 12;
constexpr float kLow = 1.0f / (1 << kLowExp);

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery's round-up method):
// with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(n, m) + n) >> s.
struct FastDiv {
    uint32_t mul = 1;
    int shift = 0, div = 1;
    FastDiv() = default;
    explicit FastDiv(int d) : div(d)
    {
        while ((1ll << shift) < d) ++shift;
        mul = (uint32_t)(((uint64_t)((1ll << shift) - d) << 32) / (uint32_t)d + 1);
    }
    __host__ __device__ int quot(int n) const
    {
        const uint32_t hi = (uint32_t)(((uint64_t)(uint32_t)n * mul) >> 32);
        return (int)((hi + (uint32_t)n) >> shift);
    }
};

// Positions from here on have no page: 2^31 with a margin, so that a position and a few blocks of
// keys add up in 32 bits.
constexpr int kPagedPositions = 0x7ffff000;

// A batch of `requests` requests over one paged cache: request r's new tokens are rows
// [cu[r], cu[r + 1]) of the step's tensors, its position p lies in row table[r][p / page] * page
// + p % page of the cache. Entries outside [0, num_pages) hold nothing: their keys are masked
// and appends to them dropped. Lengths that make no sense (below zero, past the tensors' rows
// or the table) are cut to what is there (paged_span).
struct PagedBatch {
    const int32_t* cu;
    const int32_t* past;
    const int32_t* table;
    int tokens, requests, num_pages, max_pages;
    FastDiv page;
};

// A request's rows of the step's tensors from cu[r] and cu[r + 1], whatever those hold.
struct PagedSpan {
    int first, count;
};
__host__ __device__ inline PagedSpan paged_span(int c0, int c1, int tokens)
{
    const int first = c0 < 0 ? 0 : c0 > tokens ? tokens : c0, end = c1 < first ? first : c1 > tokens ? tokens : c1;
    return {first, end - first};
}

// Tiles of bm rows of `rows` rows; at most 2^24, as many workgroups as a launch can have (2^32
// threads), so that those of 64 requests add up in 32 bits even where senseless lengths overlap.
__host__ __device__ inline int paged_tiles(int rows, int bm)
{
    const uint32_t n = ((uint32_t)rows + bm - 1) / bm;
    return n < (1u << 24) ? (int)n : 1 << 24;
}

// The request that row t belongs to, or `requests` for a row behind the last: how many end at or
// before t, counted 64 at a time. Called by whole waves with a uniform t.
__device__ __forceinline__ int paged_request(const PagedBatch& b, int t)
{
    const int lane = threadIdx.x & (kWave - 1);
    int r = 0;
    for (int base = 0; base < b.requests; base += kWave) {
        const int i = base + lane;
        const bool done = i < b.requests && b.cu[min(i, b.requests - 1) + 1] <= t;
        r += __popcll(__ballot(done));
    }
    return r;
}

// Row of the cache that holds position pos of request r, or -1.
__device__ __forceinline__ int paged_row(const PagedBatch& b, int r, int pos)
{
    const int pg = b.page.quot(pos);
    if (pg >= b.max_pages) return -1;
    const int e = b.table[(int64_t)r * b.max_pages + pg];
    return (unsigned)e < (unsigned)b.num_pages ? e * b.page.div + (pos - pg * b.page.div) : -1;
}

// Sum of x over each aligned group of G lanes (8, 16, 32 or 64), in every lane of the group.
template <int G>
__device__ __forceinline__ float group_sum_all(float x)
{
    x += dpp_read<0xB1>(x);                           // quad_perm [1,0,3,2]
    x += dpp_read<0x4E>(x);                           // quad_perm [2,3,0,1]
    x += dpp_read<0x141>(x);                          // row_half_mirror
    if constexpr (G >= 16) x += dpp_read<0x140>(x);   // row_mirror
    if constexpr (G >= 32) x += xor16_value(x);
    if constexpr (G >= 64) x += xor32_value(x);
    return x;
}

struct AppendArgs {
    PagedBatch b;               // cu null: contiguous outputs and explicit positions
    const int32_t* positions;
    const float* q;
    const float* k;
    const float* v;
    const float* gq;            // norm weights [D], or null: no norm
    const float* gk;
    const float* cos;           // [cos_rows][half]
    const float* sin;
    float* q_out;               // [tokens, H * D]
    void* k_out;                // the cache, or [tokens, kvH * D]
    void* v_out;
    int H, kvH, D;
    int64_t q_stride, k_stride, v_stride;
    int rot_half, half, cos_rows, interleaved;
    float eps;
    int f16;                    // the cache's type
    int vec;                    // 16-byte loads and stores
};
MS_INTERNAL hipError_t launch_append(const AppendArgs& p, hipStream_t s);
constexpr int kAppendMaxDim = 1024;

struct PagedAttnArgs {
    PagedBatch b;
    const float* q;
    const void* kc;
    const void* vc;
    float* out;       // [tokens, H * D]
    float* part;      // splits > 1: [splits][tokens * H][D], then [splits][tokens * H] of (max, sum)
    int H, kvH, D, window, f16, splits;
    int split_min;    // keys of a split at the least
    int blocks_grid;  // workgroups of paged_blocks()
    int few_rows;     // rows of a request that paged_rows() takes where both kinds are launched
    int64_t q_stride;
    FastDiv grp;      // query heads per kv head
    float scale2;     // scale * log2(e)
};
struct PagedAttnPlan {
    int splits = 1, split_min = 0, few_rows = 0;
    int64_t rows_grid = 0, blocks_grid = 0;   // 0: that kernel is not launched
    int64_t ws_bytes = 0;
};
MS_INTERNAL PagedAttnPlan paged_attention_plan(int64_t tokens, int requests, int64_t max_new, int64_t keys, int H,
                                               int kvH, int D, int f16, int64_t ws_avail, int cus);
MS_INTERNAL hipError_t launch_paged_attention(const PagedAttnArgs& p, const PagedAttnPlan& plan, hipStream_t s);

struct LoraArgs {
    const float* x;           // [T, K]
    const void* a;            // [adapters, rank, K]
    const void* b;            // [adapters, N, rank]
    const int32_t* ranks;     // [adapters], or null: all of them `rank`
    const float* scales;      // [adapters], or null: 1
    const int32_t* which;     // [T]
    const float* base;        // [T, N], or null: zero
    float* y;                 // [T, N]
    float* h;                 // [splits][T][rank16]
    int T, K, N, adapters, rank, rank16, f16, splits;
    int vec_x, vec_y;         // whole chunks of x and A; of B, base and y (fours, or eights of B)
};
struct LoraPlan {
    int splits = 1;
    int slots = 1, shrink_slots = 1;   // workgroups that share out a tile's classes
    int subs = 1;                      // tiles of tokens to an expand workgroup
    bool many = false;
    int64_t ws_bytes = 0;
};
MS_INTERNAL LoraPlan lora_plan(int T, int K, int N, int adapters, int rank, int cus);
MS_INTERNAL hipError_t launch_lora(const LoraArgs& p, const LoraPlan& plan, hipStream_t s);

}  // namespace msnb
