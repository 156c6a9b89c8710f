// serving_loop.h — what a server's loop needs around a serving step's attention, kernels of a
// code object of their own (ms_hip_loop.hip; formats.h says why they are apart from the others):
//
//   paged_plan.h        page tables, lengths, positions and slot maps from what requests want, and
//                       the step's end
//   paged_attention.h   attention behind prefixes that requests share (shared_attention_kernel)
//   sample.h            the next tokens from logits
#pragma once
#include "serving.h"

namespace msnb {

constexpr int kPlanRequests = 8192;   // two cumulative lengths of each in LDS: 64 KB

struct PlanArgs {
    const int32_t* want;
    const int32_t* past;
    const int32_t* free;         // a stack of pages: [0, free_count)
    const int32_t* free_count;
    int32_t* table;
    int32_t* cu;
    int32_t* used;
    int32_t* request;            // [tokens]
    int32_t* position;
    int32_t* slot;
    int tokens, requests, num_pages, max_pages;
    FastDiv page;
};
MS_INTERNAL hipError_t launch_plan(const PlanArgs& p, int cus, hipStream_t s);

struct CommitArgs {
    const int32_t* cu;
    const int32_t* used;
    const int32_t* done;         // or null: none
    const int32_t* keep;         // or null: 0
    int32_t* past;
    int32_t* table;
    int32_t* free;
    int32_t* free_count;
    int requests, num_pages, max_pages;
    FastDiv page;
};
MS_INTERNAL hipError_t launch_commit(const CommitArgs& p, hipStream_t s);

struct SharedPlan {
    int splits = 0, prefix_splits = 0;   // records of a row, and the prefix's among them; 0: not shared
    int split_min = 0, prefix_min = 0, few_rows = 0;
    bool prefix_blocks = false;
    int64_t prefix_grid = 0, blocks_grid = 0, rows_grid = 0;
    int64_t ws_bytes = 0;
};
MS_INTERNAL SharedPlan shared_attention_plan(int64_t tokens, int requests, int64_t max_new, int groups, int64_t prefix,
                                             int64_t rest, int H, int kvH, int D, int f16, int cus);
MS_INTERNAL hipError_t launch_shared_attention(const SharedAttnArgs& p, const SharedPlan& plan, hipStream_t s);

struct SampleArgs {
    const float* logits;
    const float* temperature;    // [rows], or null: 1
    const int32_t* top_k;        // or null: all
    const float* top_p;          // or null: 1
    const float* min_p;          // or null: 0
    const float* random;
    int32_t* token;
    float* logprob;              // or null
    int rows, vocab, frac;       // weights are whole multiples of 2^-frac
    int64_t stride;
};
constexpr int kSampleBins = 512;                 // of logits, by which a border is first looked for
constexpr int kSampleList = 6144;                // logits of the bins that a border lies in, at most
constexpr int kSampleChunk = 8192;               // tokens of a workgroup of the first launch
constexpr int kSampleTiles = 8;                  // tiles of a chunk: what a wave sums
constexpr int kSampleParts = 2;                  // workgroups to a chunk of the launch that sums
// The weights of a row whose largest logit is `top`: 2^(scale (l - top)), and 0 below `low`.
struct SampleScale {
    double top, scale;
    float low;
};
// What is found out about a row from its bins.
struct SampleFound {
    SampleScale weights;
    unsigned long long least;  // lower weights are cut by m
    float top;
    int lo, hi, bk;            // bins: where the last token kept may lie, and the k-th token's (kSampleBins: none)
    int by_k, by_p;
    uint32_t k_before;         // tokens before bin bk
    int wide;                  // the bins say nothing
    int every;                 // the sums weigh each logit: p, without k, where the bins say something
    int answered;              // the row's answer is there
    float step, from, none, line, line_lo, line_hi, line_k, line_k_end;
};
// The workspace of `batch` rows: rows are taken so many at a time.
struct SampleWs {
    unsigned long long* hist;  // [rows][chunks][kSampleBins]
    unsigned long long* list;  // [rows][kSampleList]
    unsigned long long* tiles; // [rows][chunks][kSampleTiles]: a wave's kept weights
    unsigned long long* sums;  // [rows][chunks][kSampleTiles][2]
    unsigned long long* all;   // [rows][chunks]: the sum of a chunk's bins
    SampleFound* found;        // [rows]
    float* top;                // [rows][chunks]: largest logit
    int32_t* first;            // [rows][chunks]: its index
    uint32_t* listed;          // [rows]
    int row0, chunks, index_bits;
};
struct SamplePlan {
    int chunks = 0, batch = 0;
    int64_t ws_bytes = 0;
};
MS_INTERNAL SamplePlan sample_plan(int rows, int vocab);
MS_INTERNAL hipError_t launch_sample(const SampleArgs& p, const SamplePlan& plan, void* workspace, hipStream_t s);
constexpr int kSampleVocab = 1 << 22, kSampleRows = 1 << 20;
// Weights are at most 2^frac: no sum over the vocabulary passes 2^62.
inline int sample_frac(int vocab)
{
    int bits = 0;
    while ((1 << bits) < vocab) ++bits;
    return bits < 18 ? 44 : 62 - bits;
}

}  // namespace msnb
