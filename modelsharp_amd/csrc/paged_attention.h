// paged_attention.h — attention of each request's new tokens over its keys and values in a paged
// cache (fp32 or fp16), causal, with an optional sliding window:
//
//   out[t, h] = sum_j w_j V[row_j, g],   w = softmax(scale q_t,h . K[row_j, g]),
//   j in [max(0, pos - window + 1), pos],  pos = past[r] + t - cu[r],  g = h / (H / kvH)
//
// The query heads of a kv head and the tokens of a request are rows of one matrix, row = token
// * group + head in group, so that a tile of K and V serves every row that reads it.
#pragma once
#include <type_traits>

#include "mfma_device.h"
#include "serving.h"

namespace msnb {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));   // rows are 4-byte aligned

// A tile of at most BM rows of one request.
struct PagedTile {
    int r, t0, row0, rows;   // request, its first token, first row and rows of the tile
    int past;                // cached tokens
    int klast;               // last position of the request that the table reaches, -1: none
};

// Inclusive scan over the wave.
__device__ __forceinline__ int wave_scan(int x)
{
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(x, o);
        x += lane >= o ? y : 0;
    }
    return x;
}

// Tile `idx` of the requests of rows_min to rows_max rows in order, each one's tiles
// from its last (the longest range of keys) to its first; false past the end. Every wave by
// itself, with a uniform idx.
template <int BM>
__device__ __forceinline__ bool paged_tile(const PagedAttnArgs& p, int idx, int rows_min, int rows_max, PagedTile& t)
{
    const PagedBatch& b = p.b;
    const int lane = threadIdx.x & (kWave - 1);
    for (int base = 0; base < b.requests; base += kWave) {
        const int i = min(base + lane, b.requests - 1);
        const PagedSpan span = paged_span(b.cu[i], b.cu[i + 1], b.tokens);
        const int c0 = span.first, past = b.past[i], n = base + lane < b.requests ? span.count : 0;
        const int nr = n * p.grp.div;
        const int tiles = nr >= rows_min && nr <= rows_max ? paged_tiles(nr, BM) : 0;
        const int sum = wave_scan(tiles);
        const uint64_t past_idx = __ballot(sum > idx);
        if (past_idx) {
            const int l = __ffsll((unsigned long long)past_idx) - 1;
            const int nt = __builtin_amdgcn_readlane(tiles, l);
            const int within = idx - (__builtin_amdgcn_readlane(sum, l) - nt);
            const int nl = __builtin_amdgcn_readlane(n, l);
            t.r = base + l;
            t.t0 = __builtin_amdgcn_readlane(c0, l);
            t.row0 = (nt - 1 - within) * BM;
            t.rows = min(BM, nl * p.grp.div - t.row0);
            t.past = min(max(__builtin_amdgcn_readlane(past, l), 0), kPagedPositions - nl);
            t.klast = min((int64_t)t.past + nl, (int64_t)b.max_pages * b.page.div) - 1;
            return true;
        }
        idx -= __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return false;
}

// The row of the cache that keys without one stand for: the request's last key's, so that what
// nobody has written does not come in; the first where that has none either.
__device__ __forceinline__ int paged_stand(const PagedBatch& b, const PagedTile& t)
{
    return t.klast >= 0 ? max(paged_row(b, t.r, t.klast), 0) : 0;
}

// Positions [lo, hi] that some row of the tile sees; split `sp` takes [klo, khi] of them, in
// whole steps of `step`, all splits alike and split_min keys or more (so that short requests take
// fewer splits, not smaller ones). Empty where khi < klo.
struct PagedRange {
    int klo, khi;
};
// The keys that a tile's splits share out: positions from `lo` on, in records rec, rec + 1, ...
struct PagedPart {
    int splits, split_min, lo, rec;
};
__device__ __forceinline__ PagedRange paged_range(const PagedAttnArgs& p, const PagedPart& part, int pos0, int pos1, int klast,
                                                  int sp, int step)
{
    const int lo = max(part.lo, p.window >= 0 ? max(0, pos0 - p.window + 1) : 0), hi = min(pos1, klast);
    const int first = lo / step, n = hi >= lo ? hi / step - first + 1 : 0;
    const int per = max((n + part.splits - 1) / part.splits, part.split_min / step);
    if ((int64_t)sp * per >= n) return {0, -1};
    const int a = sp * per, e = min(n, a + per);
    return {max(lo, (first + a) * step), min(hi, (first + e) * step - 1)};
}

// Attention behind a shared prefix (SharedAttnArgs): tile `idx` of the groups' rows, all new tokens of
// a group's requests being rows of one matrix, each of which sees the whole prefix; or of the
// requests' own keys, from the prefix's end on. part.lo is where the keys begin.
template <int BM>
__device__ __forceinline__ bool shared_tile(const SharedAttnArgs& p, bool prefix, int idx, int rows_min, int rows_max,
                                            PagedTile& t, PagedPart& part)
{
    const PagedBatch& b = p.b;
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t reach = min((int64_t)b.max_pages * b.page.div, (int64_t)kSharedPositions);
    if (!prefix) {
        if (!paged_tile<BM>(p, idx, rows_min, rows_max, t)) return false;
        part.lo = 0;
        for (int base = 0; base < p.groups; base += kWave) {
            const int i = min(base + lane, p.groups - 1);
            const bool mine = p.bounds[i] <= t.r && t.r < p.bounds[i + 1];
            const int n = (int)min((int64_t)max(p.shared[i], 0), reach);
            if (const uint64_t found = __ballot(mine && base + lane < p.groups)) {
                part.lo = __builtin_amdgcn_readlane(n, __ffsll((unsigned long long)found) - 1);
                break;
            }
        }
        return true;
    }
    for (int base = 0; base < p.groups; base += kWave) {
        const int i = min(base + lane, p.groups - 1);
        const int r0 = min(max(p.bounds[i], 0), b.requests), r1 = min(max(p.bounds[i + 1], r0), b.requests);
        const PagedSpan span = paged_span(b.cu[r0], b.cu[r1], b.tokens);
        const int keys = (int)min((int64_t)max(p.shared[i], 0), reach);
        const int c0 = span.first, n = base + lane < p.groups && keys > 0 ? span.count : 0;
        const int tiles = paged_tiles(n * p.grp.div, BM);
        const int sum = wave_scan(tiles);
        if (const uint64_t past_idx = __ballot(sum > idx)) {
            const int l = __ffsll((unsigned long long)past_idx) - 1;
            const int nt = __builtin_amdgcn_readlane(tiles, l);
            t.r = __builtin_amdgcn_readlane(r0, l);
            t.t0 = __builtin_amdgcn_readlane(c0, l);
            t.row0 = (idx - (__builtin_amdgcn_readlane(sum, l) - nt)) * BM;
            t.rows = min(BM, __builtin_amdgcn_readlane(n, l) * p.grp.div - t.row0);
            t.past = __builtin_amdgcn_readlane(keys, l);   // every row's position is past the prefix's last
            t.klast = t.past - 1;
            part.lo = 0;
            return true;
        }
        idx -= __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return false;
}

// A split's record of an output row: its normed output, and (max, sum).
__device__ __forceinline__ float* paged_part_o(const PagedAttnArgs& p, int sp, int64_t row)
{
    return p.part + ((int64_t)sp * p.b.tokens * p.H + row) * p.D;
}
__device__ __forceinline__ float* paged_part_ml(const PagedAttnArgs& p, int sp, int64_t row)
{
    const int64_t n = (int64_t)p.b.tokens * p.H;
    return p.part + p.splits * n * p.D + (sp * n + row) * 2;
}

// The first `n` records of a row that has no keys there.
__device__ __forceinline__ void paged_no_prefix(const PagedAttnArgs& p, int n, int64_t row)
{
    for (int i = 0; i < n; ++i) {
        paged_part_ml(p, i, row)[0] = -__builtin_inff();
        paged_part_ml(p, i, row)[1] = 0.0f;
    }
}

__device__ __forceinline__ bool finite4(floatx4_t v)
{
    // an infinity or NaN times zero is NaN
    const float z = (v[0] * 0.0f + v[1] * 0.0f) + (v[2] * 0.0f + v[3] * 0.0f);
    return z == 0.0f;
}

// One row over positions [klo, khi] as the definition has it, by one wave: scores in fp32, their
// maximum, the sum of the weights, then each visible key's value by its weight. For what the
// matrix cores' sums cannot carry: infinities and NaN in places that some rows of a tile see and
// others do not (a product with a weight of zero would be NaN), scores that are all -infinity, pages
// that are not there. A split's record is (max, sum) with its normed output; no visible key: sum
// 0; every score -infinity: max -infinity, sum 1; a score that is NaN or +infinity: NaN.
template <typename T>
__device__ __forceinline__ void paged_exact_row(const PagedAttnArgs& p, const PagedTile& t, int g, int lr, int sp, PagedRange kr)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int row = t.row0 + lr, tok = p.grp.quot(row);
    const int head = g * p.grp.div + row - tok * p.grp.div;
    const int pos = t.past + tok;
    const int lo = max(kr.klo, p.window >= 0 ? max(0, pos - p.window + 1) : 0), hi = min(kr.khi, pos);
    const float* const q = p.q + (int64_t)(t.t0 + tok) * p.q_stride + (int64_t)head * p.D;
    const T* const kc = static_cast<const T*>(p.kc) + (int64_t)g * p.D;
    const T* const vc = static_cast<const T*>(p.vc) + (int64_t)g * p.D;
    const int64_t hs = (int64_t)p.kvH * p.D;
    auto score = [&](int rw) {
        typedef T unit_t __attribute__((ext_vector_type(8)));
        const T* const k = kc + rw * hs;
        float s = 0.0f;
        for (int d = 0; d < p.D; d += 8) {
            const unit_t x = *reinterpret_cast<const unit_t*>(k + d);
#pragma unroll
            for (int i = 0; i < 8; ++i) s = __builtin_fmaf(q[d + i], (float)x[i], s);
        }
        return s * p.scale2;
    };
    float m = -__builtin_inff();
    bool seen = false, bad = false;
    for (int k0 = lo; k0 <= hi && !bad; k0 += kWave) {   // a score that is NaN or +infinity decides
        const int k = k0 + lane, rw = k <= hi ? paged_row(p.b, t.r, k) : -1;
        if (rw >= 0) {
            const float s = score(rw);
            seen = true;
            bad = !(s < __builtin_inff());
            m = fmaxf(m, s);
        }
        bad = __ballot(bad) != 0;
    }
    m = row16_max_all(m);
    m = fmaxf(m, xor16_value(m));
    m = fmaxf(m, xor32_value(m));
    seen = __ballot(seen) != 0;
    const bool all_low = seen && !bad && m == -__builtin_inff();
    const bool sums = seen && !bad && !all_low;
    float l = 0.0f;
    if (sums)
        for (int k = lo + lane; k <= hi; k += kWave) {
            const int rw = paged_row(p.b, t.r, k);
            if (rw >= 0) l += __builtin_amdgcn_exp2f(score(rw) - m);
        }
    l = group_sum_all<64>(l);
    if (bad) {
        m = 0.0f;
        l = __builtin_nanf("");
    }
    if (all_low) l = 1.0f;
    const int64_t orow = (int64_t)(t.t0 + tok) * p.H + head;
    float* const o = p.splits > 1 ? paged_part_o(p, sp, orow) : p.out + orow * p.D;
    constexpr int kParts = 4, kAtOnce = 4;   // 64 channels each, up to 256; keys
    float acc[kParts];
#pragma unroll
    for (int c = 0; c < kParts; ++c) acc[c] = bad || (all_low && p.splits == 1) ? __builtin_nanf("") : 0.0f;
    if (sums)
        for (int k0 = lo; k0 <= hi; k0 += kWave) {
            const int k = k0 + lane, rw = k <= hi ? paged_row(p.b, t.r, k) : -1;
            const float w = rw >= 0 ? __builtin_amdgcn_exp2f(score(rw) - m) / l : 0.0f;
            for (int j0 = 0; j0 < min(kWave, hi - k0 + 1); j0 += kAtOnce) {
                float v[kAtOnce][kParts];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
                    for (int c = 0; c < kParts; ++c)
                        v[j][c] = (float)vc[max(__builtin_amdgcn_readlane(rw, j0 + j), 0) * hs + min(64 * c + lane, p.D - 1)];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j)
                    if (__builtin_amdgcn_readlane(rw, j0 + j) >= 0)
#pragma unroll
                        for (int c = 0; c < kParts; ++c) acc[c] = __builtin_fmaf(lane_value(w, j0 + j), v[j][c], acc[c]);
            }
        }
#pragma unroll
    for (int c = 0; c < kParts; ++c)
        if (64 * c + lane < p.D) o[64 * c + lane] = acc[c];
    if (p.splits > 1 && lane == 0) {
        paged_part_ml(p, sp, orow)[0] = m;
        paged_part_ml(p, sp, orow)[1] = l;
    }
}

template <typename T> struct PagedElem;
template <> struct PagedElem<_Float16> {
    static constexpr int kStep = 32;   // channels of one operand load of K over the wave
    typedef half8_t vec_t;
};
template <> struct PagedElem<float> {
    static constexpr int kStep = 16;
    typedef floatx4_t vec_t;
};

constexpr float kGrow = 4.0f;     // the running maximum moves in steps above 2^4
constexpr int kWeightExp = 11;    // weights times 2^11: at most 2^15 in fp16
// The low halves of weights and queries are summed apart (kLowExp): 22 bits down to 2^-25 of a row's
// largest weight (2^-28 of its largest query), then an error of 2^-48 (2^-51) of the largest. With one
// scale for both, bits went from 2^-14 on: 1.4e-3 of a row where weights of 2^-30 met values 2^25
// larger. The joins of the sums cost single tokens 0 to 5%, and chunks, whose products hardly run beside
// the vector unit, 7 to 17% (512 tokens of 28 / 4 heads of 128 over 16000 keys: 230-240 us before, 253-263
// now), at 256 channels 30%. Tried against it: the low halves' sums kept over all blocks spill (64 more
// registers at 128 channels), half of them kept gain 1%; a branch for queries without small values
// costs the products their order (286 us), scores that start from their low halves' sum 264.

// Steps of 16 keys in a wave's registers: the one in use and those on their way. A third for fp16 at
// D = 128 made no difference (47.1 against 46.2 us for 32 tokens over 1000-4000 keys).
constexpr int paged_ring(int DP, bool f16) { return f16 ? 2 : (DP <= 64 ? 3 : DP <= 128 ? 2 : 1); }

// Tiles of 16 rows: single tokens and short chunks. Four waves take every fourth step of 16
// keys each, the next steps' loads in flight meanwhile, with their own running maximum (moved in
// steps above 2^4, so that the sums are seldom rescaled) and sums, and meet in LDS at the end.
//
// S^T = K Q^T (keys M, rows N) leaves lane l with the scores of row l % 16 at keys 4 (l / 16) + i,
// i = 0 .. 3, and the same lane loads V's rows of those four keys, 8 (fp32: 4) channels of each:
// O^T += V^T P^T over 16 keys then has both operands where they are, the weights as they come and
// V's by packing the four keys of a channel (fp32: one key of each lane group per product). Neither
// passes through LDS, and V's rows come in as whole lines. K in fp16 meets the queries as two
// halves, q = 2^e (qh + ql) (22 bits; e by row, so that any fp32 query fits), V in fp16 the weights
// as two halves; an fp32 cache is multiplied in fp32.
// WHOLE: pages of a multiple of 16 rows, so that a step lies in one page: one lookup a step, and a
// page that is not there is a step left out.
//
// The cache's bytes bound it (16 keys of fp16, D = 128: 8 KB against 384 cycles of the matrix cores).
// 32 tokens over 1000-4000 keys of 4 heads of 128 in fp16, 171 MB: 42.7 us (4.0 TB/s), and 4.7 of merge;
// 8 over 2000-8000 of 8 heads in fp32, 340 MB: 68 us (5.0 TB/s) and 4.6. Between the two 169 MB cost
// 26 us: what does not grow with the keys is the larger part of a call of a few of them (the chain cu,
// past -> table -> keys, the join in LDS, the merge's launch).
constexpr int kRowsLds = 4 * 4 * kWave * 16 + 2 * 4 * 16 * 4 + 16;
template <typename T, int DP, bool WHOLE, typename A>
__device__ __forceinline__ void paged_rows(const A& p, PagedPart part, bool prefix, int bid, int rows_max, uint8_t* lds)
{
    constexpr bool SHARED = std::is_same<A, SharedAttnArgs>::value;
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int VEC = F16 && DP >= 128 ? 8 : 4;   // channels of one lane's load of V
    constexpr int NC = DP / (16 * VEC);             // loads of a V row's part
    constexpr int KS = DP / PagedElem<T>::kStep;    // loads of a K row's part
    constexpr int KV = F16 ? 8 : 4;                 // channels of one lane's load of K
    typedef typename PagedElem<T>::vec_t kvec_t;
    typedef T vvec_t __attribute__((ext_vector_type(VEC)));
    constexpr int kRing = paged_ring(DP, F16);
    auto& merge = *reinterpret_cast<floatx4_t(*)[4][4][kWave]>(lds);
    auto& stat = *reinterpret_cast<float(*)[2][4][16]>(lds + sizeof(merge));
    int& flag = *reinterpret_cast<int*>(lds + sizeof(merge) + sizeof(stat));

    const int g = bid % p.kvH, rest = bid / p.kvH;
    const int sp = rest % part.splits, rec = part.rec + sp;
    PagedTile t;
    if constexpr (SHARED) {
        if (!shared_tile<16>(p, prefix, rest / part.splits, 0, rows_max, t, part)) return;
    } else {
        if (!paged_tile<16>(p, rest / part.splits, 0, rows_max, t)) return;
    }
    const int lane = threadIdx.x & 63, grp = lane >> 4, l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (threadIdx.x == 0) flag = 0;

    const int row = t.row0 + min(l16, t.rows - 1), tok = p.grp.quot(row);
    const int head = g * p.grp.div + row - tok * p.grp.div;
    const int pos = t.past + tok;
    const PagedRange kr = paged_range(p, part, t.past + p.grp.quot(t.row0), t.past + p.grp.quot(t.row0 + t.rows - 1), t.klast,
                                      sp, 16);
    const int64_t orow = (int64_t)(t.t0 + tok) * p.H + head;
    const bool mine = l16 < t.rows;
    if constexpr (SHARED)
        if (!prefix && sp == 0 && part.lo == 0 && mine && threadIdx.x < 16) paged_no_prefix(p, part.rec, orow);
    if (p.splits > 1 && kr.khi < kr.klo) {   // nothing for this split: its record's sum is 0
        if (mine && threadIdx.x < 16) {
            paged_part_ml(p, rec, orow)[0] = -__builtin_inff();
            paged_part_ml(p, rec, orow)[1] = 0.0f;
        }
        return;
    }
    const int k_lo = max(kr.klo, p.window >= 0 ? max(0, pos - p.window + 1) : 0), k_hi = min(kr.khi, pos);

    // the queries' loads, then the first keys', before either is waited for
    const float* const q = p.q + (int64_t)(t.t0 + tok) * p.q_stride + (int64_t)head * p.D;
    float x[KS][KV];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int c = KV * grp + PagedElem<T>::kStep * s;
#pragma unroll
        for (int i = 0; i < KV / 4; ++i) {
            const floatx4_t v = c < p.D ? floatx4_t(*reinterpret_cast<const f4u_t*>(q + c + 4 * i)) : floatx4_t{};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[s][4 * i + e] = v[e];
        }
    }

    const int64_t hs = (int64_t)p.kvH * p.D;   // a cache row
    const T* const kc = static_cast<const T*>(p.kc) + (int64_t)g * p.D;
    const T* const vc = static_cast<const T*>(p.vc) + (int64_t)g * p.D;
    // where 16 keys lie: looked up a step before their loads. Keys past the request's last, and keys of
    // pages that are not there, stand for the last one; both are masked. (WHOLE: steps without a page
    // are left out, their loads any row's.)
    const int stand = WHOLE ? 0 : paged_stand(p.b, t);
    struct Rows {
        int first;     // WHOLE: the row of the step's first key, -1: not there
        int k, v[4];   // else: this lane's rows of K and V, -1: not there
    };
    auto look = [&](int key, Rows& r) {
        if constexpr (WHOLE) {
            r.first = paged_row(p.b, t.r, min(key, t.klast & ~15));
        } else {
            r.k = paged_row(p.b, t.r, min(key + l16, t.klast));
#pragma unroll
            for (int i = 0; i < 4; ++i) r.v[i] = paged_row(p.b, t.r, min(key + 4 * grp + i, t.klast));
        }
    };
    struct Keys {
        kvec_t k[KS];
        vvec_t v[4][NC];
        bool there[4];
    };
    auto load = [&](int key, const Rows& r, Keys& x) {
        if constexpr (WHOLE) {
            // one base for the step, 32-bit offsets within its 16 rows (65535 heads of 256: 1 GB)
            const char* const kb = reinterpret_cast<const char*>(kc + (int64_t)max(r.first, 0) * hs);
            const char* const vb = reinterpret_cast<const char*>(vc + (int64_t)max(r.first, 0) * hs);
            const uint32_t last = min(15, t.klast - key), w = (uint32_t)hs * sizeof(T);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int c = KV * grp + PagedElem<T>::kStep * s;
                x.k[s] = *reinterpret_cast<const kvec_t*>(kb + (min((uint32_t)l16, last) * w + (c < p.D ? c : 0) * (uint32_t)sizeof(T)));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x.there[i] = r.first >= 0;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int ch = VEC * (l16 + 16 * c);
                    x.v[i][c] = *reinterpret_cast<const vvec_t*>(
                        vb + (min((uint32_t)(4 * grp + i), last) * w + (ch < p.D ? ch : 0) * (uint32_t)sizeof(T)));
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int c = KV * grp + PagedElem<T>::kStep * s;
                x.k[s] = *reinterpret_cast<const kvec_t*>(kc + (r.k >= 0 ? r.k : stand) * hs + (c < p.D ? c : 0));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x.there[i] = r.v[i] >= 0;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int ch = VEC * (l16 + 16 * c);
                    x.v[i][c] = *reinterpret_cast<const vvec_t*>(vc + (r.v[i] >= 0 ? r.v[i] : stand) * hs + (ch < p.D ? ch : 0));
                }
            }
        }
    };
    // Every load of the ring is made, past the last step that one's again: behind a load under a
    // condition the compiler could only wait for all that is under way.
    int k0 = (kr.klo & ~15) + 16 * wave;
    const int k_end = kr.khi & ~15;
    const bool some = kr.khi >= kr.klo;
    Keys ring[kRing];
    Rows next;
    if (some) {
        look(min(k0, k_end), next);
#pragma unroll
        for (int n = 0; n + 1 < kRing; ++n) {
            load(min(k0 + 64 * n, k_end), next, ring[n]);
            look(min(k0 + 64 * (n + 1), k_end), next);
        }
    }

    kvec_t qh[KS], ql[F16 ? KS : 1];
    float fac = p.scale2;
    if constexpr (F16) {
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < KV; ++i) mx = fmaxf(mx, fabsf(x[s][i]));
        mx = fmaxf(mx, xor16_value(mx));
        mx = fmaxf(mx, xor32_value(mx));
        const int e = mx > 0.0f && mx < __builtin_inff() ? __builtin_amdgcn_frexp_expf(mx) - 15 : 0;
        fac = __builtin_amdgcn_ldexpf(p.scale2, e);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < KV; ++i) {
                const float v = __builtin_amdgcn_ldexpf(x[s][i], -e);
                qh[s][i] = (_Float16)v;
                ql[s][i] = (_Float16)((v - (float)qh[s][i]) * (1 << kLowExp));
            }
    } else {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < KV; ++i) qh[s][i] = x[s][i];
    }

    floatx4_t acc[NC][VEC], low[F16 ? NC : 1][F16 ? VEC : 1];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            acc[c][j] = floatx4_t{};
            if constexpr (F16) low[c][j] = floatx4_t{};
        }
    float m = -__builtin_inff(), l = 0.0f;

    // the keys that every row of the tile sees need no mask
    const int all_lo = max(kr.klo, p.window >= 0 ? t.past + p.grp.quot(t.row0 + t.rows - 1) - p.window + 1 : 0);
    const int all_hi = min(kr.khi, t.past + p.grp.quot(t.row0));
    auto add = [&](int key, const Keys& x) {
        if (WHOLE && !x.there[0]) return;
        floatx4_t s4{}, s4l{};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if constexpr (F16) {
                s4 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[s], qh[s], s4, 0, 0, 0);
                s4l = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[s], ql[s], s4l, 0, 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[s][e], qh[s][e], s4, 0, 0, 0);
            }
        }
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (F16 ? __builtin_fmaf(s4l[i], kLow, s4[i]) : s4[i]) * fac;
        if (!WHOLE || key < all_lo || key + 15 > all_hi)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = key + 4 * grp + i;
                w[i] = x.there[i] && k >= k_lo && k <= k_hi ? w[i] : -__builtin_inff();
            }
        float mt = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
        mt = fmaxf(mt, xor16_value(mt));
        mt = fmaxf(mt, xor32_value(mt));
        if (__ballot(mt > m + kGrow)) {
            const float mn = mt > m + kGrow ? mt : m;
            const float al = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    acc[c][j] *= al;
                    if constexpr (F16) low[c][j] *= al;
                }
        }
        // (scaled behind the exponential: an argument of 11 or more would be rounded to 2^-21)
        const float off = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = __builtin_amdgcn_exp2f(w[i] - off);
            l += w[i];
        }
        if constexpr (F16) {
            half4_t ph, pl;
#pragma unroll
            for (int i = 0; i < 4; ++i) ph[i] = (_Float16)(w[i] * (1 << kWeightExp));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                pl[i] = (_Float16)__builtin_fmaf((float)ph[i], -(float)(1 << kLowExp), w[i] * (1 << (kWeightExp + kLowExp)));
            typedef uint32_t dwords_t __attribute__((ext_vector_type(VEC / 2)));
            typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    uint32_t d[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[i] = __builtin_bit_cast(dwords_t, x.v[i][c])[j / 2];
                    const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;   // the high or the low halves of two dwords
                    const half4_t a = __builtin_bit_cast(half4_t, u32x2_t{__builtin_amdgcn_perm(d[1], d[0], sel),
                                                                          __builtin_amdgcn_perm(d[3], d[2], sel)});
                    acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x16f16(a, ph, acc[c][j], 0, 0, 0);
                    low[c][j] = __builtin_amdgcn_mfma_f32_16x16x16f16(a, pl, low[c][j], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[i][c][j], w[i], acc[c][j], 0, 0, 0);
        }
    };
    for (bool more = some && k0 <= kr.khi; more;) {
#pragma unroll
        for (int n = 0; n < kRing; ++n) {
            load(min(k0 + 64 * (kRing - 1), k_end), next, ring[(n + kRing - 1) % kRing]);
            look(min(k0 + 64 * kRing, k_end), next);
            add(k0, ring[n]);
            k0 += 64;
            if (!(more = k0 <= kr.khi)) break;
        }
    }

    // the waves' sums meet: statistics, then four quads of channels at a time
    l += xor16_value(l);
    l += xor32_value(l);
    if constexpr (F16) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[c][j][i] = __builtin_fmaf(low[c][j][i], kLow, acc[c][j][i]);
    }
    if (lane < 16) {
        stat[0][wave][lane] = m;
        stat[1][wave][lane] = l;
    }
    __syncthreads();
    float mm = stat[0][0][l16], ll = 0.0f;
#pragma unroll
    for (int w = 1; w < 4; ++w) mm = fmaxf(mm, stat[0][w][l16]);
    const float ms = mm == -__builtin_inff() ? 0.0f : mm;
#pragma unroll
    for (int w = 0; w < 4; ++w) ll += stat[1][w][l16] * __builtin_amdgcn_exp2f(stat[0][w][l16] - ms);
    // (a wave without a key that any row sees has m = -infinity: a factor of 0)
    const float f = ll != 0.0f ? __builtin_amdgcn_exp2f(m - ms) / (F16 ? ll * (1 << kWeightExp) : ll) : 0.0f;
    float* const o = p.splits > 1 ? paged_part_o(p, rec, orow) : p.out + orow * p.D;
    bool odd = mine && mm == -__builtin_inff() && k_hi >= k_lo;
    // quad n of a lane's channels: chunk c, row i of the product, channels 4 b .. 4 b + 3 of VEC
    constexpr int QUADS = DP / 16;
#pragma unroll
    for (int n0 = 0; n0 < QUADS; n0 += 4) {
#pragma unroll
        for (int n = n0; n < n0 + 4; ++n) {
            const int b = n % (VEC / 4), i = n / (VEC / 4) % 4, c = n / VEC;
            merge[wave][n - n0][lane] = floatx4_t{acc[c][4 * b][i] * f, acc[c][4 * b + 1][i] * f, acc[c][4 * b + 2][i] * f,
                                                  acc[c][4 * b + 3][i] * f};
        }
        __syncthreads();
        const int n = n0 + wave, b = n % (VEC / 4), i = n / (VEC / 4) % 4, c = n / VEC;
        const floatx4_t v = (merge[0][wave][lane] + merge[1][wave][lane]) + (merge[2][wave][lane] + merge[3][wave][lane]);
        const int ch = VEC * (4 * grp + i + 16 * c) + 4 * b;
        if (mine && ch < p.D) {
            *reinterpret_cast<f4u_t*>(o + ch) = v;
            odd |= !finite4(v);
        }
        __syncthreads();
    }
    if (p.splits > 1 && mine && wave == 0 && grp == 0) {
        paged_part_ml(p, rec, orow)[0] = mm;
        paged_part_ml(p, rec, orow)[1] = ll;
    }
    if (odd) flag = 1;
    __syncthreads();
    if (flag)
        for (int lr = wave; lr < t.rows; lr += 4) paged_exact_row<T>(p, t, g, lr, rec, kr);
}

// ---- chunks: tiles of 128 rows -----------------------------------------------------------------
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4_t lds_short4_t;

// How an operand's fp32 values are held for the 16-bit matrix cores.
//   fp16 cache: K and V are fp16 already; queries and weights, times 2^EXP, are two fp16 halves (22
//   bits), the low one times 2^12 (kLowExp): two products an operand pair, each with a sum of its own.
template <typename T> struct PagedSplit;
template <> struct PagedSplit<_Float16> {
    static constexpr int kPlanes = 1, kParts = 2, kSums = 2;   // of the cache; of queries and weights
    static constexpr int kProducts = 2;
    static constexpr int pair[kProducts][3] = {{0, 0, 0}, {0, 1, 1}};   // (plane, part, sum)
    template <int EXP>
    __device__ static __forceinline__ void part(const float (&x)[8], short8_t (&out)[2])
    {
        typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
        constexpr float scale = 1 << EXP, low = 1 << (EXP + kLowExp);
        u32x4_t h, l;
        // each half is one v_fma_mixlo_f16 or v_fma_mixhi_f16: scaled, subtracted, rounded
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[i] = pack(__builtin_fmaf(x[2 * i], scale, 0.0f), __builtin_fmaf(x[2 * i + 1], scale, 0.0f));
            const h2_t v = as_h2(h[i]);
            l[i] = pack(__builtin_fmaf((float)v.x, -(float)(1 << kLowExp), x[2 * i] * low),
                        __builtin_fmaf((float)v.y, -(float)(1 << kLowExp), x[2 * i + 1] * low));
        }
        out[0] = __builtin_bit_cast(short8_t, h);
        out[1] = __builtin_bit_cast(short8_t, l);
    }
    // two fp16 of a dword, kept whole by the opaque result
    __device__ static __forceinline__ uint32_t pack(float a, float b)
    {
        uint32_t r = as_u32(h2_t{(_Float16)a, (_Float16)b});
        asm("" : "+v"(r));
        return r;
    }
    __device__ static __forceinline__ floatx16_t mfma(short8_t a, short8_t b, floatx16_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    }
};

//   fp32 cache: everything is three bf16 parts, x = x0 + x1 + x2 exactly (cut, not rounded: 8 bits
//   each, and bf16 has fp32's range, so that any finite value fits), and the products of a pair
//   whose terms are 2^-16 or more of the whole: six of nine, what is left out is below 2^-22.
//   (The matrix cores take bf16 below 2^-126 as zero: values below 2^-110 keep fewer bits.)
template <> struct PagedSplit<float> {
    static constexpr int kPlanes = 3, kParts = 3, kSums = 1;
    static constexpr int kProducts = 6;
    static constexpr int pair[kProducts][3] = {{2, 0, 0}, {1, 1, 0}, {0, 2, 0}, {1, 0, 0}, {0, 1, 0}, {0, 0, 0}};   // small terms first
    template <int EXP>
    __device__ static __forceinline__ void part(const float (&x)[8], short8_t (&out)[3])
    {
        typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
        u32x4_t o[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t b[2][3];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float v = x[2 * i + e];
                b[e][0] = __float_as_uint(v);
                const float r1 = v - __uint_as_float(b[e][0] & 0xffff0000u);
                b[e][1] = __float_as_uint(r1);
                b[e][2] = __float_as_uint(r1 - __uint_as_float(b[e][1] & 0xffff0000u));
            }
#pragma unroll
            for (int k = 0; k < 3; ++k) o[k][i] = __builtin_amdgcn_perm(b[1][k], b[0][k], 0x07060302u);   // the high halves
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) out[k] = __builtin_bit_cast(short8_t, o[k]);
    }
    __device__ static __forceinline__ floatx16_t mfma(short8_t a, short8_t b, floatx16_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0, 0);
    }
};

// A tile of a block of keys in LDS: rows of CH chunks of 8 channels, K and V each with the chunks
// of a row moved about so that the reads below meet no bank twice: K's by ds_read_b128 down 32 rows
// of one chunk, V's by the transposing read, 4 rows of two chunks for 16 lanes.
template <int CH>
__device__ __forceinline__ int k_turn(int row)
{
    return CH == 8 ? (row >> 1) & 7 : row & 15;
}
template <int CH>
__device__ __forceinline__ int k_slot(int row, int c)
{
    return row * CH + (c ^ k_turn<CH>(row));
}
template <int CH>
__device__ __forceinline__ int v_turn(int row)
{
    return CH == 8 ? ((row >> 1) & 1) << 1 | ((row >> 2) & 1) << 2 : (row & 3) << 1 | ((row >> 2) & 1) << 3;
}

// Four waves of 32 rows each take blocks of BN keys through LDS, the next block's loads in flight
// meanwhile. S^T = K Q^T (keys M, rows N) leaves lane l with scores of row l % 32 at keys 8 (v / 4)
// + 4 (l / 32) + v % 4, and O^T += V^T P^T numbers its k-slots the same way, so the weights never
// leave their lane and a row's statistics are its lane's own; V^T comes from ds_read_b64_tr_b16, which
// hands 16 lanes four keys of one channel each. The online softmax runs in base 2 and moves
// its maximum only in steps above 2^4, so that the accumulators are seldom rescaled.
//
// 128 rows, since two such workgroups fill a CU's LDS (64 KB each at D = 128: two blocks of 64 keys) and
// registers, and each block of keys is then read from L2 once for 128 rows. The matrix cores and the vector
// unit, hardly beside each other, bound a long chunk: 512 tokens of 28 / 4 heads over 16000 keys take
// 253-263 us with the merge, 460 TFLOP/s of attention and twice that of products (a library product of
// 8192 reaches 1063). Fresh prompts of 200-650 tokens (46-47 us for five) are bound by the longest tile's
// chain of blocks. An fp32 cache, with six products a pair: two chunks of 300 tokens of 32 / 8 heads of
// 96, 1024 keys visible: 62 + 9 us.
// WHOLE: pages of a multiple of 16 rows, so that a wave's rows of a load lie in one page: its lookups
// are the scalar unit's.
template <typename T, int DP>
struct PagedBlock {
    static constexpr bool F16 = sizeof(T) == 2;
    static constexpr int DPL = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;   // channels of a row in LDS
    static constexpr int BN = F16 && DP <= 128 ? 64 : 32;               // keys
    static constexpr int BUFS = F16 ? 2 : 1;                            // fp32's parts leave room for one block
    static constexpr int CH = DPL / 8, TILE = BN * CH;                  // 16-byte slots of a row, of a plane
    typedef short8_t lds_t[BUFS][2][PagedSplit<T>::kPlanes][TILE];
};
template <typename T, int DP, bool WHOLE, typename A>
__device__ __forceinline__ void paged_blocks(const A& p, PagedPart part, bool prefix, int bid, int rows_min, uint8_t* lds_bytes)
{
    constexpr bool SHARED = std::is_same<A, SharedAttnArgs>::value;
    typedef PagedSplit<T> S;
    typedef PagedBlock<T, DP> B;
    constexpr bool F16 = B::F16;
    constexpr int BN = B::BN, BUFS = B::BUFS, CH = B::CH;
    constexpr int KS = DP / 16, NT = DP / 32, KT = BN / 32;
    constexpr int UN = BN * CH / 256;   // 8-channel units a thread moves of K, and of V
    // Two sums: so many tiles of scores and of channels at a time that the low halves' sums fit the
    // registers beside the rest (what is loaded ahead among it, unless it goes straight to LDS).
    constexpr bool FEW = S::kSums == 2 && !WHOLE;
    constexpr int KG = FEW ? 1 : KT, NG = S::kSums == 1 ? NT : FEW ? 1 : 2;
    auto& lds = *reinterpret_cast<typename B::lds_t*>(lds_bytes);

    const int g = bid % p.kvH, rest = bid / p.kvH;
    const int sp = rest % part.splits, rec = part.rec + sp;
    PagedTile t;
    if constexpr (SHARED) {
        if (!shared_tile<128>(p, prefix, rest / part.splits, rows_min, INT32_MAX, t, part)) return;
    } else {
        if (!paged_tile<128>(p, rest / part.splits, rows_min, INT32_MAX, t)) return;
    }
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PagedRange kr = paged_range(p, part, t.past + p.grp.quot(t.row0), t.past + p.grp.quot(t.row0 + t.rows - 1), t.klast,
                                      sp, BN);
    const int row = t.row0 + min(32 * wave + l32, t.rows - 1), tok = p.grp.quot(row);
    const int head = g * p.grp.div + row - tok * p.grp.div, pos = t.past + tok;
    const int64_t orow = (int64_t)(t.t0 + tok) * p.H + head;
    const bool mine = 32 * wave + l32 < t.rows;
    if constexpr (SHARED)
        if (!prefix && sp == 0 && part.lo == 0 && mine && hf == 0) paged_no_prefix(p, part.rec, orow);
    if (p.splits > 1 && kr.khi < kr.klo) {   // nothing for this split: its record's sum is 0
        if (mine && hf == 0) {
            paged_part_ml(p, rec, orow)[0] = -__builtin_inff();
            paged_part_ml(p, rec, orow)[1] = 0.0f;
        }
        return;
    }
    const int k_lo = max(kr.klo, p.window >= 0 ? max(0, pos - p.window + 1) : 0), k_hi = min(kr.khi, pos);
    // the wave's rows: positions pos_a .. pos_b, and what all of them or some of them see
    const int pos_a = t.past + p.grp.quot(t.row0 + min(32 * wave, t.rows - 1));
    const int pos_b = t.past + p.grp.quot(t.row0 + min(32 * wave + 31, t.rows - 1));
    const int all_lo = max(kr.klo, p.window >= 0 ? pos_b - p.window + 1 : 0), all_hi = min(kr.khi, pos_a);
    const int any_lo = max(kr.klo, p.window >= 0 ? pos_a - p.window + 1 : 0), any_hi = min(kr.khi, pos_b);

    // a thread's units of a block: unit u is chunk u % CH of row u / CH
    const int64_t hs = (int64_t)p.kvH * p.D;
    const T* const kc = static_cast<const T*>(p.kc) + (int64_t)g * p.D;
    const T* const vc = static_cast<const T*>(p.vc) + (int64_t)g * p.D;
    const int32_t* const table = p.b.table + (int64_t)t.r * p.b.max_pages;
    const int chunk = tid % CH, urow = tid / CH;
    constexpr int RU = 256 / CH, RW = 64 / CH;   // rows of a unit step over the workgroup and over a wave
    constexpr bool DIRECT = WHOLE && F16;        // straight from memory to LDS: fp16 needs no conversion
    const int ch = 8 * chunk < p.D ? 8 * chunk : 0;
    typedef T unit_t __attribute__((ext_vector_type(8)));
    unit_t kx[DIRECT ? 1 : UN], vx[DIRECT ? 1 : UN];
    // keys past the request's last stand for that one; they are masked
    int page[UN], slot[UN], ahead[UN];   // WHOLE: of the wave's first row, and how many rows follow up to the last key
    auto look = [&](int k0) {
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int r = RU * i + (WHOLE ? RW * wave : urow);
            const int key = min(k0 + r, WHOLE ? t.klast & ~(RW - 1) : t.klast), pg = p.b.page.quot(key);
            page[i] = table[pg];
            slot[i] = key - pg * p.b.page.div;
            ahead[i] = t.klast - key;
        }
    };
    bool missing = false;   // a page that some row of the tile sees and that is not there
    // the next block's loads: into registers, or into LDS buffer `buf`, where lane i of a load
    // fills slot i of its 64, so that the lanes fetch the chunks that belong there. Rows of a
    // page that is not there are the last key's; where a row of the tile sees them, the tile is done over,
    // below.
    const int stand = paged_stand(p.b, t);
    auto fetch = [&](int buf) {
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const bool there = (unsigned)page[i] < (unsigned)p.b.num_pages;
            const int64_t at = (int64_t)(there ? page[i] * p.b.page.div + slot[i] : stand) * hs;
            const int key = t.klast - ahead[i];   // a page that no row of the tile sees may be gone
            missing |= !there && key + (WHOLE ? RW - 1 : 0) >= kr.klo && key <= kr.khi;
            if constexpr (WHOLE) {   // a scalar base and 32-bit offsets
                const int last = there ? ahead[i] : 0;
                const uint32_t off = min(lane / CH, last) * (uint32_t)hs * (uint32_t)sizeof(T);
                if constexpr (DIRECT) {
                    const int bytes = (min(RW - 1, last) + 1) * (int)hs * (int)sizeof(T), r = RU * i + urow;
                    const int ck = 8 * (chunk ^ k_turn<CH>(r)), cv = 8 * (chunk ^ v_turn<CH>(r));
                    const uint32_t m0 = RU * CH * 16 * i + 1024 * wave;
                    lds_load16(buffer_rsrc(kc + at, bytes), off + 2 * (ck < p.D ? ck : 0), 0, lds_address(&lds[buf][0][0][0]) + m0);
                    lds_load16(buffer_rsrc(vc + at, bytes), off + 2 * (cv < p.D ? cv : 0), 0, lds_address(&lds[buf][1][0][0]) + m0);
                } else {
                    kx[i] = *reinterpret_cast<const unit_t*>(reinterpret_cast<const char*>(kc + at + ch) + off);
                    vx[i] = *reinterpret_cast<const unit_t*>(reinterpret_cast<const char*>(vc + at + ch) + off);
                }
            } else {
                kx[i] = *reinterpret_cast<const unit_t*>(kc + at + ch);
                vx[i] = *reinterpret_cast<const unit_t*>(vc + at + ch);
            }
        }
    };
    auto planes = [](const unit_t& x, short8_t (&out)[S::kPlanes]) {
        if constexpr (F16) {
            out[0] = __builtin_bit_cast(short8_t, x);
        } else {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = x[i];
            S::template part<0>(f, out);
        }
    };
    auto store = [&](int buf) {   // what fetch() brought is in LDS for every wave behind the next barrier
        if constexpr (DIRECT) {
            wait_vmcnt<0>();
            return;
        }
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int r = urow + 256 / CH * i;
            short8_t kp[S::kPlanes], vp[S::kPlanes];
            planes(kx[i], kp);
            planes(vx[i], vp);
#pragma unroll
            for (int pl = 0; pl < S::kPlanes; ++pl) {
                lds[buf][0][pl][k_slot<CH>(r, chunk)] = kp[pl];
                lds[buf][1][pl][r * CH + (chunk ^ v_turn<CH>(r))] = vp[pl];
            }
        }
    };

    const int first = kr.klo / BN * BN;
    const bool any = kr.khi >= kr.klo;
    if (any) {
        look(first);
        fetch(0);
        look(first + BN);
    }
    short8_t qx[KS][S::kParts];
    float fac = fabsf(p.scale2);
    {
        const float* const q = p.q + (int64_t)(t.t0 + tok) * p.q_stride + (int64_t)head * p.D;
        const float sign = p.scale2 < 0.0f ? -1.0f : 1.0f;
        float x[KS][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int c = 16 * s + 8 * hf;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const floatx4_t v = c < p.D ? floatx4_t(*reinterpret_cast<const f4u_t*>(q + c + 4 * i)) : floatx4_t{};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[s][4 * i + e] = v[e] * sign;
                    mx = fmaxf(mx, fabsf(v[e]));
                }
            }
        }
        if constexpr (F16) {   // every row's largest value into [2^14, 2^15)
            mx = fmaxf(mx, xor32_value(mx));
            const int e = mx > 0.0f && mx < __builtin_inff() ? __builtin_amdgcn_frexp_expf(mx) - 15 : 0;
            fac = __builtin_amdgcn_ldexpf(fac, e);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[s][i] = __builtin_amdgcn_ldexpf(x[s][i], -e);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) S::template part<0>(x[s], qx[s]);
    }


    floatx16_t acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = floatx16_t{};
    float m = -__builtin_inff(), l = 0.0f;

    if (any) store(0);
    __syncthreads();
    int buf = 0;
    for (int k0 = first; k0 <= kr.khi; k0 += BN) {
        const bool more = k0 + BN <= kr.khi;
        if (more) {
            fetch(buf ^ (BUFS - 1));
            look(k0 + 2 * BN);
        }
        if (k0 <= any_hi && k0 + BN > any_lo) {
            // (two sums: this wave's products go before the CU's other waves' exponentials, 2% of a long chunk)
            if constexpr (S::kSums == 2) __builtin_amdgcn_s_setprio(1);
            floatx16_t st[KT];
#pragma unroll
            for (int t0 = 0; t0 < KT; t0 += KG) {
                floatx16_t low[KG];
#pragma unroll
                for (int kt = 0; kt < KG; ++kt) st[t0 + kt] = low[kt] = floatx16_t{};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    short8_t a[S::kPlanes][KG];
#pragma unroll
                    for (int pl = 0; pl < S::kPlanes; ++pl)
#pragma unroll
                        for (int kt = 0; kt < KG; ++kt)
                            a[pl][kt] = lds[buf][0][pl][k_slot<CH>(32 * (t0 + kt) + l32, 2 * s + hf)];
#pragma unroll
                    for (int j = 0; j < S::kProducts; ++j)
#pragma unroll
                        for (int kt = 0; kt < KG; ++kt) {
                            floatx16_t& sum = S::pair[j][2] ? low[kt] : st[t0 + kt];
                            sum = S::mfma(a[S::pair[j][0]][kt], qx[s][S::pair[j][1]], sum);
                        }
                }
                if constexpr (S::kSums == 2) {
                    if (t0 + KG == KT) __builtin_amdgcn_s_setprio(0);
#pragma unroll
                    for (int kt = 0; kt < KG; ++kt)
#pragma unroll
                        for (int v = 0; v < 16; ++v) st[t0 + kt][v] = __builtin_fmaf(low[kt][v], kLow, st[t0 + kt][v]);
                }
            }
            if (k0 < all_lo || k0 + BN - 1 > all_hi)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const int key = k0 + 32 * kt + 8 * (v >> 2) + 4 * hf + (v & 3);
                        st[kt][v] = key >= k_lo && key <= k_hi ? st[kt][v] : -__builtin_inff();
                    }
            float mx = -__builtin_inff();
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int v = 0; v < 16; ++v) mx = fmaxf(mx, st[kt][v]);
            mx = fmaxf(mx, xor32_value(mx)) * fac;
            if (__ballot(mx > m + kGrow)) {
                const float mn = mx > m + kGrow ? mx : m;
                const float al = mn == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= al;
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[n] *= al;
            }
            // (fp16's scale comes behind the exponential: an argument of 11 or more would be rounded to 2^-21)
            const float off = m == -__builtin_inff() ? 0.0f : -m;
            short8_t px[2 * KT][S::kParts];
#pragma unroll
            for (int n0 = 0; n0 < NT; n0 += NG) {
                floatx16_t low[NG];
#pragma unroll
                for (int n = 0; n < NG; ++n) low[n] = floatx16_t{};
#pragma unroll
                for (int s = 0; s < 2 * KT; ++s) {
                    if (n0 == 0) {
                        float w[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[s >> 1][8 * (s & 1) + j], fac, off));
                            l += w[j];
                        }
                        S::template part<kWeightExp>(w, px[s]);
                    }
#pragma unroll
                    for (int n = n0; n < min(n0 + NG, NT); ++n) {
                        // rows 16 s + 8 e + 4 hf + i / 4, 16 channels of 8-byte quarters of two chunks
                        const int i = lane & 15;
                        short8_t a[S::kPlanes];
#pragma unroll
                        for (int pl = 0; pl < S::kPlanes; ++pl)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int r = 16 * s + 8 * e + 4 * hf + (i >> 2);
                                const int c = 4 * n + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
                                const short4_t h = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (lds_short4_t*)((short4_t*)&lds[buf][1][pl][r * CH + (c ^ v_turn<CH>(r))] + (i & 1)));
#pragma unroll
                                for (int x = 0; x < 4; ++x) a[pl][4 * e + x] = h[x];
                            }
#pragma unroll
                        for (int j = 0; j < S::kProducts; ++j) {
                            floatx16_t& sum = S::pair[j][2] ? low[n - n0] : acc[n];
                            sum = S::mfma(a[S::pair[j][0]], px[s][S::pair[j][1]], sum);
                        }
                    }
                }
                if constexpr (S::kSums == 2)
#pragma unroll
                    for (int n = n0; n < min(n0 + NG, NT); ++n)
#pragma unroll
                        for (int v = 0; v < 16; ++v) acc[n][v] = __builtin_fmaf(low[n - n0][v], kLow, acc[n][v]);
            }
        }
        if constexpr (BUFS == 2)
            buf ^= 1;
        else
            __syncthreads();
        if (more) store(buf);
        __syncthreads();
    }

    int* const said = reinterpret_cast<int*>(lds);   // the blocks are done with
    if (const bool any_missing = __ballot(missing); lane == 0) said[wave] = any_missing;
    __syncthreads();
    missing = said[0] | said[1] | said[2] | said[3];

    l += xor32_value(l);
    const float f = l != 0.0f ? 1.0f / (F16 ? l * (1 << kWeightExp) : l) : 0.0f;
    float* const o = p.splits > 1 ? paged_part_o(p, rec, orow) : p.out + orow * p.D;
    bool odd = mine && (missing || (m == -__builtin_inff() && k_hi >= k_lo));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const floatx4_t v = floatx4_t{acc[n][4 * b], acc[n][4 * b + 1], acc[n][4 * b + 2], acc[n][4 * b + 3]} * f;
            const int c = 32 * n + 8 * b + 4 * hf;
            if (mine && c < p.D) {
                *reinterpret_cast<f4u_t*>(o + c) = v;
                odd |= !finite4(v);
            }
        }
    if (p.splits > 1 && mine && hf == 0) {
        paged_part_ml(p, rec, orow)[0] = m;
        paged_part_ml(p, rec, orow)[1] = l;
    }
    // rows that met an infinity, a NaN or a page that is not there
    uint64_t redo = __ballot(odd);
    for (uint32_t rows = (uint32_t)(redo | redo >> 32); rows; rows &= rows - 1)
        paged_exact_row<T>(p, t, g, 32 * wave + __ffs(rows) - 1, rec, kr);
}

// A launch's workgroups: the first p.blocks_grid take tiles of 128 rows of the requests of more than
// p.few_rows rows (the longest work first), the others tiles of 16 rows of the rest, beside them:
// one is bound by the matrix cores, the other by memory. Without the one or the other kind the
// kind that is there takes every request.
enum PagedMode { kPagedRows, kPagedBlocks, kPagedBoth };
template <typename T, int DP, bool WHOLE, PagedMode MODE>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void paged_attention_kernel(PagedAttnArgs p)
{
    constexpr int DPR = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;
    constexpr int kBlocksLds = MODE == kPagedRows ? 0 : (int)sizeof(typename PagedBlock<T, DP>::lds_t);
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBlocksLds > kRowsLds ? kBlocksLds : kRowsLds];
    const PagedPart part{p.splits, p.split_min, 0, 0};
    if constexpr (MODE == kPagedRows) {
        paged_rows<T, DPR, WHOLE>(p, part, false, blockIdx.x, INT32_MAX, lds);
    } else if constexpr (MODE == kPagedBlocks) {
        paged_blocks<T, DP, WHOLE>(p, part, false, blockIdx.x, 0, lds);
    } else {
        if ((int)blockIdx.x < p.blocks_grid)
            paged_blocks<T, DP, WHOLE>(p, part, false, blockIdx.x, p.few_rows + 1, lds);
        else
            paged_rows<T, DPR, WHOLE>(p, part, false, blockIdx.x - p.blocks_grid, p.few_rows, lds);
    }
}

// Attention behind shared prefixes: the prefixes' tiles first (128 rows, or 16), then those of the requests'
// own keys, all of a launch beside each other. MODE as above; both kinds where either has both. A prefix's keys
// are read once for all rows of a tile instead of once for each request: 64 tokens of 28 / 4 heads behind 16,000
// shared keys 59 us with the merge (152 by themselves), bound by the products of tiles of 128 rows; 32 behind
// 4000 21 us, in tiles of 16.
template <typename T, int DP, bool WHOLE, PagedMode MODE>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void shared_attention_kernel(SharedAttnArgs p)
{
    constexpr int DPR = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;
    constexpr int kBlocksLds = MODE == kPagedRows ? 0 : (int)sizeof(typename PagedBlock<T, DP>::lds_t);
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBlocksLds > kRowsLds ? kBlocksLds : kRowsLds];
    const bool prefix = (int)blockIdx.x < p.prefix_grid;
    const int bid = blockIdx.x - (prefix ? 0 : p.prefix_grid);
    const PagedPart part = prefix ? PagedPart{p.prefix_splits, p.prefix_min, 0, 0}
                                  : PagedPart{p.splits - p.prefix_splits, p.split_min, 0, p.prefix_splits};
    if constexpr (MODE == kPagedRows) {
        paged_rows<T, DPR, WHOLE>(p, part, prefix, bid, INT32_MAX, lds);
    } else {
        if (prefix ? p.prefix_blocks : bid < p.blocks_grid)
            paged_blocks<T, DP, WHOLE>(p, part, prefix, bid, prefix ? 0 : p.few_rows + 1, lds);
        else
            paged_rows<T, DPR, WHOLE>(p, part, prefix, bid - (prefix ? 0 : p.blocks_grid), prefix ? INT32_MAX : p.few_rows, lds);
    }
}

// The splits' records of one output row, joined in the splits' order. A wave per row: lane s holds
// split s's weight, and the outputs' loads do not wait for them (what a split of weight zero left
// is not used).
static __global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs p)
{
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= (int64_t)p.b.tokens * p.H) return;
    const int tok = (int)(row / p.H);
    const int c0 = p.b.cu[0], c1 = p.b.cu[p.b.requests];
    const float* const ml = paged_part_ml(p, min(lane, p.splits - 1), row);
    float m = ml[0], l = lane < p.splits ? ml[1] : 0.0f;
    constexpr int kAtOnce = 8;
    const float* const part = paged_part_o(p, 0, row);
    const int64_t step = (int64_t)p.b.tokens * p.H * p.D;
    if (l == 0.0f) m = -__builtin_inff();
    float mx = row16_max_all(m);
    mx = fmaxf(mx, xor16_value(mx));
    mx = fmaxf(mx, xor32_value(mx));
    // every score -infinity wherever there was a key: the definition's NaN
    const bool low = mx == -__builtin_inff() && __ballot(l != 0.0f);
    float w = m == -__builtin_inff() ? 0.0f : l * __builtin_amdgcn_exp2f(m - mx);
    const float sum = group_sum_all<64>(w);
    w = sum != 0.0f ? w / sum : 0.0f;   // NaN stays
    for (int cw = 0; cw < p.D; cw += 4 * kWave) {   // uniform: the weights are read across lanes
        const int c = min(cw + 4 * lane, p.D - 4);
        floatx4_t o{};
        for (int s0 = 0; s0 < p.splits; s0 += kAtOnce) {
            floatx4_t v[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                v[i] = *reinterpret_cast<const floatx4_t*>(part + min(s0 + i, p.splits - 1) * step + c);
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (const float ws = s0 + i < p.splits ? lane_value(w, s0 + i) : 0.0f; ws != 0.0f) o += ws * v[i];
        }
        if (low) o = floatx4_t{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        if (cw + 4 * lane < p.D && tok >= c0 && tok < c1)   // rows of no request stay
            *reinterpret_cast<f4u_t*>(p.out + row * p.D + c) = o;
    }
}

}  // namespace msnb
