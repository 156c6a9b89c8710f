// sample.h — the next token of each row of logits l from a given random number u:
//
//   w_i = exp((l_i - max l) / t), tokens in order of falling logits, ties by rising index;
//   kept: the first k; of these the fewest whose sum of w is at least p of theirs; of these the ones
//   with w >= m (the likeliest always);  token = the first i, by index, with
//   sum of the kept w_j, j <= i, above u W, W the sum of all kept w;  logprob = log(w / W)
//
// Every limit keeps a prefix of the same order, so that one border (a logit and an index) says
// which tokens are left. A token drawn must not depend on how a sum was rounded: weights are computed in
// 64 bits and held as whole multiples of 2^-frac (frac 44 up to 2^18 tokens, so that no sum passes 2^62),
// and sums of whole numbers are exact in any order. In fp32 a sum over 150,000 tokens is off by 1e-7 and
// more, the distance of two neighbours in it.
#pragma once
#include "serving_loop.h"

namespace msnb {

typedef unsigned long long u64;

// A logit as the order has it: NaN as -infinity, -0 as 0.
__device__ __forceinline__ float sample_logit(float l) { return l != l ? -__builtin_inff() : l + 0.0f; }

// Ascending in the order: falling logits, then rising indexes.
__device__ __forceinline__ uint32_t sample_key(float l)
{
    const uint32_t b = __float_as_uint(l);
    return ~(b ^ ((int32_t)b < 0 ? ~0u : 0x80000000u));
}
__device__ __forceinline__ float sample_unkey(uint32_t k)
{
    const uint32_t b = ~k;
    return __uint_as_float(b ^ ((int32_t)b < 0 ? 0x80000000u : ~0u));
}
// A logit and its index in one number, the index in the low `bits`.
__device__ __forceinline__ u64 sample_place(float l, int i, int bits) { return (u64)sample_key(l) << bits | (uint32_t)i; }

// 2^y by 2^k 2^f, k the nearest whole number, f in [-1/2, 1/2] by the series of e^(f ln 2) up to the
// eleventh power (the next term is below 2^-46), in multiples of 2^-frac; 0 from y = -64 down and for NaN.
__device__ __forceinline__ u64 sample_exp2(double y, int frac)
{
    constexpr double c[12] = {1.0,
                              0.69314718055994530942,      // ln(2)^n / n!
                              0.24022650695910071233,
                              0.055504108664821579953,
                              0.0096181291076284771620,
                              0.0013333558146428443423,
                              0.00015403530393381609954,
                              1.5252733804059840280e-5,
                              1.3215486790144309488e-6,
                              1.0178086009239699728e-7,
                              7.0549116208011233299e-9,
                              4.4455382718708114976e-10};
    const bool some = y > -64.0;
    y = some ? y : 0.0;
    const double k = __builtin_rint(y), f = y - k;
    double s = c[11];
#pragma unroll
    for (int n = 10; n >= 0; --n) s = __builtin_fma(s, f, c[n]);
    // below 2^52 the sum's low bits are the whole number, rounded
    const u64 w = __builtin_bit_cast(u64, __builtin_ldexp(s, (int)k + frac) + 0x1p52) & ((1ull << 52) - 1);
    return some ? w : 0;
}

// What a row's settings say.
struct SampleRow {
    double scale;    // log2(e) / t
    float t, p, m, u;
    int k;
    bool greedy;
};
__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, int r)
{
    SampleRow s;
    s.t = a.temperature ? a.temperature[r] : 1.0f;
    s.greedy = !(s.t > 0.0f);
    s.scale = 1.4426950408889634074 / (double)s.t;
    const int k = a.top_k ? a.top_k[r] : 0;
    s.k = k <= 0 || k > a.vocab ? a.vocab : k;
    s.p = a.top_p ? a.top_p[r] : 1.0f;
    s.m = a.min_p ? a.min_p[r] : 0.0f;
    s.u = a.random[r];
    return s;
}
__device__ __forceinline__ u64 sample_weight(float l, float top, const SampleRow& s, int frac)
{
    // (a difference from an infinite largest is -infinity, and so is that from a logit of -infinity)
    const u64 w = sample_exp2(((double)l - (double)top) * s.scale, frac);
    return l == top ? 1ull << frac : w;
}
// The least whole number a sum has to reach to be at least x of w, and the largest it must pass to be above it.
__device__ __forceinline__ u64 sample_part(float x, u64 w, bool up)
{
    if (!(x > 0.0f)) return up ? 1 : 0;
    const double y = (double)x * (double)w;
    const double z = up ? __builtin_ceil(y) : __builtin_floor(y);
    if (z >= (double)w) return up ? w : w - 1;
    const u64 n = (u64)z;
    return up ? (n ? n : 1) : n;
}
// Weights below it are cut by m (m above 1 keeps the likeliest, as 1 does).
__device__ __forceinline__ u64 sample_least(const SampleRow& s, int frac)
{
    return s.m > 0.0f ? (u64)__builtin_rint(__builtin_ldexp((double)fminf(s.m, 1.0f), frac)) : 0;
}

// e^(d / t) in fp32, to 2^-17 of it where it counts; where d and t are infinite, 0
__device__ __forceinline__ float sample_rough(float d, float scale) { return fmaxf(__builtin_amdgcn_exp2f(d * scale), 0.0f); }

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / kWave;
constexpr int kSampleTile = 4 * kSampleThreads, kSampleTiles = 4;   // tokens of a tile; tiles of a chunk
constexpr int kSampleDigit = 11;                                     // bits of a border found at a time

// A 64-bit value moved by one DPP control; lanes whose source is outside the row, or whose row the mask leaves
// out, read 0.
template <int CTRL, int ROW_MASK, typename T>
__device__ __forceinline__ T dpp64(T x)
{
    const u64 b = __builtin_bit_cast(u64, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROW_MASK, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROW_MASK, 0xF, false);
    return __builtin_bit_cast(T, (u64)hi << 32 | lo);
}
// Inclusive sums over the wave of whole numbers or doubles.
template <typename T>
__device__ __forceinline__ T wave_scan64(T x)
{
    x += dpp64<0x111, 0xF>(x);   // row_shr:1
    x += dpp64<0x112, 0xF>(x);
    x += dpp64<0x114, 0xF>(x);
    x += dpp64<0x118, 0xF>(x);
    x += dpp64<0x142, 0xA>(x);   // row_bcast:15 -> rows 1, 3
    return x + dpp64<0x143, 0xC>(x);   // row_bcast:31 -> rows 2, 3
}
// Sums over the workgroup, in every thread.
template <int N>
__device__ __forceinline__ void block_sums(u64 (&x)[N], u64* scratch)
{
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = wave_scan64(x[n]);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == kWave - 1)
#pragma unroll
        for (int n = 0; n < N; ++n) scratch[n * kSampleWaves + (threadIdx.x >> 6)] = x[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        x[n] = 0;
#pragma unroll
        for (int w = 0; w < kSampleWaves; ++w) x[n] += scratch[n * kSampleWaves + w];
    }
}
__device__ __forceinline__ float block_max(float x, u64* scratch)
{
    x = row16_max_all(x);
    x = fmaxf(x, xor16_value(x));
    x = fmaxf(x, xor32_value(x));
    __syncthreads();
    float* const s = reinterpret_cast<float*>(scratch);
    if ((threadIdx.x & (kWave - 1)) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    x = s[0];
#pragma unroll
    for (int w = 1; w < kSampleWaves; ++w) x = fmaxf(x, s[w]);
    return x;
}
// Inclusive sums of x over the workgroup's threads.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T* scratch)
{
    const int wave = threadIdx.x >> 6;
    x = wave_scan64(x);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) scratch[wave] = x;
    __syncthreads();
    T before = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves - 1; ++w) {
        const T y = scratch[w];
        before += w < wave ? y : T(0);
    }
    return x + before;
}

// The row's logits that thread `tid` holds of tile `j` of a chunk: four neighbours; -infinity behind the end.
template <bool VEC>
__device__ __forceinline__ floatx4_t sample_load(const float* x, int i, int V)
{
    floatx4_t v;
    if (VEC && i + 3 < V) {
        v = *reinterpret_cast<const floatx4_t*>(x + i);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < V ? x[i + e] : -__builtin_inff();
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = sample_logit(v[e]);
    return v;
}

// Bins of logits on a grid that does not depend on the row: of a sixteenth, or a sixteenth of t where t is
// below 1, so that 512 of them reach down to weights of e^-32 (t up to 1) or 32 below the largest logit, the
// last one holding all that is lower. A bin of 150,000 normal logits of deviation 2 has at most 1900.
// (Whole floats: the differences of two of them are exact wherever they are below 512.)
__device__ __forceinline__ float sample_grid(float l, const SampleRow& s)
{
    return floorf(fminf(fmaxf(l * (16.0f / fminf(s.t, 1.0f)), -0x1p30f), 0x1p30f));
}
__device__ __forceinline__ int sample_bin(float l, float top_grid, const SampleRow& s)
{
    return (int)fminf(top_grid - sample_grid(l, s), (float)(kSampleBins - 1));
}

// 1. Each chunk of a row: its largest logit (and that one's index, for the likeliest token), and, where k or p
// is set, how many logits fall into each bin and, roughly, their weights relative to the chunk's largest: a count in
// the low 15 bits (a chunk has 2^14), the weights in fp32 as multiples of 2^-31 above, in one whole number, so that an
// addition in LDS does both and the order of additions does not matter.
template <bool VEC>
__global__ __launch_bounds__(kSampleThreads) void sample_scan_kernel(SampleArgs a, SampleWs ws)
{
    __shared__ u64 hist[kSampleBins], scratch[kSampleWaves];
    __shared__ int first;
    const int r = blockIdx.y, c = blockIdx.x, tid = threadIdx.x;
    const float* const x = a.logits + (ws.row0 + r) * a.stride;
    const SampleRow s = sample_row(a, ws.row0 + r);
    const int at = c * kSampleTile * kSampleTiles + 4 * tid;
    floatx4_t v[kSampleTiles];
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j) v[j] = sample_load<VEC>(x, at + j * kSampleTile, a.vocab);
    if (tid < kSampleBins) hist[tid] = 0;
    if (tid == 0) first = INT32_MAX;
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, v[j][e]);
    top = block_max(top, scratch);
    if (tid == 0) ws.top[(int64_t)r * ws.chunks + c] = top;
    if (s.greedy) {
        int mine = INT32_MAX;
#pragma unroll
        for (int j = kSampleTiles - 1; j >= 0; --j)
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (v[j][e] == top) mine = at + j * kSampleTile + e;
        if (mine != INT32_MAX) atomicMin(&first, mine);
        __syncthreads();
        if (tid == 0) ws.first[(int64_t)r * ws.chunks + c] = first;
        return;
    }
    if (s.k == a.vocab && !(s.p < 1.0f)) return;
    if (top > -__builtin_inff()) {
        const float grid = sample_grid(top, s), scale = (float)s.scale;
#pragma unroll
        for (int j = 0; j < kSampleTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float l = v[j][e];
                if (l == -__builtin_inff()) continue;
                const float w = l == top ? 1.0f : sample_rough(l - top, scale);
                atomicAdd(&hist[sample_bin(l, grid, s)], (u64)(uint32_t)__builtin_fmaf(w, 0x1p31f, 0.5f) << 15 | 1);
            }
    }
    __syncthreads();
    u64 all[1] = {tid < kSampleBins ? hist[tid] : 0};
    if (tid < kSampleBins) ws.hist[((int64_t)r * ws.chunks + c) * kSampleBins + tid] = all[0];
    block_sums(all, scratch);
    if (tid == 0) ws.all[(int64_t)r * ws.chunks + c] = all[0];
}

// 2. Each chunk again, with the whole row's largest logit and bins. The bins that a border may lie in are known but
// for the rough sums' error: [lo, hi] for the last token kept, and k's where p needs the sum of the first k. Their
// logits go to the row's list (as places, in the chunks' order); what lies before them is kept and summed
// exactly, tile by tile. (Every chunk's workgroup finds the bins for itself: 4 KB a chunk, from L2.)
template <bool VEC>
__global__ __launch_bounds__(kSampleThreads) void sample_sum_kernel(SampleArgs a, SampleWs ws)
{
    __shared__ double mass[2][kSampleBins], factor[kSampleChunks];
    __shared__ uint32_t counts[2][kSampleBins];
    __shared__ int16_t offset[kSampleChunks];
    __shared__ u64 scratch[(kSampleTiles + 2) * kSampleWaves];
    __shared__ int found[4];
    __shared__ uint32_t place;
    const int r = blockIdx.y, c = blockIdx.x, tid = threadIdx.x;
    const SampleRow s = sample_row(a, ws.row0 + r);
    if (s.greedy) return;
    const int at = c * kSampleTile * kSampleTiles + 4 * tid;
    floatx4_t v[kSampleTiles];
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j)
        v[j] = sample_load<VEC>(a.logits + (ws.row0 + r) * a.stride, at + j * kSampleTile, a.vocab);
    const float mine = tid < ws.chunks ? ws.top[(int64_t)r * ws.chunks + tid] : -__builtin_inff();
    const float top = block_max(mine, scratch);
    if (top == -__builtin_inff()) return;
    const float grid = sample_grid(top, s);
    bool by_k = s.k < a.vocab;
    const bool by_p = s.p < 1.0f;
    int lo = kSampleBins, hi = kSampleBins, bk = kSampleBins;
    uint32_t k_before = 0, listed = 0;
    if (by_k || by_p) {
        // a chunk's bins begin `offset` below the row's; its weights count by its largest logit's
        u64 rest = 0;
        if (tid < ws.chunks) {
            const bool some = mine > -__builtin_inff();
            offset[tid] = some ? (int16_t)fminf(grid - sample_grid(mine, s), (float)kSampleBins) : (int16_t)kSampleBins;
            factor[tid] = mine == top ? 1.0 : (double)sample_rough(mine - top, (float)s.scale);
            rest = some ? ws.all[(int64_t)r * ws.chunks + tid] : 0;
        }
        if (tid < 4) found[tid] = kSampleBins - 1;
        __syncthreads();
        const int bin = tid & (kSampleBins - 1), half = tid / kSampleBins;
        const u64* const hists = ws.hist + (int64_t)r * ws.chunks * kSampleBins;
        double m = 0.0;
        uint32_t n = 0;
#pragma unroll 4
        for (int i = half; i < ws.chunks; i += kSampleThreads / kSampleBins) {
            const int b = bin - offset[i];
            const u64 h = hists[(int64_t)i * kSampleBins + max(b, 0)];
            n += b >= 0 ? (uint32_t)(h & 0x7fff) : 0;
            m += b >= 0 ? (double)(h >> 15) * factor[i] : 0.0;
        }
        mass[half][bin] = m;
        counts[half][bin] = n;
        // all of the row: its last bin holds what none of the others does
        const double all_mass = block_scan((double)(rest >> 15) * (tid < ws.chunks ? factor[tid] : 0.0), reinterpret_cast<double*>(scratch));
        const u64 all_count = block_scan((u64)(rest & 0x7fff), scratch);
        if (tid == kSampleThreads - 1) {
            mass[0][kSampleBins - 1] = all_mass;
            counts[0][kSampleBins - 1] = (uint32_t)all_count;
        }
        m = tid < kSampleBins - 1 ? mass[0][tid] + mass[1][tid] : 0.0;
        n = tid < kSampleBins - 1 ? counts[0][tid] + counts[1][tid] : 0;
        m = block_scan(m, reinterpret_cast<double*>(scratch));
        n = (uint32_t)block_scan((u64)n, scratch);
        if (tid < kSampleBins - 1) {
            mass[0][tid] = m;
            counts[0][tid] = n;
        }
        __syncthreads();
        if (tid == kSampleBins - 1) {
            m = mass[0][tid];
            n = counts[0][tid];
        }
        const uint32_t all = counts[0][kSampleBins - 1];
        by_k = by_k && (uint32_t)s.k < all;
        if (by_k) {
            if (tid < kSampleBins && n >= (uint32_t)s.k) atomicMin(&found[0], tid);
            __syncthreads();
            bk = found[0];
            k_before = bk ? counts[0][bk - 1] : 0;
        }
        if (by_p) {
            // two of fp32's exponentials, off by 2^-17 each (arguments up to 64, rounded twice), and half a step each
            const double off = 0x1p-14 * mass[0][kSampleBins - 1] + (double)all;
            const double w0 = by_k ? bk ? mass[0][bk - 1] : 0.0 : mass[0][kSampleBins - 1];
            const double w1 = mass[0][by_k ? bk : kSampleBins - 1], p = s.p > 0.0f ? s.p : 0.0;
            if (tid < kSampleBins && m >= p * w0 - off) atomicMin(&found[1], tid);
            if (tid < kSampleBins && m >= p * w1 + off) atomicMin(&found[2], tid);
            __syncthreads();
            hi = min(found[2], by_k ? bk : kSampleBins - 1);
            lo = min(found[1], hi);
        } else if (by_k) {
            lo = hi = bk;
        }
        // how many are listed, and how many of them by the chunks before this one
        if (lo < kSampleBins) {
            const bool two = by_p && by_k && bk > hi;
            listed = counts[0][hi] - (lo ? counts[0][lo - 1] : 0) + (two ? counts[0][bk] - counts[0][bk - 1] : 0);
            u64 before[1] = {};
            if (tid < c) {
                const u64* const h = hists + (int64_t)tid * kSampleBins;
                const int off = offset[tid];
                // bin b of the row; the last one: all that the others do not hold
                auto count = [&](int b) {
                    if (b < kSampleBins - 1) return b >= off ? (uint32_t)(h[b - off] & 0x7fff) : 0;
                    uint32_t q = (uint32_t)(rest & 0x7fff);
                    for (int k = 0; k < kSampleBins - 1 - off; ++k) q -= (uint32_t)(h[k] & 0x7fff);
                    return q;
                };
                for (int b = lo; b <= hi; ++b) before[0] += count(b);
                if (two) before[0] += count(bk);
            }
            block_sums(before, scratch);
            if (tid == 0) place = (uint32_t)before[0];
            __syncthreads();
        }
    }
    const bool list = listed && listed <= kSampleList;
    if (c == 0 && tid == 0) ws.found[r] = {top, lo, hi, bk, by_k, by_p, k_before, list ? listed : 0};

    // sums: each tile's kept weights before `lo`; the weights before `lo`; all weights that p is a part of
    const u64 least = sample_least(s, a.frac);
    const int whole = by_p ? by_k ? bk : kSampleBins : 0, bins = max(lo, whole);
    u64* const out = ws.list + (int64_t)r * kSampleList;
    u64 sums[kSampleTiles + 2] = {};
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j) {
        int b[4];
        bool any = false, some = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            b[e] = lo < kSampleBins ? sample_bin(v[j][e], grid, s) : 0;
            if (v[j][e] == -__builtin_inff()) b[e] = kSampleBins;
            any |= b[e] < bins;
            some |= b[e] >= lo && (b[e] <= hi || b[e] == bk);
        }
        if (__ballot(any)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u64 w = sample_weight(v[j][e], top, s, a.frac);
                const u64 before = b[e] < lo ? w : 0;
                sums[j] += before >= least ? before : 0;
                sums[kSampleTiles] += before;
                sums[kSampleTiles + 1] += b[e] < whole ? w : 0;
            }
        }
        if (list && some)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (b[e] < kSampleBins && ((b[e] >= lo && b[e] <= hi) || (by_p && b[e] == bk)))
                    if (const uint32_t to = atomicAdd(&place, 1); to < kSampleList)   // (or the logits have changed since)
                        out[to] = sample_place(v[j][e], at + j * kSampleTile + e, ws.index_bits);
    }
    block_sums(sums, scratch);
    const int64_t chunk = (int64_t)r * ws.chunks + c;
    if (tid == 0) {
#pragma unroll
        for (int j = 0; j < kSampleTiles; ++j) ws.tiles[chunk * kSampleTiles + j] = sums[j];
        ws.sums[chunk * 2] = sums[kSampleTiles];
        ws.sums[chunk * 2 + 1] = sums[kSampleTiles + 1];
    }
}

// 3. Each row: the borders among the listed logits (or, where those are too many for the list, among the
// row's), and the draw.
struct SampleLds {
    u64 hist[1 << kSampleDigit];
    uint32_t counts[1 << kSampleDigit];
    u64 list[kSampleList];
    u64 digit[256], digit_weight[256];
    u64 few[kWave];
    u64 scratch[2 * kSampleWaves];
    u64 found[8];
    u64 tiles[1];   // [chunks * kSampleTiles]
};

// By one wave: the place at which the counts or weights of its n lanes' places, in order and up to `last`, sum to
// `target`; the last of them where they do not. And the sum up to it.
struct SampleBorder {
    u64 place, sum;
};
__device__ __forceinline__ SampleBorder sample_rank(u64 c, u64 w, int n, u64 last, u64 target)
{
    const int lane = threadIdx.x & (kWave - 1);
    const bool in = lane < n && c <= last;
    u64 sum = 0;
    for (int i = 0; i < n; ++i) {
        const u64 ci = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(c >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)c, i);
        const u64 wi = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)w, i);
        sum += ci <= c && ci <= last ? wi : 0;
    }
    // the lowest sum that reaches it, else the highest
    SampleBorder b{0, 0};
    bool reached = false;
    for (int i = 0; i < n; ++i) {
        const u64 ci = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(c >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)c, i);
        const u64 si = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(sum >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)sum, i);
        if (!__builtin_amdgcn_readlane((int)in, i)) continue;
        const bool enough = si >= target;
        if (enough ? !reached || ci < b.place : !reached && ci >= b.place) b = {ci, si};
        reached |= enough;
    }
    return b;
}

__global__ __launch_bounds__(kSampleThreads) void sample_draw_kernel(SampleArgs a, SampleWs ws)
{
    extern __shared__ u64 sample_lds[];
    SampleLds& lds = *reinterpret_cast<SampleLds*>(sample_lds);
    const int r = blockIdx.x, row = ws.row0 + r, tid = threadIdx.x, V = a.vocab;
    const float* const x = a.logits + row * a.stride;
    const SampleRow s = sample_row(a, row);
    auto answer = [&](int token, float logprob) {
        a.token[row] = token;
        if (a.logprob) a.logprob[row] = logprob;
    };
    // everything that lies at a known place is loaded before any of it is waited for
    const SampleFound f = ws.found[r];
    const int64_t chunk0 = (int64_t)r * ws.chunks;
    const int tiles = ws.chunks * kSampleTiles;
    const float mine_top = tid < ws.chunks ? ws.top[chunk0 + tid] : -__builtin_inff();
    u64 sums[2] = {};
    if (tid < ws.chunks) {
        sums[0] = ws.sums[(chunk0 + tid) * 2];
        sums[1] = ws.sums[(chunk0 + tid) * 2 + 1];
    }
    for (int i = tid; i < tiles; i += kSampleThreads) lds.tiles[i] = ws.tiles[chunk0 * kSampleTiles + i];
    const float top = block_max(mine_top, lds.scratch);
    if (s.greedy || top == -__builtin_inff()) {
        if (top == -__builtin_inff()) {   // nothing to draw from
            if (tid == 0) answer(-1, __builtin_nanf(""));
        } else {
            const uint64_t here = __ballot(mine_top == top);   // the first chunk's
            if ((tid & (kWave - 1)) == 0) lds.scratch[tid >> 6] = here;
            __syncthreads();
            if (tid == 0) {
                int w = 0;
                while (w < kSampleWaves - 1 && !lds.scratch[w]) ++w;
                answer(ws.first[chunk0 + w * kWave + __ffsll(lds.scratch[w]) - 1], 0.0f);
            }
        }
        return;
    }
    const float grid = sample_grid(top, s);
    const bool borders = f.lo < kSampleBins;
    const u64 least = sample_least(s, a.frac);
    const int n = (int)f.listed;   // 0: the row itself
    u64 last = ~0ull;
    if (borders) {
        const bool two = f.by_k && f.by_p && f.bk > f.hi;
        // fine bins: as many to each bin that is listed, by the logit's place in it
        const int fine = (1 << kSampleDigit) / (f.hi - f.lo + 1 + two);
        const float inv = 16.0f / fminf(s.t, 1.0f);
        auto fine_bin = [&](float l, int b) {
            const float q = l * inv, part = 1.0f - (q - floorf(q));
            const int k = b == kSampleBins - 1 || !(part >= 0.0f) ? fine - 1 : min((int)(part * (float)fine), fine - 1);
            return (b > f.hi ? f.hi + 1 - f.lo : b - f.lo) * fine + k;
        };
        // every listed place: fn(place, logit, bin)
        auto each = [&](auto&& fn) {
            const int m = n ? n : V;
            for (int i = tid; i < m; i += kSampleThreads) {
                const u64 c = n ? lds.list[i] : sample_place(sample_logit(x[i]), i, ws.index_bits);
                const float l = sample_unkey((uint32_t)(c >> ws.index_bits));
                if (l == -__builtin_inff()) continue;
                const int b = sample_bin(l, grid, s);
                if ((b >= f.lo && b <= f.hi) || (two && b == f.bk)) fn(c, l, b);
            }
        };
        for (int i = tid; i < 1 << kSampleDigit; i += kSampleThreads) {
            lds.hist[i] = 0;
            lds.counts[i] = 0;
        }
        for (int i = tid; i < n; i += kSampleThreads) lds.list[i] = ws.list[(int64_t)r * kSampleList + i];
        if (tid < 8) lds.found[tid] = (1 << kSampleDigit) - 1;
        block_sums(sums, lds.scratch);   // (its barriers are the list's too)
        each([&](u64, float l, int b) {
            const int k = fine_bin(l, b);
            atomicAdd(&lds.counts[k], 1);
            if (f.by_p) atomicAdd(&lds.hist[k], sample_weight(l, top, s, a.frac));
        });
        __syncthreads();
        {   // sums up to and with each fine bin, two to a thread
            const uint32_t n0 = lds.counts[2 * tid], n1 = lds.counts[2 * tid + 1];
            const u64 h0 = lds.hist[2 * tid], h1 = lds.hist[2 * tid + 1];
            const uint32_t up = (uint32_t)block_scan((u64)n0 + n1, lds.scratch);
            lds.counts[2 * tid] = up - n1;
            lds.counts[2 * tid + 1] = up;
            if (f.by_p) {
                const u64 sum = block_scan(h0 + h1, lds.scratch);
                lds.hist[2 * tid] = sum - h1;
                lds.hist[2 * tid + 1] = sum;
            }
        }
        __syncthreads();

        // The place in fine bin `k` at which the counts or weights of its places, up to `up_to`, sum to `target`,
        // and their sum of weights up to it.
        auto border = [&](int k, u64 up_to, u64 target, bool count) -> SampleBorder {
            const uint32_t m = lds.counts[k] - (k ? lds.counts[k - 1] : 0);
            if (m <= kWave) {   // by one wave
                if (tid == 0) lds.found[0] = 0;
                __syncthreads();
                each([&](u64 c, float l, int b) {
                    if (fine_bin(l, b) == k)
                        if (const u64 to = atomicAdd(&lds.found[0], 1); to < kWave) lds.few[to] = c;
                });
                __syncthreads();
                if (tid < kWave) {
                    const u64 c = lds.few[tid];
                    const u64 w = sample_weight(sample_unkey((uint32_t)(c >> ws.index_bits)), top, s, a.frac);
                    SampleBorder q = sample_rank(c, count ? 1 : w, (int)m, up_to, target);
                    if (count) {
                        u64 sum = tid < (int)m && c <= q.place ? w : 0;
                        sum = wave_scan64(sum);
                        q.sum = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(sum >> 32), 63) << 32 |
                                (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
                    }
                    if (tid == 0) {
                        lds.found[1] = q.place;
                        lds.found[2] = q.sum;
                    }
                }
                __syncthreads();
                return {lds.found[1], lds.found[2]};
            }
            // many, as equal logits are: by digits of 8 bits below what they have in common
            u64 low = ~0ull, high = 0;
            each([&](u64 c, float l, int b) {
                if (fine_bin(l, b) == k && c <= up_to) {
                    low = min(low, c);
                    high = max(high, c);
                }
            });
            if (tid < 2) lds.found[tid] = tid ? 0 : ~0ull;
            __syncthreads();
            atomicMin(&lds.found[0], low);
            atomicMax(&lds.found[1], high);
            __syncthreads();
            low = lds.found[0];
            high = lds.found[1];
            if (low >= high) return {high, sample_weight(sample_unkey((uint32_t)(high >> ws.index_bits)), top, s, a.frac)};
            int above = 64 - __builtin_clzll(low ^ high);
            u64 prefix = above < 64 ? low >> above : 0, before = 0, weights = 0;
            while (above > 0) {
                const int shift = max(0, above - 8);
                __syncthreads();
                if (tid < 256) lds.digit[tid] = lds.digit_weight[tid] = 0;
                if (tid < 2) lds.found[tid] = 0;
                __syncthreads();
                each([&](u64 c, float l, int b) {
                    if (fine_bin(l, b) != k || c > up_to || (above < 64 && c >> above != prefix)) return;
                    const int d = (int)(c >> shift) & ((1 << (above - shift)) - 1);
                    const u64 w = sample_weight(l, top, s, a.frac);
                    atomicAdd(&lds.digit_weight[d], w);
                    atomicAdd(&lds.digit[d], count ? 1 : w);
                    atomicMax(&lds.found[0], (u64)d);   // the last there is, should the target not be reached
                });
                __syncthreads();
                const u64 mine = tid < 256 ? lds.digit[tid] : 0, heavy = tid < 256 ? lds.digit_weight[tid] : 0;
                const u64 up = before + block_scan(mine, lds.scratch), up_weights = weights + block_scan(heavy, lds.scratch);
                const int end = (int)lds.found[0];
                __syncthreads();
                if (tid <= end && up - mine < target && (up >= target || tid == end)) {
                    lds.found[1] = tid;
                    lds.found[0] = up - mine;
                    lds.found[2] = up_weights - heavy;
                }
                __syncthreads();
                prefix = prefix << (above - shift) | lds.found[1];
                before = lds.found[0];
                weights = lds.found[2];
                above = shift;
            }
            return {prefix, weights + sample_weight(sample_unkey((uint32_t)(prefix >> ws.index_bits)), top, s, a.frac)};
        };
        // the fine bin at which the sums reach a target
        auto reach = [&](int slot, const auto& at, u64 target) {
            const bool here0 = at[2 * tid] >= target, here1 = at[2 * tid + 1] >= target;
            if (here0 || here1) atomicMin(&lds.found[slot], (u64)(2 * tid + !here0));
            __syncthreads();
            return (int)lds.found[slot];
        };
        u64 whole = sums[1];   // what p is a part of
        if (f.by_k) {
            const int first = (two ? f.hi + 1 - f.lo : f.bk - f.lo) * fine;   // bk's first fine bin
            const u64 target = (u64)s.k - f.k_before + (first ? lds.counts[first - 1] : 0);
            const int k = reach(3, lds.counts, target);
            const SampleBorder q = border(k, ~0ull, target - (k ? lds.counts[k - 1] : 0), true);
            last = q.place;
            if (f.by_p) whole += (k ? lds.hist[k - 1] : 0) - (first ? lds.hist[first - 1] : 0) + q.sum;
        }
        if (f.by_p) {
            const u64 all = sample_part(s.p, whole, true), target = all > sums[0] ? all - sums[0] : 0;
            const int k = reach(4, lds.hist, target);
            last = target ? border(k, last, target - (k ? min(lds.hist[k - 1], target - 1) : 0), false).place : 0;
        }
        __syncthreads();
        each([&](u64 c, float l, int b) {
            const u64 w = sample_weight(l, top, s, a.frac);
            const int tile = ((uint32_t)c & ((1u << ws.index_bits) - 1)) / kSampleTile;
            if (b <= f.hi && c <= last && w >= least && tile < tiles) atomicAdd(&lds.tiles[tile], w);
        });
    }
    __syncthreads();

    // the tile that the draw falls into, then its token
    u64 sum[1] = {};
    for (int i = tid; i < tiles; i += kSampleThreads) sum[0] += lds.tiles[i];
    block_sums(sum, lds.scratch);
    const u64 total = sum[0];
    u64 target = sample_part(s.u, total, false), before = 0;
    if (tid == 0) lds.found[0] = lds.found[1] = 0;
    for (int base = 0; base < tiles; base += kSampleThreads) {
        const u64 mine = base + tid < tiles ? lds.tiles[base + tid] : 0;
        const u64 up_to = before + block_scan(mine, lds.scratch);
        if (up_to > target && up_to - mine <= target) {
            lds.found[0] = base + tid;
            lds.found[1] = up_to - mine;
        }
        if (tid == kSampleThreads - 1) lds.found[2] = up_to;
        __syncthreads();
        before = lds.found[2];
        if (before > target) break;
    }
    const int tile = (int)lds.found[0];
    target -= lds.found[1];
    const int at = tile * kSampleTile + 4 * tid;
    u64 w[4], mine = 0;
    const floatx4_t v = sample_load<false>(x, at, V);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool kept = v[e] > -__builtin_inff() &&
                          (sample_place(v[e], at + e, ws.index_bits) <= last || sample_bin(v[e], grid, s) < f.lo);
        const u64 we = kept ? sample_weight(v[e], top, s, a.frac) : 0;
        w[e] = we >= least ? we : 0;
        mine += w[e];
    }
    u64 up_to = block_scan(mine, lds.scratch);
    if (up_to > target && up_to - mine <= target) {
        up_to -= mine;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            up_to += w[e];
            if (up_to > target) {
                answer(at + e, (float)log((double)w[e] / (double)total));
                break;
            }
        }
    }
}

}  // namespace msnb
