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
// eleventh power (the next term is below 2^-46), in multiples of 2^-frac.
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
    if (!(y > -64.0)) return 0;
    const double k = __builtin_rint(y), f = y - k;
    double s = c[11];
#pragma unroll
    for (int n = 10; n >= 0; --n) s = __builtin_fma(s, f, c[n]);
    // below 2^52 the sum's low bits are the whole number, rounded
    return __builtin_bit_cast(u64, __builtin_ldexp(s, (int)k + frac) + 0x1p52) & ((1ull << 52) - 1);
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
    if (l == top) return 1ull << frac;
    // (a difference from an infinite largest is -infinity, and so is that from a logit of -infinity)
    return sample_exp2(((double)l - (double)top) * s.scale, frac);
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

__device__ __forceinline__ u64 wave_sum_all(u64 x)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
// Sums over the workgroup, in every thread.
template <int N>
__device__ __forceinline__ void block_sums(u64 (&x)[N], u64* scratch)
{
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = wave_sum_all(x[n]);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0)
#pragma unroll
        for (int n = 0; n < N; ++n) scratch[n * kSampleWaves + (threadIdx.x >> 6)] = x[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        x[n] = 0;
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
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const T y = __shfl_up(x, o);
        x += lane >= o ? y : T(0);
    }
    __syncthreads();
    if (lane == kWave - 1) scratch[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) x += scratch[w];
    return x;
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
    if (tid < kSampleBins) ws.hist[((int64_t)r * ws.chunks + c) * kSampleBins + tid] = hist[tid];
}

// 2. Each chunk again, with the whole row's largest logit and bins. The bins that a border may lie in are known but
// for the rough sums' error: [lo, hi] for the last token kept, and k's where p needs the sum of the first k. Their
// logits go to the row's list (as places, in the chunks' order); what lies before them is kept and summed
// exactly, tile by tile.
template <bool VEC>
__global__ __launch_bounds__(kSampleThreads) void sample_sum_kernel(SampleArgs a, SampleWs ws)
{
    __shared__ double mass[kSampleBins];
    __shared__ uint32_t counts[kSampleBins];
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
    const float* const tops = ws.top + (int64_t)r * ws.chunks;
    float top = -__builtin_inff();
    for (int i = tid; i < ws.chunks; i += kSampleThreads) top = fmaxf(top, tops[i]);
    top = block_max(top, scratch);
    if (top == -__builtin_inff()) return;
    const float grid = sample_grid(top, s);
    const u64* const hists = ws.hist + (int64_t)r * ws.chunks * kSampleBins;
    bool by_k = s.k < a.vocab;
    const bool by_p = s.p < 1.0f;
    int lo = kSampleBins, hi = kSampleBins, bk = kSampleBins;
    uint32_t k_before = 0, listed = 0;
    if (by_k || by_p) {
        // a chunk's bins begin `off` below the row's; its weights count by its largest logit's
        if (tid < kSampleBins) {
            mass[tid] = 0.0;
            counts[tid] = 0;
        }
        double m = 0.0;
        uint32_t n = 0;
        if (tid < kSampleBins) {
            for (int i = 0; i < ws.chunks; ++i) {
                const float ti = tops[i];
                if (ti == -__builtin_inff()) continue;
                const int off = (int)fminf(grid - sample_grid(ti, s), (float)(kSampleBins - 1));
                const double f = ti == top ? 1.0 : (double)sample_rough(ti - top, (float)s.scale);
                // the last bin takes all that falls past it
                for (int b = max(tid - off, 0); b <= (tid == kSampleBins - 1 ? tid : tid - off); ++b) {
                    const u64 h = hists[(int64_t)i * kSampleBins + b];
                    n += (uint32_t)(h & 0x7fff);
                    m += (double)(h >> 15) * f;
                }
            }
        }
        m = block_scan(m, reinterpret_cast<double*>(scratch));
        n = block_scan(n, reinterpret_cast<uint32_t*>(scratch));
        if (tid < kSampleBins) {
            mass[tid] = m;
            counts[tid] = n;
        }
        if (tid < 4) found[tid] = kSampleBins - 1;
        __syncthreads();
        const uint32_t all = counts[kSampleBins - 1];
        by_k = by_k && (uint32_t)s.k < all;
        if (by_k) {
            if (tid < kSampleBins && n >= (uint32_t)s.k) atomicMin(&found[0], tid);
            __syncthreads();
            bk = found[0];
            k_before = bk ? counts[bk - 1] : 0;
        }
        if (by_p) {
            // two of fp32's exponentials, off by 2^-17 each (arguments up to 64, rounded twice), and half a step each
            const double off = 0x1p-14 * mass[kSampleBins - 1] + (double)all;
            const double w0 = by_k ? bk ? mass[bk - 1] : 0.0 : mass[kSampleBins - 1], w1 = mass[by_k ? bk : kSampleBins - 1];
            const double p = s.p > 0.0f ? s.p : 0.0;
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
            listed = counts[hi] - (lo ? counts[lo - 1] : 0);
            if (by_p && by_k && bk > hi) listed += counts[bk] - counts[bk - 1];
            uint32_t before = 0;
            for (int i = tid; i < c; i += kSampleThreads) {
                const float ti = tops[i];
                if (ti == -__builtin_inff()) continue;
                const int off = (int)fminf(grid - sample_grid(ti, s), (float)(kSampleBins - 1));
                auto count = [&](int b) {   // bin b of the row
                    uint32_t q = 0;
                    for (int k = max(b - off, 0); k <= (b == kSampleBins - 1 ? b : b - off); ++k)
                        q += (uint32_t)(hists[(int64_t)i * kSampleBins + k] & 0x7fff);
                    return q;
                };
                for (int b = lo; b <= hi; ++b) before += count(b);
                if (by_p && by_k && bk > hi) before += count(bk);
            }
            u64 sum[1] = {before};
            block_sums(sum, scratch);
            if (tid == 0) place = (uint32_t)sum[0];
            __syncthreads();
        }
    }
    const bool list = listed && listed <= kSampleList;
    if (c == 0 && tid == 0) ws.found[r] = {top, lo, hi, bk, by_k, by_p, k_before, list ? listed : 0};

    // sums: each tile's kept weights before `lo`; all weights that p is a part of; the weights before `lo`
    const u64 least = sample_least(s, a.frac);
    const int whole = by_p ? by_k ? bk : kSampleBins : lo;
    u64* const out = ws.list + (int64_t)r * kSampleList;
    u64 sums[kSampleTiles + 2] = {};
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float l = v[j][e];
            if (l == -__builtin_inff()) continue;
            const int b = lo < kSampleBins ? sample_bin(l, grid, s) : 0;
            if (b < whole || b < lo) {
                const u64 w = sample_weight(l, top, s, a.frac);
                if (b < lo) {
                    sums[j] += w >= least ? w : 0;
                    sums[kSampleTiles] += w;
                }
                if (b < whole) sums[kSampleTiles + 1] += w;
            }
            if (list && ((b >= lo && b <= hi) || (by_p && b == bk)))
                if (const uint32_t to = atomicAdd(&place, 1); to < kSampleList)   // (or the logits have changed since)
                    out[to] = sample_place(l, at + j * kSampleTile + e, ws.index_bits);
        }
    block_sums(sums, scratch);
    if (tid < kSampleTiles) ws.tiles[((int64_t)r * ws.chunks + c) * kSampleTiles + tid] = sums[tid];
    if (tid == 0) {
        ws.sums[((int64_t)r * ws.chunks + c) * 2] = sums[kSampleTiles];
        ws.sums[((int64_t)r * ws.chunks + c) * 2 + 1] = sums[kSampleTiles + 1];
    }
}

// 3. Each row: the borders among the listed logits (or, where those are too many for the list, among the
// row's), and the draw.
struct SampleLds {
    u64 hist[1 << kSampleDigit];
    uint32_t counts[1 << kSampleDigit];
    u64 list[kSampleList];
    u64 scratch[2 * kSampleWaves];
    u64 found[4];
    u64 tiles[1];   // [chunks * kSampleTiles]
};

__global__ __launch_bounds__(kSampleThreads) void sample_draw_kernel(SampleArgs a, SampleWs ws)
{
    extern __shared__ u64 sample_lds[];
    SampleLds& lds = *reinterpret_cast<SampleLds*>(sample_lds);
    const int r = blockIdx.x, row = ws.row0 + r, tid = threadIdx.x, V = a.vocab;
    const float* const x = a.logits + row * a.stride;
    const SampleRow s = sample_row(a, row);
    const float* const tops = ws.top + (int64_t)r * ws.chunks;
    auto answer = [&](int token, float logprob) {
        a.token[row] = token;
        if (a.logprob) a.logprob[row] = logprob;
    };
    float top = -__builtin_inff();
    for (int i = tid; i < ws.chunks; i += kSampleThreads) top = fmaxf(top, tops[i]);
    top = block_max(top, lds.scratch);
    if (top == -__builtin_inff()) {   // nothing to draw from
        if (tid == 0) answer(-1, __builtin_nanf(""));
        return;
    }
    if (s.greedy) {
        if (tid == 0) {
            int i = 0;
            while (i < ws.chunks - 1 && tops[i] != top) ++i;
            answer(ws.first[(int64_t)r * ws.chunks + i], 0.0f);
        }
        return;
    }
    const SampleFound f = ws.found[r];
    const float grid = sample_grid(top, s);
    const bool borders = f.lo < kSampleBins;
    const int n = f.listed;   // 0: the row itself
    if (borders)
        for (int i = tid; i < n; i += kSampleThreads) lds.list[i] = ws.list[(int64_t)r * kSampleList + i];
    for (int i = tid; i < ws.chunks * kSampleTiles; i += kSampleThreads) lds.tiles[i] = ws.tiles[(int64_t)r * ws.chunks * kSampleTiles + i];
    u64 sums[2] = {};
    for (int i = tid; i < ws.chunks; i += kSampleThreads) {
        sums[0] += ws.sums[((int64_t)r * ws.chunks + i) * 2];
        sums[1] += ws.sums[((int64_t)r * ws.chunks + i) * 2 + 1];
    }
    block_sums(sums, lds.scratch);

    // every place in bins [b0, b1], up to `last`
    auto each = [&](int b0, int b1, u64 last, auto&& fn) {
        const int m = n ? n : V;
        for (int i = tid; i < m; i += kSampleThreads) {
            const u64 c = n ? lds.list[i] : sample_place(sample_logit(x[i]), i, ws.index_bits);
            const float l = sample_unkey((uint32_t)(c >> ws.index_bits));
            if (c > last || l == -__builtin_inff()) continue;
            const int b = sample_bin(l, grid, s);
            if (b >= b0 && b <= b1) fn(c, l);
        }
    };
    // The place at which their counts or weights, in order, sum to `target`; the last of them where they do not.
    auto border = [&](int b0, int b1, u64 last, u64 target, bool count) -> u64 {
        if (tid == 0) {
            lds.found[0] = ~0ull;
            lds.found[1] = 0;
        }
        __syncthreads();
        u64 least = ~0ull, most = 0;
        each(b0, b1, last, [&](u64 c, float) {
            least = min(least, c);
            most = max(most, c);
        });
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            least = min(least, (u64)__shfl_xor(least, o));
            most = max(most, (u64)__shfl_xor(most, o));
        }
        if ((tid & (kWave - 1)) == 0) {
            atomicMin(&lds.found[0], least);
            atomicMax(&lds.found[1], most);
        }
        __syncthreads();
        least = lds.found[0];
        most = lds.found[1];
        if (least >= most) return most;
        const int bits = 64 - __builtin_clzll(least ^ most);
        int shift = max(0, bits - kSampleDigit);
        u64 prefix = bits < 64 ? least >> bits : 0;   // what the places left have in common, from bit `above` on
        int above = bits;
        u64 before = 0;
        for (;;) {
            __syncthreads();
            for (int i = tid; i < 1 << kSampleDigit; i += kSampleThreads) {
                lds.hist[i] = 0;
                lds.counts[i] = 0;
            }
            if (tid < 4) lds.found[tid] = tid == 0 ? ~0ull : 0;
            __syncthreads();
            const uint32_t mask = (1u << (above - shift)) - 1;
            each(b0, b1, last, [&](u64 c, float l) {
                if (above < 64 && c >> above != prefix) return;
                const uint32_t d = (uint32_t)(c >> shift) & mask;
                atomicAdd(&lds.hist[d], count ? 1 : sample_weight(l, top, s, a.frac));
                atomicAdd(&lds.counts[d], 1);
            });
            __syncthreads();
            // the first digit at which the sum reaches the target, else the last one that has any
            const int d0 = 2 * tid;
            const u64 h0 = lds.hist[d0], h1 = lds.hist[d0 + 1];
            const u64 sum = block_scan(h0 + h1, lds.scratch) + before;
            if (sum >= target) atomicMin(&lds.found[0], (u64)d0 + (sum - h1 < target));
            if (lds.counts[d0] || lds.counts[d0 + 1]) atomicMax(&lds.found[1], (u64)d0 + (lds.counts[d0 + 1] != 0));
            __syncthreads();
            const u64 d = min(lds.found[0], lds.found[1]);
            if ((u64)(d0 >> 1) == d >> 1) lds.found[2] = sum - (d & 1 ? h1 : h0 + h1);
            __syncthreads();
            before = lds.found[2];
            prefix = prefix << (above - shift) | d;
            above = shift;
            if (shift == 0) return prefix;
            if (lds.counts[d] == 1) {   // the only one left
                each(b0, b1, last, [&](u64 c, float) {
                    if (c >> above == prefix) lds.found[3] = c;
                });
                __syncthreads();
                return lds.found[3];
            }
            shift = max(0, shift - kSampleDigit);
        }
    };
    u64 last = ~0ull;
    if (f.by_k) last = border(f.bk, f.bk, ~0ull, (u64)s.k - f.k_before, true);
    if (f.by_p) {
        u64 w[1] = {};
        if (f.by_k) {
            each(f.bk, f.bk, last, [&](u64, float l) { w[0] += sample_weight(l, top, s, a.frac); });
            block_sums(w, lds.scratch);
        }
        const u64 target = sample_part(s.p, sums[1] + w[0], true);
        last = target > sums[0] ? border(f.lo, f.hi, last, target - sums[0], false) : 0;
    }
    const u64 least = sample_least(s, a.frac);
    __syncthreads();
    if (borders)
        each(f.lo, f.hi, last, [&](u64 c, float l) {
            const u64 w = sample_weight(l, top, s, a.frac);
            const int tile = ((uint32_t)c & ((1u << ws.index_bits) - 1)) / kSampleTile;
            if (w >= least && tile < ws.chunks * kSampleTiles) atomicAdd(&lds.tiles[tile], w);
        });
    __syncthreads();

    // the tile that the draw falls into, then its token
    const int tiles = ws.chunks * kSampleTiles;
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
    __syncthreads();
    const int tile = (int)lds.found[0];
    target -= lds.found[1];
    const int at = tile * kSampleTile + 4 * tid;
    u64 w[4], mine = 0;
    const floatx4_t v = sample_load<false>(x, at, V);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool kept = v[e] > -__builtin_inff() &&
                          (sample_place(v[e], at + e, ws.index_bits) <= last || sample_bin(v[e], grid, s) < f.lo);
        w[e] = kept ? sample_weight(v[e], top, s, a.frac) : 0;
        if (w[e] < least) w[e] = 0;
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
