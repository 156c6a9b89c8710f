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

// A logit as the order has it: NaN as -infinity, +infinity as the largest finite value.
__device__ __forceinline__ float sample_logit(float l) { return fminf(fmaxf(l, -__builtin_inff()), 3.402823466e38f); }

// Ascending in the order: falling logits (-0 as 0), then rising indexes.
__device__ __forceinline__ uint32_t sample_key(float l)
{
    const uint32_t b = __float_as_uint(l + 0.0f);
    return ~(b ^ ((int32_t)b < 0 ? ~0u : 0x80000000u));
}
__device__ __forceinline__ float sample_unkey(uint32_t k)
{
    const uint32_t b = ~k;
    return __uint_as_float(b ^ ((int32_t)b < 0 ? 0x80000000u : ~0u));
}
// A logit and its index in one number, the index in the low `bits`.
__device__ __forceinline__ u64 sample_place(float l, int i, int bits) { return (u64)sample_key(l) << bits | (uint32_t)i; }

// What a row's settings say.
struct SampleRow {
    float scale;     // log2(e) / t, roughly
    float t, p, m, u;
    int k;
    bool greedy;
};
__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, int r)
{
    SampleRow s;
    s.t = fminf(a.temperature ? a.temperature[r] : 1.0f, 1e30f);
    s.greedy = !(s.t > 0.0f) || (a.temperature && a.temperature[r] != a.temperature[r]);
    s.scale = 1.44269504f * __builtin_amdgcn_rcpf(s.t);
    const int k = a.top_k ? a.top_k[r] : 0;
    s.k = k <= 0 || k > a.vocab ? a.vocab : k;
    s.p = a.top_p ? a.top_p[r] : 1.0f;
    s.m = a.min_p ? a.min_p[r] : 0.0f;
    s.u = a.random[r];
    return s;
}
// A value that is the same in every lane, in scalar registers (there is no scalar arithmetic on floats, so the
// compiler holds a row's numbers once for each lane: spills at 64 registers, 10 of 43 us).
template <typename T>
__device__ __forceinline__ T uniform(T x)
{
    if constexpr (sizeof(T) == 8) {
        const u64 b = __builtin_bit_cast(u64, x);
        const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)b), hi = __builtin_amdgcn_readfirstlane((int)(b >> 32));
        return __builtin_bit_cast(T, (u64)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
    }
}

// scale = log2(e) / t, `low` where scale (l - top) is -60 (above -160 at `low` itself: where a step of fp32 at `top` is
// worth more than 2^64, no other logit than `top` counts and t may be more).
__device__ __forceinline__ float sample_below(float x)
{
    const uint32_t b = __float_as_uint(x);
    return x > 0.0f ? __uint_as_float(b - 1) : x < 0.0f ? __uint_as_float(b + 1) : -0x1p-149f;
}
__device__ __forceinline__ SampleScale sample_scale(float top, const SampleRow& s)
{
    const float below = fmaxf(sample_below(top), -3.402823466e38f);
    const double t = __builtin_fmax(s.t, below < top ? ((double)top - (double)below) * (1.4426950408889634074 / 64.0) : 0x1p98);
    return {uniform((double)top), uniform(1.4426950408889634074 / t),
            uniform(fmaxf(sample_below(top - 41.6f * s.t), -3.402823466e38f))};   // 60 ln 2
}
// A logit as its weight needs it: NaN and what is lower than `low` as that, +infinity as the largest finite value.
__device__ __forceinline__ float sample_clamp(float l, float low) { return __builtin_amdgcn_fmed3f(l, low, 3.402823466e38f); }

// 2^y, y = scale (l - top), by 2^k 2^f, k the nearest whole number, f in [-1/2, 1/2] by a polynomial (through 2^f at
// the zeros of a Chebyshev polynomial, 1 at 0; off by 2^-44 of it), as a whole multiple of 2^-frac in the low bits of
// a double's (the sum with 2^52 rounds it): kSampleBits above it. A logit's 16 operations in 64 bits (3 additions, 11
// fma, a conversion and a ldexp) are most of what bounds sampling by p, where every logit's weight counts. Four at a
// time, so that none waits for its own.
constexpr u64 kSampleBits = 0x433ull << 52;
template <int N>
__device__ __forceinline__ void sample_raw(const float (&l)[N], const SampleScale& e, int frac, u64 (&out)[N])
{
    constexpr double c[10] = {1.0,
                              0.6931471805599453,
                              0.2402265069581299,
                              0.055504108664760424,
                              0.009618129159402558,
                              0.0013333558179043112,
                              0.00015403455852453838,
                              1.525268684626772e-05,
                              1.3255224878668817e-06,
                              1.0203121063391729e-07};
    const double magic = 0x1.8p52 + frac;
    double t[N], f[N], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const double d = (double)l[i] - e.top;
        t[i] = __builtin_fma(d, e.scale, magic);   // k + frac in the low bits
        f[i] = __builtin_fma(d, e.scale, -(t[i] - magic));
        s[i] = c[9];
    }
#pragma unroll
    for (int n = 8; n >= 0; --n)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = __builtin_fma(s[i], f[i], c[n]);
#pragma unroll
    for (int i = 0; i < N; ++i)
        out[i] = __builtin_bit_cast(u64, __builtin_amdgcn_ldexp(s[i], (int)(uint32_t)__builtin_bit_cast(u64, t[i])) + 0x1p52);
}
__device__ __forceinline__ u64 sample_weight(float l, const SampleScale& e, int frac)
{
    const float x[1] = {sample_clamp(l, e.low)};
    u64 raw[1];
    sample_raw<1>(x, e, frac, raw);
    return raw[0] - kSampleBits;
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

constexpr int kSampleThreads = 512, kSampleWaves = kSampleThreads / kWave;
constexpr int kSampleLoads = 4;                                      // of a thread, 16 bytes each: a chunk's
constexpr int kSampleTile = 4 * kWave * kSampleLoads;                // tokens of a wave
static_assert(kSampleTiles == kSampleWaves, "a chunk's tiles to the waves of a workgroup");
constexpr int kSampleEach = kSampleBins / kWave;                     // bins of a lane

// A 64-bit value moved by one DPP control; lanes whose source is outside the row, or whose row the mask leaves
// out, read 0.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ u64 dpp64(u64 x)
{
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROW_MASK, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROW_MASK, 0xF, false);
    return (u64)hi << 32 | lo;
}
// Inclusive sums over the wave.
__device__ __forceinline__ u64 wave_scan64(u64 x)
{
    x += dpp64<0x111, 0xF>(x);   // row_shr:1
    x += dpp64<0x112, 0xF>(x);
    x += dpp64<0x114, 0xF>(x);
    x += dpp64<0x118, 0xF>(x);
    x += dpp64<0x142, 0xA>(x);   // row_bcast:15 -> rows 1, 3
    return x + dpp64<0x143, 0xC>(x);   // row_bcast:31 -> rows 2, 3
}
// x of lane l (a wave-uniform index), in every lane.
__device__ __forceinline__ u64 lane_value64(u64 x, int l)
{
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, l);
}
__device__ __forceinline__ u64 wave_sum64(u64 x) { return lane_value64(wave_scan64(x), kWave - 1); }
__device__ __forceinline__ float wave_max_all(float x)
{
    x = row16_max_all(x);
    x = fmaxf(x, xor16_value(x));
    return fmaxf(x, xor32_value(x));
}
// Inclusive sums of x over the workgroup's threads. The scratch is used again behind the next barrier.
template <int WAVES>
__device__ __forceinline__ u64 block_scan(u64 x, u64 (&scratch)[WAVES])
{
    const int wave = threadIdx.x >> 6;
    x = wave_scan64(x);
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) scratch[wave] = x;
    __syncthreads();
    u64 before = 0;
#pragma unroll
    for (int w = 0; w < WAVES - 1; ++w) {
        const u64 y = scratch[w];
        before += w < wave ? y : 0;
    }
    return x + before;
}
// Inclusive sums over the wave of 32-bit values.
template <int CTRL, int ROW_MASK, typename T>
__device__ __forceinline__ T dpp32(T x)
{
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROW_MASK, 0xF, false));
}
template <typename T>
__device__ __forceinline__ T wave_sums(T x)
{
    if constexpr (sizeof(T) == 8) {
        return wave_scan64(x);
    } else {
        x += dpp32<0x111, 0xF>(x);
        x += dpp32<0x112, 0xF>(x);
        x += dpp32<0x114, 0xF>(x);
        x += dpp32<0x118, 0xF>(x);
        x += dpp32<0x142, 0xA>(x);
        return x + dpp32<0x143, 0xC>(x);
    }
}
// 512 sums in order, eight to a lane, by each wave for itself.
template <typename T>
struct SampleSums {
    T up[kSampleEach];   // up to and with each of the lane's
    __device__ __forceinline__ void scan()
    {
#pragma unroll
        for (int e = 1; e < kSampleEach; ++e) up[e] += up[e - 1];
        const T before = wave_sums(up[kSampleEach - 1]) - up[kSampleEach - 1];
#pragma unroll
        for (int e = 0; e < kSampleEach; ++e) up[e] += before;
    }
    // the sum up to and with `bin`, 0 for -1
    __device__ __forceinline__ T at(int bin) const
    {
        T x = 0;
#pragma unroll
        for (int e = 0; e < kSampleEach; ++e) x = e == (bin & (kSampleEach - 1)) ? up[e] : x;
        if (bin < 0) return 0;
        if constexpr (sizeof(T) == 8)
            return lane_value64(x, bin / kSampleEach);
        else
            return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), bin / kSampleEach));
    }
    // the first bin whose sum is at least `target`; the last bin where none is
    __device__ __forceinline__ int reach(T target) const
    {
        int e = 0;
#pragma unroll
        for (int i = 0; i < kSampleEach - 1; ++i) e += up[i] < target;
        const uint64_t there = __ballot(up[kSampleEach - 1] >= target);
        if (!there) return kSampleBins - 1;
        const int l = __ffsll((unsigned long long)there) - 1;
        return kSampleEach * l + __builtin_amdgcn_readlane(e, l);
    }
};

// Where a row's tokens lie: four neighbours at 16 bytes to a load, so tile and chunk borders are `lead` tokens
// before multiples of theirs, lead being how many floats the row begins behind 16 bytes.
__device__ __forceinline__ int sample_lead(const float* x) { return (int)(reinterpret_cast<uintptr_t>(x) / 4 & 3); }
__device__ __forceinline__ floatx4_t sample_edge(const float* x, int i, int V)
{
    floatx4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e >= 0 && i + e < V ? x[i + e] : -__builtin_inff();
    return v;
}
// A thread's tokens of a chunk. What follows goes from load to load in loops that are not unrolled (a code of 23 KB
// run through once took 12 us for a row, most of it for the instructions), so they move down a place each time.
struct SampleChunk {
    floatx4_t v[kSampleLoads];
    // the thread's first token of a workgroup of WAVES; its loads are 256 tokens apart
    template <int WAVES>
    __device__ __forceinline__ static int first(const float* x, int c)
    {
        return (c * WAVES + (int)(threadIdx.x >> 6)) * kSampleTile + 4 * (int)(threadIdx.x & (kWave - 1)) - sample_lead(x);
    }
    __device__ __forceinline__ void load(const float* x, int at, int V)
    {
        const int begin = __builtin_amdgcn_readfirstlane(at);
        if (begin >= 0 && begin + kSampleTile <= V) {   // all of the wave's
#pragma unroll
            for (int j = 0; j < kSampleLoads; ++j) v[j] = *reinterpret_cast<const floatx4_t*>(x + at + 4 * kWave * j);
        } else {
#pragma unroll
            for (int j = 0; j < kSampleLoads; ++j) v[j] = sample_edge(x, at + 4 * kWave * j, V);
        }
    }
    __device__ __forceinline__ floatx4_t next()
    {
        const floatx4_t x = v[0];
#pragma unroll
        for (int j = 0; j + 1 < kSampleLoads; ++j) v[j] = v[j + 1];
        return x;
    }
};

// Bins of logits on a grid that does not depend on the row: of a sixteenth, or a sixteenth of t where t is
// below 1, so that the 512 from the largest logit's down reach weights of e^-32 (t up to 1) or 32 below it; the last
// one holds all that is lower. A bin of 150,000 normal logits of deviation 2 has at most 1900.
// (t below 2^-100: that of 2^-100, since 1 / t may be infinite.)
__device__ __forceinline__ float sample_step(const SampleRow& s)
{
    return 16.0f * __builtin_amdgcn_rcpf(fminf(fmaxf(s.t, 0x1p-100f), 1.0f));
}
__device__ __forceinline__ int sample_grid(float l, float step)
{
    return (int)floorf(fminf(fmaxf(l * step, -0x1p29f), 0x1p29f));
}
__device__ __forceinline__ int sample_bin(float l, int top_grid, float step)
{
    return min(top_grid - sample_grid(l, step), kSampleBins - 1);
}
// Where the grid's lines are no whole numbers in fp32, or t is next to infinity, the bins say nothing; nor where t is
// so small that a weight's exponent cannot be had by `scale` in fp32 (below 2^-100 alone: from there on top * scale is
// below 2^19 where top * step is below 2^22; an infinite scale times 0 is NaN). Where the
// largest logit is next to the lowest value there is, `low` does not tell -infinity from it.
__device__ __forceinline__ bool sample_wide(float top, float step, bool borders, const SampleRow& s)
{
    return (borders && (!(fabsf(top * step) < 0x1p22f) || !(fabsf(top * s.scale) < 0x1p20f) || !(s.t < 1e29f))) || top < -1e37f;
}
constexpr float kSampleNone = -46.0f;   // weights of 2^-46 and less are 0: such logits need not be counted

// 1. Each chunk of a row: its largest logit (and that one's index, for the likeliest token), and, where k or p
// is set, how many logits fall into each bin and, roughly, their weights relative to the chunk's largest: a count in
// the low 15 bits (a chunk has 2^13), the weights in fp32 as multiples of 2^-31 above, in one whole number, so that an
// addition in LDS does both and the order of additions does not matter. A bin's place is its grid line modulo
// 512, the same in every chunk. 13 us for 200 rows of 50001 (3.0 TB/s; the copy's 5.1 would be 8): the loads wait for
// each other at the barrier behind the largest logit (17 in workgroups of 1024 threads).
__global__ __launch_bounds__(kSampleThreads, 8) void sample_scan_kernel(SampleArgs a, SampleWs ws)
{
    __shared__ u64 hist[kSampleBins], all;
    __shared__ float tops[kSampleWaves];
    __shared__ int first;
    const int r = blockIdx.y, c = blockIdx.x, tid = threadIdx.x;
    const float* const x = a.logits + (ws.row0 + r) * a.stride;
    const SampleRow s = sample_row(a, ws.row0 + r);
    const int at = SampleChunk::first<kSampleWaves>(x, c);
    SampleChunk mine;
    mine.load(x, at, a.vocab);
    if (tid < kSampleBins) hist[tid] = 0;
    if (tid == 0) {
        first = INT32_MAX;
        all = 0;
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kSampleLoads; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, mine.v[j][e]);   // (NaN does not count)
    top = wave_max_all(fminf(top, 3.402823466e38f));
    if ((tid & (kWave - 1)) == 0) tops[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) top = fmaxf(top, tops[w]);
    const int64_t chunk = (int64_t)r * ws.chunks + c;
    if (tid == 0) ws.top[chunk] = top;
    if (s.greedy) {
        int here = INT32_MAX;
#pragma unroll 1
        for (int j = 0; j < kSampleLoads; ++j) {
            const floatx4_t v = mine.next();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = at + 4 * kWave * j + e;
                here = sample_logit(v[e]) == top && i >= 0 ? min(here, i) : here;
            }
        }
        if (here != INT32_MAX) atomicMin(&first, here);
        __syncthreads();
        if (tid == 0) ws.first[chunk] = first;
        return;
    }
    if (s.k == a.vocab && !(s.p < 1.0f)) return;
    u64 sum = 0;
    const float step = sample_step(s), grid = floorf(top * step), shift = 31.0f - top * s.scale;
    if (fabsf(shift) < __builtin_inff()) {   // (else nothing here counts beside another chunk, or the row is wide)
        const float scale = s.scale;
#pragma unroll 1
        for (int j = 0; j < kSampleLoads; ++j) {
            const floatx4_t v = mine.next();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float l = v[e], y = __builtin_fmaf(l, scale, shift), g = floorf(l * step);
                const uint32_t w = (uint32_t)__builtin_amdgcn_exp2f(y);
                const u64 add = (u64)w << 15 | (y >= 31.0f + kSampleNone ? 1 : 0);
                sum += add;
                if (grid - g < (float)kSampleBins) atomicAdd(&hist[(int)g & (kSampleBins - 1)], add);
            }
        }
    }
    sum = wave_scan64(sum);
    if ((tid & (kWave - 1)) == kWave - 1) atomicAdd(&all, sum);
    __syncthreads();
    if (tid < kSampleBins) ws.hist[chunk * kSampleBins + tid] = hist[tid];
    if (tid == 0) ws.all[chunk] = all;
}

// What the later launches need of a row. The weights' numbers and the logits from which on a tile has something to keep
// or to list: from (or, without borders, to keep), none (what is lower weighs nothing), and on the grid line (of all
// that is kept or listed), line_lo (in a bin before lo), line_hi (before or in hi), line_k (before bk), line_k_end (in bk).
__device__ __forceinline__ SampleFound sample_limits(const SampleArgs& a, const SampleRow& s, float top, bool wide, int lo, int hi,
                                                     int bk, bool by_k, bool by_p, uint32_t k_before)
{
    const float step = sample_step(s), inf = __builtin_inff();
    const int grid = sample_grid(top, step), deep = by_k ? max(hi, bk) : hi;
    const u64 least = sample_least(s, a.frac);
    const SampleScale es = sample_scale(top, s);
    const float slack = 0.01f + 0x1p-20f * fminf(fabsf(top * s.scale), 0x1p30f), to_logit = 0.693147181f * s.t;   // of the sums here
    const float none = fmaxf(top + (kSampleNone - slack) * to_logit, es.low);
    SampleFound f{};
    f.weights = es;
    f.least = least;
    f.top = top;
    f.lo = lo;
    f.hi = hi;
    f.bk = bk;
    f.by_k = by_k;
    f.by_p = by_p;
    f.k_before = k_before;
    f.wide = wide;
    f.every = by_p && !by_k && !wide;   // (of a wide row the draw weighs them)
    f.step = step;
    f.none = none;
    f.from = lo == kSampleBins && least ? top + (__builtin_amdgcn_logf(fminf(s.m, 1.0f)) - slack) * to_logit : none;
    f.line = deep < kSampleBins - 1 ? (float)(grid - deep) : -inf;
    f.line_lo = lo < kSampleBins ? (float)(grid - lo + 1) : -inf;
    f.line_hi = hi < kSampleBins - 1 ? (float)(grid - hi) : -inf;
    f.line_k = by_k ? (float)(grid - bk + 1) : inf;
    f.line_k_end = by_p && by_k && bk > hi ? bk < kSampleBins - 1 ? (float)(grid - bk) : -inf : inf;
    return f;
}
// By a wave: the row's answer where nothing is drawn, the likeliest token or none (top of -infinity).
__device__ __forceinline__ void sample_answer(const SampleArgs& a, const SampleWs& ws, int r, float top)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t chunk0 = (int64_t)r * ws.chunks;
    int i = INT32_MAX;
    if (top > -__builtin_inff())   // the first chunk that has it
        for (int j = lane; j < ws.chunks; j += kWave) i = ws.top[chunk0 + j] == top ? min(i, j) : i;
#pragma unroll
    for (int o = 32; o; o >>= 1) i = min(i, __shfl_xor(i, o));
    if (lane == 0) {
        a.token[ws.row0 + r] = i < ws.chunks ? ws.first[chunk0 + i] : -1;
        if (a.logprob) a.logprob[ws.row0 + r] = i < ws.chunks ? 0.0f : __builtin_nanf("");
        ws.found[r].answered = 1;
    }
}
__device__ __forceinline__ float sample_top(const SampleWs& ws, int64_t chunk0)
{
    float top = -__builtin_inff();
    for (int i = threadIdx.x & (kWave - 1); i < ws.chunks; i += kWave) top = fmaxf(top, ws.top[chunk0 + i]);
    return uniform(wave_max_all(top));
}

// 2. Each row, where k or p is set for any: the bins that a border may lie in are known but for the rough sums'
// error: [lo, hi] for the last token kept, and k's where p needs the sum of the first k. The chunks' bins are added up two
// threads to a bin's place; then one wave searches. (By every workgroup of the next launch for itself, that launch took
// 38 us for 200 x 50001 by p, 22 of its 27 thousand cycles before the first weight.)
constexpr int kFindThreads = 2 * kSampleBins;
__global__ __launch_bounds__(kFindThreads, 4) void sample_find_kernel(SampleArgs a, SampleWs ws)
{
    __shared__ float mass[2][kSampleBins];
    __shared__ uint32_t counts[2][kSampleBins];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t chunk0 = (int64_t)r * ws.chunks;
    const SampleRow s = sample_row(a, ws.row0 + r);
    // the bins of the first chunks (where there are none, they are not used; 20 take in vocabularies of 152,000)
    constexpr int kEarly = 10;
    const int q = tid & (kSampleBins - 1), half = tid / kSampleBins;
    const u64* const hists = ws.hist + chunk0 * kSampleBins + q;
    u64 early[kEarly];
#pragma unroll
    for (int i = 0; i < kEarly; ++i) early[i] = hists[(int64_t)min(half + 2 * i, ws.chunks - 1) * kSampleBins];
    const float top = sample_top(ws, chunk0);
    if (s.greedy || top == -__builtin_inff()) {
        if (wave == 0) sample_answer(a, ws, r, top);
        return;
    }
    const float step = uniform(sample_step(s)), scale = uniform(s.scale);
    const int grid = uniform(sample_grid(top, step));
    bool by_k = s.k < a.vocab;
    const bool by_p = s.p < 1.0f, borders = by_k || by_p, wide = sample_wide(top, step, borders, s);
    int lo = kSampleBins, hi = kSampleBins, bk = kSampleBins;
    uint32_t k_before = 0;
    if (wide) {   // any bin
        lo = 0;
        hi = kSampleBins - 1;
        bk = by_k ? 0 : kSampleBins;
    } else if (borders) {
        // place q of a chunk's bins holds grid line grid - b with b = (grid - q) mod 512, or one too far down
        const int b0 = (grid - q) & (kSampleBins - 1);
        float m = 0.0f;
        uint32_t n = 0;
        auto add = [&](int i, u64 h) {
            const float t = ws.top[chunk0 + i];
            const bool in = (float)b0 >= (float)grid - floorf(t * step);   // no higher than the chunk's largest
            n += in ? (uint32_t)(h & 0x7fff) : 0;
            m += in ? (float)(h >> 15) * __builtin_amdgcn_exp2f((t - top) * scale) : 0.0f;
        };
        for (int i0 = 0;;) {
#pragma unroll
            for (int i = 0; i < kEarly; ++i)
                if (i0 + half + 2 * i < ws.chunks) add(i0 + half + 2 * i, early[i]);
            i0 += 2 * kEarly;
            if (i0 >= ws.chunks) break;
#pragma unroll
            for (int i = 0; i < kEarly; ++i) early[i] = hists[(int64_t)min(i0 + half + 2 * i, ws.chunks - 1) * kSampleBins];
        }
        const bool last = b0 == kSampleBins - 1;
        mass[half][b0] = last ? 0.0f : m;
        counts[half][b0] = last ? 0 : n;
        __syncthreads();
        if (wave) return;
        float all_mass = 0.0f;
        uint32_t all_count = 0;
        for (int i = lane; i < ws.chunks; i += kWave) {
            const float y = (ws.top[chunk0 + i] - top) * scale;
            const u64 h = ws.all[chunk0 + i];
            if (y >= kSampleNone) {
                all_mass += (float)(h >> 15) * __builtin_amdgcn_exp2f(y);
                all_count += (uint32_t)(h & 0x7fff);
            }
        }
        all_mass = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_sums(all_mass)), kWave - 1));
        all_count = (uint32_t)__builtin_amdgcn_readlane((int)wave_sums(all_count), kWave - 1);
        SampleSums<float> ms;
        SampleSums<uint32_t> ns;
#pragma unroll
        for (int e = 0; e < kSampleEach; ++e) {
            ms.up[e] = mass[0][kSampleEach * lane + e] + mass[1][kSampleEach * lane + e];
            ns.up[e] = counts[0][kSampleEach * lane + e] + counts[1][kSampleEach * lane + e];
        }
        ms.scan();
        ns.scan();
        if (lane == kWave - 1) {   // the row's last bin: what none of the others holds
            ms.up[kSampleEach - 1] = fmaxf(all_mass, ms.up[kSampleEach - 1]);
            ns.up[kSampleEach - 1] = max(all_count, ns.up[kSampleEach - 1]);
        }
        by_k = by_k && (uint32_t)s.k < ns.at(kSampleBins - 1);
        if (by_k) {
            bk = ns.reach(s.k);
            k_before = ns.at(bk - 1);
        }
        if (by_p) {
            // In units of 2^-20 of a weight: 6.1 for scale (2^-22.4 of it, at 46 bits below the largest), 1.4 for the
            // argument in the scan (31 at the most), 4 for the one here (46, two roundings), 3 for the exponentials and
            // the sums of bins, a sixteenth for each chunk's sum: held as 32 and an eighth. The shift by a chunk's
            // largest logit is off by two of its roundings, each weight by a step of 2^-31.
            const float all = ms.at(kSampleBins - 1);
            const float off = (0x1p-15f + 0x1p-23f * ws.chunks + 0x1p-22f * fabsf(top * scale)) * all + (float)ns.at(kSampleBins - 1);
            const float w0 = by_k ? ms.at(bk - 1) : all, w1 = by_k ? ms.at(bk) : all, p = fmaxf(s.p, 0.0f);
            hi = min(ms.reach(p * w1 + off), by_k ? bk : kSampleBins - 1);
            lo = min(ms.reach(p * w0 - off), hi);
        } else if (by_k) {
            lo = hi = bk;
        }
    }
    if (tid == 0) {
        ws.found[r] = sample_limits(a, s, top, wide, lo, hi, bk, by_k, by_p, k_before);
        ws.listed[r] = 0;
    }
}

// 3. Each chunk again, by two workgroups: what lies before bin lo is kept and summed exactly, tile by tile, the logits
// of the bins in question go to the row's list (as places, in any order: what is done with them does not depend on it),
// by way of LDS so that a workgroup asks for its places in the list once. ALONE: no row has k or p, and each
// workgroup finds the row's numbers for itself. 21 us for 200 rows of 50001 by p, where each logit's weight counts, 14 for
// 64 of 151936 of mixed settings: issue (VALU busy for more than 80% of the cycles), a logit's 16 operations in 64 bits, the
// sum of its weight, and its tests.
constexpr int kSumWaves = kSampleWaves / kSampleParts, kSumList = 1024;
template <bool ALONE>
__global__ __launch_bounds__(kSumWaves * kWave, 8) void sample_sum_kernel(SampleArgs a, SampleWs ws)
{
    __shared__ u64 out[kSumList];
    __shared__ uint32_t place, place0;
    const int r = blockIdx.y, c = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t chunk0 = (int64_t)r * ws.chunks;
    const float* const x = a.logits + (ws.row0 + r) * a.stride;
    const int at = SampleChunk::first<kSumWaves>(x, c);
    SampleChunk chunk;
    chunk.load(x, at, a.vocab);
    SampleFound f;
    if constexpr (ALONE) {
        const SampleRow s = sample_row(a, ws.row0 + r);
        const float top = sample_top(ws, chunk0);
        if (s.greedy || top == -__builtin_inff()) {
            if (c == 0 && wave == 0) sample_answer(a, ws, r, top);
            return;
        }
        f = sample_limits(a, s, top, sample_wide(top, sample_step(s), false, s), kSampleBins, kSampleBins, kSampleBins, false,
                          false, 0);
        if (f.wide) {
            f.lo = 0;
            f.hi = kSampleBins - 1;
        }
        if (c == 0 && tid == 0) ws.found[r] = f;
    } else {
        f = ws.found[r];
        if (f.answered) return;
    }
    const bool borders = f.lo < kSampleBins;
    if (borders) {
        if (tid == 0) place = 0;
        __syncthreads();
    }
    // sums: each tile's kept weights before `lo`; the weights before `lo`; all weights that p is a part of
    const u64 least = uniform(f.least);
    const SampleScale es = {uniform(f.weights.top), uniform(f.weights.scale), uniform(f.weights.low)};
    const bool every = f.every, simple = !borders && !least;
    const float step = uniform(f.step), none = uniform(f.none), from = uniform(f.from), line = uniform(f.line);
    const float line_lo = uniform(f.line_lo), line_hi = uniform(f.line_hi), line_k = uniform(f.line_k);
    const float line_k_end = uniform(f.line_k_end);
    u64 tile = 0, before_lo = 0, part = 0;
#pragma unroll 1
    for (int j = 0; j < kSampleLoads; ++j) {
        const floatx4_t v = chunk.next();
        float l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) l[e] = sample_clamp(v[e], es.low);
        const float high = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3]));
        const bool some = __ballot((high >= from) & (high * step >= line)) && !f.wide;
        if (!some && !every) continue;
        u64 raw[4];
        sample_raw<4>(l, es, a.frac, raw);
        const u64 all = (raw[0] + raw[1]) + (raw[2] + raw[3]) - 4 * kSampleBits;
        if (every) part += all;
        if (!some) continue;
        if (simple) {
            tile += all;
        } else {
            uint32_t listed = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float g = l[e] * step;
                const u64 w = raw[e] - kSampleBits, before = g >= line_lo ? w : 0;
                tile += before >= least ? before : 0;
                before_lo += before;
                if (!every) part += g >= line_k ? w : 0;
                const bool in = (g < line_lo) & (l[e] >= none) & ((g >= line_hi) | ((g < line_k) & (g >= line_k_end)));
                listed |= in ? 1u << e : 0;
            }
            while (const uint64_t ready = __ballot(listed != 0)) {   // (a lane's in order)
                uint32_t to = 0;
                if (lane == 0) to = atomicAdd(&place, __popcll(ready));
                to = __builtin_amdgcn_readfirstlane(to) +
                     __builtin_amdgcn_mbcnt_hi((uint32_t)(ready >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ready, 0));
                if (listed) {
                    const int e = __ffs(listed) - 1;
                    const float x = e & 2 ? e & 1 ? l[3] : l[2] : e & 1 ? l[1] : l[0];
                    if (to < kSumList) out[to] = sample_place(x, at + 4 * kWave * j + e, ws.index_bits);
                    listed &= listed - 1;
                }
            }
        }
    }
    const int64_t mine = chunk0 * kSampleTiles + c * kSumWaves + wave;
    tile = wave_scan64(tile);
    if (lane == kWave - 1) ws.tiles[mine] = tile;
    if (f.by_p) {
        before_lo = wave_scan64(before_lo);
        part = wave_scan64(part);
        if (lane == kWave - 1) {
            ws.sums[2 * mine] = before_lo;
            ws.sums[2 * mine + 1] = part;
        }
    }
    if (borders) {
        __syncthreads();   // what the waves have listed
        const uint32_t n = place;
        if (n == 0) return;
        if (tid == 0) place0 = atomicAdd(&ws.listed[r], n <= kSumList ? n : kSampleList + 1);   // (too many: the row itself)
        __syncthreads();
        u64* const list = ws.list + (int64_t)r * kSampleList;
        for (uint32_t i = tid; i < min(n, (uint32_t)kSumList); i += kSumWaves * kWave)
            if (place0 + i < kSampleList) list[place0 + i] = out[i];
    }
}

// 4. Each row: the borders among the listed logits (or, where those are too many for the list, among the
// row's), and the draw. Fine bins of the listed logits, the few of a border's fine bin ranked by a wave, then the
// tile that the draw falls into and the token; as above every wave searches for itself. (Four waves, one to a SIMD: with
// sixteen the searches, the same in each, took 6 of 13 us, with eight a row 9.3 instead of 8.5.) Where the list is too
// long the row itself is searched, by its one workgroup, slower than the plain form, which sorts it (0.35 ms): 150,000
// logits of deviation 0.1 by p 0.6 ms, all equal 2.7 ms.
constexpr int kDrawThreads = 256, kDrawWaves = kDrawThreads / kWave;
struct SampleLds {
    u64 list[kSampleList], weight[kSampleList];   // places and their weights
    uint16_t bin[kSampleList];                    // fine bins, the top bit set where it is not in [lo, hi]
    u64 mass[kSampleBins];
    uint32_t counts[kSampleBins];
    u64 few[2][kWave], few_weight[2][kWave];
    u64 digit[256], digit_weight[256];
    u64 scratch[kDrawWaves];
    u64 found[3];
    u64 sums[2];
    uint32_t n_few[2];
    u64 tiles[1];   // [chunks * kSampleTiles]
};

// By one wave: the place at which the counts or weights of its n lanes' places, in order and up to `last`, sum to
// `target`; the last of them where they do not. And the sum of weights up to it.
struct SampleBorder {
    u64 place, sum;
};
__device__ __forceinline__ SampleBorder sample_rank(u64 c, u64 w, int n, u64 last, u64 target, bool count)
{
    const bool in = (int)(threadIdx.x & (kWave - 1)) < n && c <= last;
    u64 sum = 0, weights = 0;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const u64 ci = lane_value64(c, i), wi = lane_value64(w, i);
        const bool upto = ci <= c && ci <= last;
        weights += upto ? wi : 0;
        sum += upto ? count ? 1 : wi : 0;
    }
    // the first in order that reaches it, else the last
    SampleBorder b{0, 0};
    bool reached = false;
#pragma unroll 1
    for (uint64_t todo = __ballot(in); todo; todo &= todo - 1) {
        const int i = __ffsll((unsigned long long)todo) - 1;
        const u64 ci = lane_value64(c, i);
        const bool enough = lane_value64(sum, i) >= target;
        if (enough ? !reached || ci < b.place : !reached && ci >= b.place) b = {ci, lane_value64(weights, i)};
        reached |= enough;
    }
    return b;
}

// What the borders' search needs of a row.
struct SampleSearch {
    const float* x;
    SampleRow s;
    SampleScale e;
    SampleFound f;
    float step;
    int grid, V, frac, index_bits, lead, tiles, n;
    u64 least;
};

// The last place that is kept; the weights of those in [lo, hi] are added to their tiles. LIST: among the n listed
// places, else among the row's.
template <bool LIST>
__device__ __forceinline__ u64 sample_borders(const SampleSearch& q, SampleLds& lds)
{
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const SampleFound& f = q.f;
    const bool two = f.by_k && f.by_p && f.bk > f.hi;
    // fine bins: as many to each bin that is listed, by the logit's place in it
    const int fine = kSampleBins / min(f.hi - f.lo + 1 + two, kSampleBins);
    auto weigh = [&](u64 c) { return sample_weight(sample_unkey((uint32_t)(c >> q.index_bits)), q.e, q.frac); };
    auto fine_bin = [&](float l) {
        const float g = l * q.step, part = 1.0f - (g - floorf(g));
        const int b = sample_bin(l, q.grid, q.step);
        const int k = b == kSampleBins - 1 || !(part >= 0.0f) ? fine - 1 : min((int)(part * (float)fine), fine - 1);
        const int base = b > f.hi ? f.hi + 1 - f.lo : b - f.lo;
        const bool in = b >= f.lo && (b <= f.hi || (two && b == f.bk));
        return in ? min(base * fine + k, kSampleBins - 1) | (b > f.hi ? 0x8000 : 0) : 0x7fff;
    };
    // every place in question: fn(place, weight, fine bin, whether in [lo, hi])
    auto each = [&](auto&& fn) {
        if constexpr (LIST) {
#pragma unroll 1
            for (int i = tid; i < q.n; i += kDrawThreads) {
                const uint32_t b = lds.bin[i];
                fn(lds.list[i], lds.weight[i], (int)(b & 0x7fff), b < 0x8000);
            }
        } else {   // (the next four under way)
            auto load = [&](int i) {
                return i >= 0 && i + 3 < q.V ? *reinterpret_cast<const floatx4_t*>(q.x + i) : sample_edge(q.x, i, q.V);
            };
            floatx4_t next = load(4 * tid - q.lead);
#pragma unroll 1
            for (int i = 4 * tid - q.lead; i < q.V; i += 4 * kDrawThreads) {
                floatx4_t v = next;
                next = load(min(i + 4 * kDrawThreads, q.V));
#pragma unroll 1
                for (int e = 0; e < 4; ++e) {
                    const float l = sample_logit(v[0]);
                    v = floatx4_t{v[1], v[2], v[3], v[3]};
                    if (!(((double)l - q.e.top) * q.e.scale >= kSampleNone)) continue;
                    const int b = fine_bin(l);
                    const u64 c = sample_place(l, i + e, q.index_bits);
                    if (b != 0x7fff) fn(c, weigh(c), b & 0x7fff, b < 0x8000);
                }
            }
        }
    };
    if constexpr (LIST) {
#pragma unroll 1
        for (int i = tid; i < q.n; i += kDrawThreads) {
            const u64 c = lds.list[i], w = weigh(c);
            const int b = fine_bin(sample_unkey((uint32_t)(c >> q.index_bits)));
            lds.weight[i] = w;
            lds.bin[i] = (uint16_t)b;
            atomicAdd(&lds.counts[b & (kSampleBins - 1)], 1);
            atomicAdd(&lds.mass[b & (kSampleBins - 1)], w);
        }
    } else {
        each([&](u64, u64 w, int b, bool) {
            atomicAdd(&lds.counts[b], 1);
            atomicAdd(&lds.mass[b], w);
        });
    }
    __syncthreads();
    SampleSums<uint32_t> counts;
    SampleSums<u64> mass;
#pragma unroll
    for (int e = 0; e < kSampleEach; ++e) {
        counts.up[e] = lds.counts[kSampleEach * lane + e];
        mass.up[e] = lds.mass[kSampleEach * lane + e];
    }
    counts.scan();
    mass.scan();
    // The place in fine bin k at which the counts or weights of its places, up to `up_to`, sum to `target`,
    // and their sum of weights up to it: first k's, then p's.
    // (Of a wide row the bins hold all that weighs anything, and not -infinity, which the sums take for `low`, the
    // largest logit itself in rows of the lowest values.)
    u64 last = ~0ull, whole = f.wide && !f.by_k ? mass.at(kSampleBins - 1) : lds.sums[1];
    const u64 before = lds.sums[0];
#pragma unroll 1
    for (int slot = f.by_k ? 0 : 1; slot < (f.by_p ? 2 : 1); ++slot) {
        const bool count = slot == 0;
        const int first = (two ? f.hi + 1 - f.lo : f.bk - f.lo) * fine;   // bk's first fine bin
        u64 target;
        int k;
        bool there;
        if (count) {
            target = (uint32_t)q.s.k - f.k_before + counts.at(first - 1);
            k = counts.reach((uint32_t)target);
            there = counts.at(kSampleBins - 1) >= target;
            target -= counts.at(k - 1);
        } else {
            const u64 all = sample_part(q.s.p, whole, true);
            if (all <= before) {   // (as the rough sums have it, it is not)
                last = 0;
                break;
            }
            target = all - before;
            k = mass.reach(target);
            there = mass.at(kSampleBins - 1) >= target;
            target -= min(mass.at(k - 1), target - 1);
        }
        SampleBorder b{last, mass.at(k) - mass.at(k - 1)};   // (fewer with a weight: all of them)
        const int m = (int)(counts.at(k) - counts.at(k - 1));
        if (!there) {
        } else if (m <= kWave) {
            each([&](u64 c, u64 w, int b, bool) {
                if (b == k)
                    if (const uint32_t to = atomicAdd(&lds.n_few[slot], 1); to < kWave) {
                        lds.few[slot][to] = c;
                        lds.few_weight[slot][to] = w;
                    }
            });
            __syncthreads();
            b = sample_rank(lds.few[slot][lane], lds.few_weight[slot][lane], m, last, target, count);
        } else {
            // many, as equal logits are: by digits of 8 bits below what they have in common
            u64 low = ~0ull, high = 0;
            each([&](u64 c, u64, int b, bool) {
                if (b == k && c <= last) {
                    low = min(low, c);
                    high = max(high, c);
                }
            });
            __syncthreads();
            if (tid < 2) lds.found[tid] = tid ? 0 : ~0ull;
            __syncthreads();
            atomicMin(&lds.found[0], low);
            atomicMax(&lds.found[1], high);
            __syncthreads();
            low = lds.found[0];
            high = lds.found[1];
            int above = low < high ? 64 - __builtin_clzll(low ^ high) : 0;
            u64 prefix = low < high ? above < 64 ? low >> above : 0 : high, sum = 0, weights = 0;
#pragma unroll 1
            while (above > 0) {
                const int shift = max(0, above - 8);
                __syncthreads();
                if (tid < 256) lds.digit[tid] = lds.digit_weight[tid] = 0;
                if (tid < 2) lds.found[tid] = 0;
                __syncthreads();
                each([&](u64 c, u64 w, int b, bool) {
                    if (b != k || c > last || (above < 64 && c >> above != prefix)) return;
                    const int d = (int)(c >> shift) & ((1 << (above - shift)) - 1);
                    atomicAdd(&lds.digit_weight[d], w);
                    atomicAdd(&lds.digit[d], count ? 1 : w);
                    atomicMax(&lds.found[0], (u64)d);   // the last there is, should the target not be reached
                });
                __syncthreads();
                const u64 mine = tid < 256 ? lds.digit[tid] : 0, heavy = tid < 256 ? lds.digit_weight[tid] : 0;
                const int end = (int)lds.found[0];
                const u64 up = sum + block_scan(mine, lds.scratch);
                __syncthreads();
                const u64 up_weights = weights + block_scan(heavy, lds.scratch);
                if (tid <= end && up - mine < target && (up >= target || tid == end)) {
                    lds.found[1] = tid;
                    lds.found[0] = up - mine;
                    lds.found[2] = up_weights - heavy;
                }
                __syncthreads();
                prefix = prefix << (above - shift) | lds.found[1];
                sum = lds.found[0];
                weights = lds.found[2];
                above = shift;
            }
            b = {prefix, weights + weigh(prefix)};
        }
        last = b.place;
        if (count) whole += mass.at(k - 1) - mass.at(first - 1) + b.sum;
    }
    each([&](u64 c, u64 w, int, bool kept) {
        const int tile = (((uint32_t)c & ((1u << q.index_bits) - 1)) + q.lead) / kSampleTile;
        if (kept && c <= last && w >= q.least && tile < q.tiles) atomicAdd(&lds.tiles[tile], w);
    });
    return last;
}

__global__ __launch_bounds__(kDrawThreads) void sample_draw_kernel(SampleArgs a, SampleWs ws)
{
    extern __shared__ u64 sample_lds[];
    SampleLds& lds = *reinterpret_cast<SampleLds*>(sample_lds);
    const int r = blockIdx.x, row = ws.row0 + r, tid = threadIdx.x, lane = tid & (kWave - 1), V = a.vocab;
    const float* const x = a.logits + row * a.stride;
    const int lead = sample_lead(x);
    // everything that lies at a known place is loaded before any of it is waited for
    const SampleRow s = sample_row(a, row);
    const SampleFound f = ws.found[r];
    const int64_t chunk0 = (int64_t)r * ws.chunks;
    const int tiles = ws.chunks * kSampleTiles;
    const u64* const list = ws.list + (int64_t)r * kSampleList;
    constexpr int kEarly = 8;
    u64 early[kEarly];   // (what is not listed is not used)
#pragma unroll
    for (int i = 0; i < kEarly; ++i) early[i] = list[i * kDrawThreads + tid];
    const uint32_t listed = ws.listed[r];
    u64 sum0 = 0, sum1 = 0;
    for (int i = tid; i < tiles; i += kDrawThreads) {
        lds.tiles[i] = ws.tiles[chunk0 * kSampleTiles + i];
        sum0 += ws.sums[(chunk0 * kSampleTiles + i) * 2];
        sum1 += ws.sums[(chunk0 * kSampleTiles + i) * 2 + 1];
    }
    if (f.answered) return;
    const float step = f.step;
    const int grid = sample_grid(f.top, step);
    const u64 least = f.least;
    const SampleScale es = f.weights;
    u64 last = ~0ull;
    if (f.lo < kSampleBins) {
        for (int i = tid; i < kSampleBins; i += kDrawThreads) {
            lds.mass[i] = 0;
            lds.counts[i] = 0;
        }
        if (tid < 2) {
            lds.sums[tid] = 0;
            lds.n_few[tid] = 0;
        }
        const bool fits = !f.wide && listed <= kSampleList;
        const int n = fits ? (int)listed : 0;
#pragma unroll
        for (int i = 0; i < kEarly; ++i)
            if (i * kDrawThreads + tid < n) lds.list[i * kDrawThreads + tid] = early[i];
        for (int i = kEarly * kDrawThreads + tid; i < n; i += kDrawThreads) lds.list[i] = list[i];
        __syncthreads();
        if (f.by_p) {   // (additions of all threads to one place took 4 us)
            sum0 = wave_scan64(sum0);
            sum1 = wave_scan64(sum1);
            if (lane == kWave - 1) {
                atomicAdd(&lds.sums[0], sum0);
                atomicAdd(&lds.sums[1], sum1);
            }
        }
        const SampleSearch q{x, s, es, f, step, grid, V, a.frac, ws.index_bits, lead, tiles, n, least};
        last = fits ? sample_borders<true>(q, lds) : sample_borders<false>(q, lds);
    }
    __syncthreads();

    // the tile that the draw falls into: a run of tiles to a lane
    const int run = (tiles + kWave - 1) / kWave;
    u64 sum = 0;
#pragma unroll 1
    for (int i = lane * run; i < min((lane + 1) * run, tiles); ++i) sum += lds.tiles[i];
    const u64 runs = wave_scan64(sum), total = lane_value64(runs, kWave - 1);
    u64 target = sample_part(s.u, total, false);
    const uint64_t past = __ballot(runs > target);
    int tile = (past ? __ffsll((unsigned long long)past) - 1 : 0) * run;
    target -= past ? lane_value64(runs - sum, tile / run) : 0;
#pragma unroll 1
    for (; tile < tiles - 1 && lds.tiles[tile] <= target; ++tile) target -= lds.tiles[tile];
    // its token: four to a thread
    static_assert(kSampleTile <= 4 * kDrawThreads, "a tile to a workgroup");
    const int at = tile * kSampleTile + 4 * tid - lead;
    u64 w[4] = {}, mine = 0;
    if (4 * tid < kSampleTile) {
        const floatx4_t v = at >= 0 && at + 3 < V ? *reinterpret_cast<const floatx4_t*>(x + at) : sample_edge(x, at, V);
        float l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) l[e] = sample_clamp(v[e], es.low);
        sample_raw<4>(l, es, a.frac, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = v[e] > -__builtin_inff() &&
                            (sample_place(l[e], at + e, ws.index_bits) <= last || sample_bin(l[e], grid, step) < f.lo);
            const u64 we = in ? w[e] - kSampleBits : 0;
            w[e] = we >= least ? we : 0;
            mine += w[e];
        }
    }
    u64 up_to = block_scan(mine, lds.scratch);
    if (up_to > target && up_to - mine <= target) {
        up_to -= mine;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            up_to += w[e];
            if (up_to > target) {
                a.token[row] = at + e;
                if (a.logprob) a.logprob[row] = (float)log((double)w[e] / (double)total);
                break;
            }
        }
    }
}

}  // namespace msnb
