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
__device__ __forceinline__ u64 block_scan(u64 x, u64 (&scratch)[kSampleWaves])
{
    const int wave = threadIdx.x >> 6;
    x = wave_scan64(x);
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) scratch[wave] = x;
    __syncthreads();
    u64 before = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves - 1; ++w) {
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
__device__ __forceinline__ floatx4_t sample_load(const float* x, int i, int V)
{
    floatx4_t v;
    if (i >= 0 && i + 3 < V) {
        v = *reinterpret_cast<const floatx4_t*>(x + i);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e >= 0 && i + e < V ? x[i + e] : -__builtin_inff();
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = sample_logit(v[e]);
    return v;
}

// Bins of logits on a grid that does not depend on the row: of a sixteenth, or a sixteenth of t where t is
// below 1, so that the 512 from the largest logit's down reach weights of e^-32 (t up to 1) or 32 below it; the last
// one holds all that is lower. A bin of 150,000 normal logits of deviation 2 has at most 1900.
__device__ __forceinline__ float sample_step(const SampleRow& s) { return 16.0f / fminf(s.t, 1.0f); }
__device__ __forceinline__ int sample_grid(float l, float step)
{
    return (int)floorf(fminf(fmaxf(l * step, -0x1p29f), 0x1p29f));
}
__device__ __forceinline__ int sample_bin(float l, int top_grid, float step)
{
    return min(top_grid - sample_grid(l, step), kSampleBins - 1);
}

// 1. Each chunk of a row: its largest logit (and that one's index, for the likeliest token), and, where k or p
// is set, how many logits fall into each bin and, roughly, their weights relative to the chunk's largest: a count in
// the low 15 bits (a chunk has 2^14), the weights in fp32 as multiples of 2^-31 above, in one whole number, so that an
// addition in LDS does both and the order of additions does not matter. A bin's place is its grid line modulo
// 512, the same in every chunk.
__global__ __launch_bounds__(kSampleThreads) void sample_scan_kernel(SampleArgs a, SampleWs ws)
{
    __shared__ u64 hist[kSampleBins], all;
    __shared__ float tops[kSampleWaves];
    __shared__ int first;
    const int r = blockIdx.y, c = blockIdx.x, tid = threadIdx.x;
    const float* const x = a.logits + (ws.row0 + r) * a.stride;
    const SampleRow s = sample_row(a, ws.row0 + r);
    const int at = c * kSampleTile * kSampleTiles + 4 * tid - sample_lead(x);
    floatx4_t v[kSampleTiles];
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j) v[j] = sample_load(x, at + j * kSampleTile, a.vocab);
    if (tid < kSampleBins) hist[tid] = 0;
    if (tid == 0) {
        first = INT32_MAX;
        all = 0;
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, v[j][e]);
    top = wave_max_all(top);
    if ((tid & (kWave - 1)) == 0) tops[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) top = fmaxf(top, tops[w]);
    const int64_t chunk = (int64_t)r * ws.chunks + c;
    if (tid == 0) ws.top[chunk] = top;
    if (s.greedy) {
        int mine = INT32_MAX;
#pragma unroll
        for (int j = kSampleTiles - 1; j >= 0; --j)
#pragma unroll
            for (int e = 3; e >= 0; --e) mine = v[j][e] == top && at + j * kSampleTile + e >= 0 ? at + j * kSampleTile + e : mine;
        if (mine != INT32_MAX) atomicMin(&first, mine);
        __syncthreads();
        if (tid == 0) ws.first[chunk] = first;
        return;
    }
    if (s.k == a.vocab && !(s.p < 1.0f)) return;
    u64 sum = 0;
    if (top > -__builtin_inff()) {
        const float step = sample_step(s), scale = (float)s.scale;
        const int grid = sample_grid(top, step);
#pragma unroll
        for (int j = 0; j < kSampleTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float l = v[j][e];
                const float w = l == top ? 1.0f : sample_rough(l - top, scale);
                const u64 add = l > -__builtin_inff() ? (u64)(uint32_t)__builtin_fmaf(w, 0x1p31f, 0.5f) << 15 | 1 : 0;
                const int g = sample_grid(l, step);
                sum += add;
                if (add && grid - g < kSampleBins) atomicAdd(&hist[g & (kSampleBins - 1)], add);
            }
    }
    sum = wave_scan64(sum);
    if ((tid & (kWave - 1)) == kWave - 1) atomicAdd(&all, sum);
    __syncthreads();
    if (tid < kSampleBins) ws.hist[chunk * kSampleBins + tid] = hist[tid];
    if (tid == 0) ws.all[chunk] = all;
}

// 2. Each chunk again, with the whole row's largest logit and bins. The bins that a border may lie in are known but
// for the rough sums' error: [lo, hi] for the last token kept, and k's where p needs the sum of the first k. Their
// logits go to the row's list (as places, in the chunks' order); what lies before them is kept and summed
// exactly, tile by tile. Every workgroup adds up the chunks' bins for itself (4 KB each, from L2, a chunk to a wave), and
// every wave finds the borders' bins for itself: what is waited for is one round of loads and three barriers. (With a
// barrier at each step of the search this launch took 54 us for 64 x 151936 of mixed settings.)
__global__ __launch_bounds__(kSampleThreads, 8) void sample_sum_kernel(SampleArgs a, SampleWs ws)
{
    __shared__ u64 mass[kSampleBins], all_mass, sums[kSampleTiles + 2];
    __shared__ uint32_t counts[kSampleBins], all_count, place;
    const int r = blockIdx.y, c = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t chunk0 = (int64_t)r * ws.chunks;
    const float* const x = a.logits + (ws.row0 + r) * a.stride;
    const SampleRow s = sample_row(a, ws.row0 + r);
    const int at = c * kSampleTile * kSampleTiles + 4 * tid - sample_lead(x);
    floatx4_t v[kSampleTiles];
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j) v[j] = sample_load(x, at + j * kSampleTile, a.vocab);
    if (tid < kSampleBins) {
        mass[tid] = 0;
        counts[tid] = 0;
    }
    if (tid < kSampleTiles + 2) sums[tid] = 0;
    if (tid == 0) {
        all_mass = 0;
        all_count = place = 0;
    }
    float top = -__builtin_inff();
    int which = 0;
    for (int i = lane; i < ws.chunks; i += kWave) {
        const float t = ws.top[chunk0 + i];
        which = t > top ? i : which;
        top = fmaxf(top, t);
    }
    const float mine = top;
    top = wave_max_all(top);
    if (s.greedy || top == -__builtin_inff()) {   // the first chunk that has it; nothing to draw from
        if (c == 0 && wave == 0) {
            int i = top > -__builtin_inff() && mine == top ? which : INT32_MAX;
#pragma unroll
            for (int o = 32; o; o >>= 1) i = min(i, __shfl_xor(i, o));
            if (lane == 0) {
                a.token[ws.row0 + r] = i < ws.chunks ? ws.first[chunk0 + i] : -1;
                if (a.logprob) a.logprob[ws.row0 + r] = i < ws.chunks ? 0.0f : __builtin_nanf("");
                ws.found[r].answered = 1;
            }
        }
        return;
    }
    const float step = sample_step(s);
    const int grid = sample_grid(top, step);
    bool by_k = s.k < a.vocab;
    const bool by_p = s.p < 1.0f;
    int lo = kSampleBins, hi = kSampleBins, bk = kSampleBins;
    uint32_t k_before = 0, listed = 0;
    __syncthreads();
    if (by_k || by_p) {
        // a lane has eight places of a chunk's bins; place q holds grid line grid - b with b = (grid - q) mod 512
        const u64* const hists = ws.hist + chunk0 * kSampleBins;
        for (int i = wave; i < ws.chunks; i += kSampleWaves) {
            const float ti = ws.top[chunk0 + i];
            if (ti == -__builtin_inff()) continue;
            const float f = ti == top ? 1.0f : sample_rough(ti - top, (float)s.scale);
            const int below = grid - sample_grid(ti, step);   // the chunk's bins begin so far below the row's
            const u64 rest = ws.all[chunk0 + i];
#pragma unroll
            for (int e = 0; e < kSampleEach; ++e) {
                const u64 h = hists[(int64_t)i * kSampleBins + kSampleEach * lane + e];
                const int b = (grid - (kSampleEach * lane + e)) & (kSampleBins - 1);
                if (h && b >= below && b < kSampleBins - 1) {
                    atomicAdd(&mass[b], (u64)((double)(h >> 15) * f));
                    atomicAdd(&counts[b], (uint32_t)(h & 0x7fff));
                }
            }
            if (lane == 0) {
                atomicAdd(&all_mass, (u64)((double)(rest >> 15) * f));
                atomicAdd(&all_count, (uint32_t)(rest & 0x7fff));
            }
        }
        __syncthreads();
        SampleSums<float> m;
        SampleSums<uint32_t> n;
#pragma unroll
        for (int e = 0; e < kSampleEach; ++e) {
            m.up[e] = (float)mass[kSampleEach * lane + e];
            n.up[e] = counts[kSampleEach * lane + e];
        }
        m.scan();
        n.scan();
        if (lane == kWave - 1) {   // the row's last bin: what none of the others holds
            m.up[kSampleEach - 1] = (float)all_mass;
            n.up[kSampleEach - 1] = all_count;
        }
        by_k = by_k && (uint32_t)s.k < all_count;
        if (by_k) {
            bk = n.reach(s.k);
            k_before = n.at(bk - 1);
        }
        if (by_p) {
            // two of fp32's exponentials, off by 2^-17 each (arguments up to 64, rounded twice), a sum in fp32, half a
            // step for each logit and a step of each bin and chunk
            const float off = 0x1p-14f * (float)all_mass + (float)all_count + (float)ws.chunks * kSampleBins;
            const float w0 = m.at(by_k ? bk - 1 : kSampleBins - 1), w1 = m.at(by_k ? bk : kSampleBins - 1);
            const float p = fmaxf(s.p, 0.0f);
            hi = min(m.reach(p * w1 + off), by_k ? bk : kSampleBins - 1);
            lo = min(m.reach(p * w0 - off), hi);
        } else if (by_k) {
            lo = hi = bk;
        }
        // how many are listed, and how many of them by the chunks before this one
        if (lo < kSampleBins) {
            const bool two = by_p && by_k && bk > hi;
            listed = n.at(hi) - n.at(lo - 1) + (two ? n.at(bk) - n.at(bk - 1) : 0);
            for (int i = wave; i < c; i += kSampleWaves) {
                const float ti = ws.top[chunk0 + i];
                if (ti == -__builtin_inff()) continue;
                const int below = grid - sample_grid(ti, step);
                u64 in = 0;      // listed, and in any bin but the last
#pragma unroll
                for (int e = 0; e < kSampleEach; ++e) {
                    const u64 h = hists[(int64_t)i * kSampleBins + kSampleEach * lane + e] & 0x7fff;
                    const int b = (grid - (kSampleEach * lane + e)) & (kSampleBins - 1);
                    if (b >= below && b < kSampleBins - 1) in += h << 32 | ((b >= lo && b <= hi) || (two && b == bk) ? h : 0);
                }
                in = wave_scan64(in);
                if (lane == kWave - 1) {
                    const bool last = hi == kSampleBins - 1 || (two && bk == kSampleBins - 1);
                    atomicAdd(&place, (uint32_t)in + (last ? (uint32_t)(ws.all[chunk0 + i] & 0x7fff) - (uint32_t)(in >> 32) : 0));
                }
            }
            __syncthreads();
        }
    }
    const bool list = listed && listed <= kSampleList;
    if (c == 0 && tid == 0) ws.found[r] = {top, lo, hi, bk, by_k, by_p, k_before, list ? listed : 0, 0, 0};

    // sums: each tile's kept weights before `lo`; the weights before `lo`; all weights that p is a part of
    const u64 least = sample_least(s, a.frac);
    const int whole = by_p ? by_k ? bk : kSampleBins : 0, bins = max(lo, whole);
    u64* const out = ws.list + (int64_t)r * kSampleList;
    u64 before_lo = 0, part = 0;
#pragma unroll
    for (int j = 0; j < kSampleTiles; ++j) {
        int b[4];
        bool any = false, some = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            b[e] = lo < kSampleBins ? sample_bin(v[j][e], grid, step) : 0;
            b[e] = v[j][e] == -__builtin_inff() ? kSampleBins : b[e];
            any |= b[e] < bins;
            some |= b[e] >= lo && (b[e] <= hi || b[e] == bk);
        }
        if (__ballot(any)) {
            u64 tile = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u64 w = sample_weight(v[j][e], top, s, a.frac);
                const u64 before = b[e] < lo ? w : 0;
                tile += before >= least ? before : 0;
                before_lo += before;
                part += b[e] < whole ? w : 0;
            }
            tile = wave_scan64(tile);
            if (lane == kWave - 1) atomicAdd(&sums[j], tile);
        }
        if (list && some)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (b[e] < kSampleBins && ((b[e] >= lo && b[e] <= hi) || (by_p && b[e] == bk)))
                    if (const uint32_t to = atomicAdd(&place, 1); to < kSampleList)   // (or the logits have changed since)
                        out[to] = sample_place(v[j][e], at + j * kSampleTile + e, ws.index_bits);
    }
    if (by_p) {
        before_lo = wave_scan64(before_lo);
        part = wave_scan64(part);
        if (lane == kWave - 1) {
            atomicAdd(&sums[kSampleTiles], before_lo);
            atomicAdd(&sums[kSampleTiles + 1], part);
        }
    }
    __syncthreads();
    if (tid < kSampleTiles) ws.tiles[(chunk0 + c) * kSampleTiles + tid] = sums[tid];
    else if (tid < kSampleTiles + 2) ws.sums[(chunk0 + c) * 2 + tid - kSampleTiles] = sums[tid];
}

// 3. Each row: the borders among the listed logits (or, where those are too many for the list, among the
// row's), and the draw. Fine bins of the listed logits, the few of a border's fine bin ranked by a wave, then the
// tile that the draw falls into and the token; as above every wave searches for itself.
struct SampleLds {
    u64 list[kSampleList];
    u64 mass[kSampleBins];
    uint32_t counts[kSampleBins];
    u64 few[2][kWave];
    u64 digit[256], digit_weight[256];
    u64 scratch[kSampleWaves];
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
    for (int i = 0; i < n; ++i) {
        const u64 ci = lane_value64(c, i), wi = lane_value64(w, i);
        const bool upto = ci <= c && ci <= last;
        weights += upto ? wi : 0;
        sum += upto ? count ? 1 : wi : 0;
    }
    // the first in order that reaches it, else the last
    SampleBorder b{0, 0};
    bool reached = false;
    for (uint64_t todo = __ballot(in); todo; todo &= todo - 1) {
        const int i = __ffsll((unsigned long long)todo) - 1;
        const u64 ci = lane_value64(c, i);
        const bool enough = lane_value64(sum, i) >= target;
        if (enough ? !reached || ci < b.place : !reached && ci >= b.place) b = {ci, lane_value64(weights, i)};
        reached |= enough;
    }
    return b;
}

__global__ __launch_bounds__(kSampleThreads) void sample_draw_kernel(SampleArgs a, SampleWs ws)
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
    u64 early[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) early[i] = ws.list[(int64_t)r * kSampleList + i * kSampleThreads + tid];
    u64 sum0 = 0, sum1 = 0;
    for (int i = tid; i < ws.chunks; i += kSampleThreads) {
        sum0 += ws.sums[(chunk0 + i) * 2];
        sum1 += ws.sums[(chunk0 + i) * 2 + 1];
    }
    for (int i = tid; i < tiles; i += kSampleThreads) lds.tiles[i] = ws.tiles[chunk0 * kSampleTiles + i];
    if (s.greedy || f.answered) return;
    const float step = sample_step(s);
    const int grid = sample_grid(f.top, step);
    const u64 least = sample_least(s, a.frac);
    const int n = (int)f.listed;   // 0: the row itself
    u64 last = ~0ull;
    auto weight = [&](float l) { return sample_weight(l, f.top, s, a.frac); };
    auto place_weight = [&](u64 c) { return weight(sample_unkey((uint32_t)(c >> ws.index_bits))); };
    if (f.lo < kSampleBins) {
        const bool two = f.by_k && f.by_p && f.bk > f.hi;
        // fine bins: as many to each bin that is listed, by the logit's place in it
        const int fine = kSampleBins / min(f.hi - f.lo + 1 + two, kSampleBins);
        auto fine_bin = [&](float l, int b) {
            const float q = l * step, part = 1.0f - (q - floorf(q));
            const int k = b == kSampleBins - 1 || !(part >= 0.0f) ? fine - 1 : min((int)(part * (float)fine), fine - 1);
            return min((b > f.hi ? f.hi + 1 - f.lo : b - f.lo) * fine + k, kSampleBins - 1);
        };
        // every listed place: fn(place, logit, fine bin, whether in [lo, hi])
        auto each = [&](auto&& fn) {
            const int m = n ? n : V;
            for (int i = tid; i < m; i += kSampleThreads) {
                const u64 c = n ? lds.list[i] : sample_place(sample_logit(x[i]), i, ws.index_bits);
                const float l = sample_unkey((uint32_t)(c >> ws.index_bits));
                if (l == -__builtin_inff()) continue;
                const int b = sample_bin(l, grid, step);
                if ((b >= f.lo && b <= f.hi) || (two && b == f.bk)) fn(c, l, fine_bin(l, b), b <= f.hi);
            }
        };
        if (tid < kSampleBins) {
            lds.mass[tid] = 0;
            lds.counts[tid] = 0;
        }
        if (tid < 2) {
            lds.sums[tid] = 0;
            lds.n_few[tid] = 0;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i * kSampleThreads + tid < n) lds.list[i * kSampleThreads + tid] = early[i];
        for (int i = 2 * kSampleThreads + tid; i < n; i += kSampleThreads) lds.list[i] = ws.list[(int64_t)r * kSampleList + i];
        __syncthreads();
        if (f.by_p && sum0 | sum1) {
            atomicAdd(&lds.sums[0], sum0);
            atomicAdd(&lds.sums[1], sum1);
        }
        each([&](u64, float l, int k, bool) {
            atomicAdd(&lds.counts[k], 1);
            if (f.by_p) atomicAdd(&lds.mass[k], weight(l));
        });
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
        // and their sum of weights up to it.
        auto border = [&](int slot, int k, u64 up_to, u64 target, bool count) -> SampleBorder {
            const int m = (int)(counts.at(k) - counts.at(k - 1));
            if (m <= kWave) {
                each([&](u64 c, float, int b, bool) {
                    if (b == k)
                        if (const uint32_t to = atomicAdd(&lds.n_few[slot], 1); to < kWave) lds.few[slot][to] = c;
                });
                __syncthreads();
                const u64 c = lds.few[slot][lane];
                return sample_rank(c, place_weight(c), m, up_to, target, count);
            }
            // many, as equal logits are: by digits of 8 bits below what they have in common
            u64 low = ~0ull, high = 0;
            each([&](u64 c, float, int b, bool) {
                if (b == k && c <= up_to) {
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
            if (low >= high) return {high, place_weight(high)};
            int above = 64 - __builtin_clzll(low ^ high);
            u64 prefix = above < 64 ? low >> above : 0, before = 0, weights = 0;
            while (above > 0) {
                const int shift = max(0, above - 8);
                __syncthreads();
                if (tid < 256) lds.digit[tid] = lds.digit_weight[tid] = 0;
                if (tid < 2) lds.found[tid] = 0;
                __syncthreads();
                each([&](u64 c, float l, int b, bool) {
                    if (b != k || c > up_to || (above < 64 && c >> above != prefix)) return;
                    const int d = (int)(c >> shift) & ((1 << (above - shift)) - 1);
                    const u64 w = weight(l);
                    atomicAdd(&lds.digit_weight[d], w);
                    atomicAdd(&lds.digit[d], count ? 1 : w);
                    atomicMax(&lds.found[0], (u64)d);   // the last there is, should the target not be reached
                });
                __syncthreads();
                const u64 mine = tid < 256 ? lds.digit[tid] : 0, heavy = tid < 256 ? lds.digit_weight[tid] : 0;
                const int end = (int)lds.found[0];
                const u64 up = before + block_scan(mine, lds.scratch);
                __syncthreads();
                const u64 up_weights = weights + block_scan(heavy, lds.scratch);
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
            return {prefix, weights + place_weight(prefix)};
        };
        u64 whole = lds.sums[1];   // what p is a part of
        if (f.by_k) {
            const int first = (two ? f.hi + 1 - f.lo : f.bk - f.lo) * fine;   // bk's first fine bin
            const uint32_t target = (uint32_t)s.k - f.k_before + counts.at(first - 1);
            const int k = counts.reach(target);
            const SampleBorder q = border(0, k, ~0ull, target - counts.at(k - 1), true);
            last = q.place;
            whole += mass.at(k - 1) - mass.at(first - 1) + q.sum;
        }
        if (f.by_p) {
            const u64 all = sample_part(s.p, whole, true), before = lds.sums[0], target = all > before ? all - before : 0;
            const int k = mass.reach(target);
            last = target ? border(1, k, last, target - min(mass.at(k - 1), target - 1), false).place : 0;
        }
        each([&](u64 c, float l, int, bool kept) {
            const u64 w = weight(l);
            const int tile = (((uint32_t)c & ((1u << ws.index_bits) - 1)) + lead) / kSampleTile;
            if (kept && c <= last && w >= least && tile < tiles) atomicAdd(&lds.tiles[tile], w);
        });
    }
    __syncthreads();

    // the tile that the draw falls into: a run of tiles to a lane
    const int run = (tiles + kWave - 1) / kWave;
    u64 sum = 0;
    for (int i = lane * run; i < min((lane + 1) * run, tiles); ++i) sum += lds.tiles[i];
    const u64 runs = wave_scan64(sum), total = lane_value64(runs, kWave - 1);
    u64 target = sample_part(s.u, total, false);
    const uint64_t past = __ballot(runs > target);
    int tile = (past ? __ffsll((unsigned long long)past) - 1 : 0) * run;
    target -= past ? lane_value64(runs - sum, tile / run) : 0;
    for (; tile < tiles - 1 && lds.tiles[tile] <= target; ++tile) target -= lds.tiles[tile];
    // its token
    const int at = tile * kSampleTile + 4 * tid - lead;
    u64 w[4], mine = 0;
    const floatx4_t v = sample_load(x, at, V);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool kept = v[e] > -__builtin_inff() &&
                          (sample_place(v[e], at + e, ws.index_bits) <= last || sample_bin(v[e], grid, step) < f.lo);
        const u64 we = kept ? weight(v[e]) : 0;
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
                a.token[row] = at + e;
                if (a.logprob) a.logprob[row] = (float)log((double)w[e] / (double)total);
                break;
            }
        }
    }
}

}  // namespace msnb
