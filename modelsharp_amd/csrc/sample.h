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
__device__ __forceinline__ u64 sample_place(float l, int i) { return (u64)sample_key(l) << 32 | (uint32_t)i; }

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

constexpr int kSampleThreads = 1024;

template <typename T>
__device__ __forceinline__ T wave_sum_all(T x)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
// Sum over the workgroup, in every thread.
__device__ __forceinline__ u64 block_sum(u64 x, u64 (&scratch)[kSampleThreads / kWave])
{
    x = wave_sum_all(x);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int w = 0; w < kSampleThreads / kWave; ++w) s += scratch[w];
    return s;
}
__device__ __forceinline__ float block_max(float x, u64 (&scratch)[kSampleThreads / kWave])
{
#pragma unroll
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) scratch[threadIdx.x >> 6] = __float_as_uint(x);
    __syncthreads();
    float s = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kSampleThreads / kWave; ++w) s = fmaxf(s, __uint_as_float((uint32_t)scratch[w]));
    return s;
}

// A row by one workgroup, reading it once for every 8 bits of a border.
__global__ __launch_bounds__(kSampleThreads) void sample_any_kernel(SampleArgs a)
{
    __shared__ u64 hist[256], scratch[kSampleThreads / kWave], found[4];
    const int r = blockIdx.x, tid = threadIdx.x, V = a.vocab;
    const float* const x = a.logits + r * a.stride;
    const SampleRow s = sample_row(a, r);

    float top = -__builtin_inff();
    for (int i = tid; i < V; i += kSampleThreads) top = fmaxf(top, sample_logit(x[i]));
    top = block_max(top, scratch);
    if (top == -__builtin_inff()) {   // nothing to draw from
        if (tid == 0) {
            a.token[r] = -1;
            if (a.logprob) a.logprob[r] = __builtin_nanf("");
        }
        return;
    }

    // The place of the last token that a sum over the order needs to reach `target`, of counts or weights.
    const int index_bits = 32 - __builtin_clz(max(V - 1, 1));
    auto border = [&](u64 target, bool count) {
        u64 lo = 0, before = 0;
        for (int shift = 56;;) {
            for (int i = tid; i < 256; i += kSampleThreads) hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += kSampleThreads) {
                const float l = sample_logit(x[i]);
                const u64 c = sample_place(l, i);
                if (shift == 56 || c >> (shift + 8) == lo >> (shift + 8))
                    atomicAdd(&hist[(c >> shift) & 255], count ? 1 : sample_weight(l, top, s, a.frac));
            }
            __syncthreads();
            if (tid == 0) {
                int b = 0;
                u64 sum = before;
                while (b < 255 && sum + hist[b] < target) sum += hist[b++];
                found[0] = b;
                found[1] = sum;
            }
            __syncthreads();
            lo |= found[0] << shift;
            before = found[1];
            if (shift == 0) return lo;
            shift = shift > 32 ? shift - 8 : shift == 32 ? (index_bits + 7) / 8 * 8 - 8 : shift - 8;
        }
    };
    auto weight_up_to = [&](u64 last, u64 least) {
        u64 sum = 0;
        for (int i = tid; i < V; i += kSampleThreads) {
            const float l = sample_logit(x[i]);
            const u64 w = sample_place(l, i) <= last ? sample_weight(l, top, s, a.frac) : 0;
            sum += w >= least ? w : 0;
        }
        return block_sum(sum, scratch);
    };
    u64 last = ~0ull;
    if (s.greedy)
        last = border(1, true);
    else if (s.k < V)
        last = border(s.k, true);
    if (!s.greedy && s.p < 1.0f) last = border(sample_part(s.p, weight_up_to(last, 0), true), false);
    // (m above 1 keeps the likeliest, as 1 does)
    const u64 least = s.greedy || !(s.m > 0.0f) ? 0 : (u64)__builtin_rint(__builtin_ldexp((double)fminf(s.m, 1.0f), a.frac));
    const u64 total = weight_up_to(last, least);
    const u64 target = sample_part(s.u, total, false);

    // the first by index whose sum passes the target: blocks of 1024 in order
    u64 before = 0;
    for (int base = 0; base < V; base += kSampleThreads) {
        const int i = base + tid;
        u64 w = 0;
        if (i < V) {
            const float l = sample_logit(x[i]);
            w = sample_place(l, i) <= last ? sample_weight(l, top, s, a.frac) : 0;
            if (w < least) w = 0;
        }
        const u64 all = block_sum(w, scratch);
        if (before + all > target) {   // uniform: here
            u64 sum = w;
#pragma unroll
            for (int o = 1; o < kWave; o <<= 1) {
                const u64 y = __shfl_up(sum, o);
                if ((tid & (kWave - 1)) >= o) sum += y;
            }
            __syncthreads();
            if ((tid & (kWave - 1)) == kWave - 1) scratch[tid >> 6] = sum;
            __syncthreads();
            sum += before;
            for (int v = 0; v < tid >> 6; ++v) sum += scratch[v];
            if (sum > target && sum - w <= target) {
                a.token[r] = i;
                if (a.logprob) a.logprob[r] = (float)log((double)w / (double)total);
            }
            return;
        }
        before += all;
    }
}

}  // namespace msnb
