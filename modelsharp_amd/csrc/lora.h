// lora.h — low-rank adapters of many requests beside a shared projection:
//
//   y[t] = base[t] + scale[a] B_a (A_a x[t]),   a = which[t]  (no adapter: y[t] = base[t])
//
// with A_a [rank, K] and B_a [N, rank]. Tokens are taken 16 at a time, in their order; the
// distinct adapters among the 16 are the tile's classes, and each class is a product on the fp32
// matrix cores of which the class's own columns are kept: no sorting, no copies, and every output
// has one writer, so that results do not depend on the order of anything.
//
//   lora_shrink_kernel   h[split][t] = A_a x[t] over the split's part of K
//   lora_expand_kernel   y[t] = base[t] + scale[a] (B_a (sum of the splits' h[t]))
#pragma once
#include "serving.h"

namespace msnb {

constexpr int kLoraTokens = 16;   // tokens of a tile
constexpr int kLoraRows = 256;    // outputs of an expand workgroup

// A tile's tokens' adapters in lanes 0..15 (-1: none; -2: no token), one class after another.
struct LoraClasses {
    int mine;          // this lane's token's (lane % 16)
    uint32_t left;     // tokens whose class has not come yet
    __device__ __forceinline__ explicit LoraClasses(int adapter) : mine(adapter)
    {
        left = (uint32_t)__ballot(mine != -2) & 0xffffu;
    }
    // the next class's adapter; call while left != 0
    __device__ __forceinline__ int next()
    {
        const int a = __builtin_amdgcn_readlane(mine, __ffs(left) - 1);
        left &= ~(uint32_t)__ballot(mine == a);
        return a;
    }
};
__device__ __forceinline__ int lora_adapter(const LoraArgs& p, int t)
{
    const int a = p.which[min(t, p.T - 1)];
    return t >= p.T ? -2 : (unsigned)a >= (unsigned)p.adapters ? -1 : a;
}

__device__ __forceinline__ int lora_rank(const LoraArgs& p, int a)
{
    return p.ranks ? min(max(p.ranks[a], 0), p.rank) : p.rank;
}

// E consecutive values from base + at, those from `n` on zero; vec: one load, then n is at most 0 or
// at least E wherever E divides the row.
template <int E, typename T>
__device__ __forceinline__ auto lora_load(const T* base, int64_t at, int n, int vec)
{
    typedef T tv __attribute__((ext_vector_type(E)));
    tv x{};
    if (vec && n >= E) {
        x = *reinterpret_cast<const tv*>(base + at);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < n) x[i] = base[at + i];
    }
    return x;
}

// grid: tiles * rank groups * slots * splits; slot s takes the tile's classes s, s + slots, ... The
// waves take every WAVES'th step of 32 of the split's K, the next steps' loads in flight meanwhile,
// and meet in LDS. RT: rank tiles of 16 in a group.
template <typename T, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void lora_shrink_kernel(LoraArgs p, int slots)
{
    __shared__ floatx4_t sums[WAVES][RT][kWave];
    const int sp = blockIdx.x % p.splits, rest = blockIdx.x / p.splits;
    const int slot = rest % slots, groups = (p.rank16 + 16 * RT - 1) / (16 * RT);
    const int r0 = rest / slots % groups * (16 * RT), t0 = rest / slots / groups * kLoraTokens;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, grp = lane >> 4, t = t0 + l16;
    const int steps = (p.K + 31) / 32, per = (steps + p.splits - 1) / p.splits;
    const int s0 = sp * per, s1 = min(steps, s0 + per);
    const float* const x = p.x + (int64_t)min(t, p.T - 1) * p.K;
    LoraClasses cls(lora_adapter(p, t));
    for (int c = 0; cls.left; ++c) {
        const int a = cls.next();
        if (c % slots != slot || a < 0) continue;
        const int rank = lora_rank(p, a);
        if (r0 >= rank) continue;
        const T* const A = static_cast<const T*>(p.a) + (int64_t)a * p.rank * p.K;
        struct Step {
            floatx4_t x[2];
            T __attribute__((ext_vector_type(8))) a[RT];
        };
        auto load = [&](int s, Step& v) {
            const int k = 32 * s + 8 * grp;
            v.x[0] = lora_load<4>(x, k, p.K - k, p.vec);
            v.x[1] = lora_load<4>(x, k + 4, p.K - k - 4, p.vec);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int r = r0 + 16 * rt + l16;
                v.a[rt] = lora_load<8>(A, (int64_t)min(r, rank - 1) * p.K + k, r < rank ? p.K - k : 0, p.vec);
            }
        };
        floatx4_t acc[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt] = floatx4_t{};
        auto add = [&](const Step& v) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    acc[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)v.a[rt][j], v.x[j >> 2][j & 3], acc[rt], 0, 0, 0);
        };
        constexpr int kRing = 3;
        Step ring[kRing];
        int s = s0 + wave;
#pragma unroll
        for (int n = 0; n + 1 < kRing; ++n)
            if (s + WAVES * n < s1) load(s + WAVES * n, ring[n]);
        while (s < s1) {
#pragma unroll
            for (int n = 0; n < kRing; ++n) {
                if (s >= s1) break;
                if (s + WAVES * (kRing - 1) < s1) load(s + WAVES * (kRing - 1), ring[(n + kRing - 1) % kRing]);
                add(ring[n]);
                s += WAVES;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sums[wave][rt][lane] = acc[rt];
        __syncthreads();
        if (wave < RT) {
            floatx4_t v = sums[0][wave][lane];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) v += sums[w][wave][lane];
            const int r = r0 + 16 * wave + 4 * grp;
            if (cls.mine == a && r < p.rank16)
                *reinterpret_cast<floatx4_t*>(p.h + ((int64_t)sp * p.T + t) * p.rank16 + r) = v;
        }
        __syncthreads();
    }
}

// The products of a chunk of C = 16 or 32 ranks: B's rows n (lane % 16) and the tokens' h (lane % 16),
// E = C / 4 ranks in a row a lane. fp16 weights go to the fp16 matrix cores as they are, h as two
// halves of h 2^-e (22 bits, e by token: any fp32 h fits); fp32 weights to the fp32 ones.
template <int E>
struct LoraHalves {
    _Float16 __attribute__((ext_vector_type(E))) hi, lo;
    __device__ __forceinline__ void set(const float (&x)[E], int e)
    {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float v = __builtin_amdgcn_ldexpf(x[j], -e);
            hi[j] = (_Float16)v;
            lo[j] = (_Float16)(v - (float)hi[j]);
        }
    }
};

// grid: tiles of 16 `sub` tokens * slots * ceil(N / 256); a wave takes 64 outputs of 16 tokens after 16, B_a
// staying in its registers as long as the class does, CH chunks of C ranks at a time. What does not
// depend on the class (the base, h) is on its way before the class is known, the next 16 tokens'
// while these are worked on. ONE: h has one split.
// Memory bounds it: base and y once, 8 bytes an output against 2 ranks flops.
template <typename T, int C, int CH, bool ONE>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs p, int slots, int subs)
{
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int E = C / 4;
    const int nb = (p.N + kLoraRows - 1) / kLoraRows;
    const int rest = blockIdx.x / nb, slot = rest % slots, t00 = rest / slots * (kLoraTokens * subs);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, grp = lane >> 4;
    const int n0 = blockIdx.x % nb * kLoraRows + 64 * wave;
    typedef T bvec_t __attribute__((ext_vector_type(E)));
    bvec_t bv[CH][4];
    int held = -1;   // whose ranks 0 .. C CH - 1 those are
    struct Ahead {
        int adapter;
        floatx4_t base[4], h[ONE ? CH : 1][ONE ? E / 4 : 1];
    };
    auto fetch = [&](int t0, Ahead& x) {
        const int t = t0 + l16;
        const bool in = t < p.T;
        x.adapter = lora_adapter(p, t);
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            const int n = n0 + 16 * nt + 4 * grp;
            x.base[nt] = p.base && in ? lora_load<4>(p.base, (int64_t)t * p.N + n, p.N - n, p.vec) : floatx4_t{};
        }
        if constexpr (ONE)
#pragma unroll
            for (int q = 0; q < CH; ++q)
#pragma unroll
                for (int e = 0; e < E / 4; ++e) {
                    const int r = min(C * q + E * grp + 4 * e, p.rank16 - 4);
                    x.h[q][e] = *reinterpret_cast<const floatx4_t*>(p.h + (int64_t)min(t, p.T - 1) * p.rank16 + r);
                }
    };
    Ahead next;
    fetch(t00, next);
#pragma unroll 1
    for (int sub = 0; sub < subs; ++sub) {
        const int t0 = t00 + kLoraTokens * sub, t = t0 + l16;
        if (t0 >= p.T) return;
        const Ahead now = next;
        if (sub + 1 < subs) fetch(t0 + kLoraTokens, next);
        LoraClasses cls(now.adapter);
        for (int c = 0; cls.left; ++c) {
            const int a = cls.next();
            if (c % slots != slot || (a < 0 && p.base == p.y)) continue;
            const int rank = a < 0 ? 0 : lora_rank(p, a);
            const float scale = a < 0 || !p.scales ? 1.0f : p.scales[a];
            const T* const B = static_cast<const T*>(p.b) + (int64_t)max(a, 0) * p.N * p.rank;
            const bool mine = cls.mine == a;
            floatx4_t sum[4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) sum[nt] = floatx4_t{};
            for (int r0 = 0; r0 < rank; r0 += C * CH) {
                if (held != a || r0 > 0 || rank > C * CH) {
#pragma unroll
                    for (int q = 0; q < CH; ++q)
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt) {
                            const int n = min(n0 + 16 * nt + l16, p.N - 1), r = r0 + C * q + E * grp;
                            bv[q][nt] = lora_load<E>(B, (int64_t)n * p.rank + r, rank - r, p.vec);
                        }
                    held = r0 == 0 ? a : -1;
                }
                float h[CH][E], mx = 0.0f;
#pragma unroll
                for (int q = 0; q < CH; ++q) {
                    const int r = r0 + C * q + E * grp;
#pragma unroll
                    for (int j = 0; j < E; ++j) h[q][j] = 0.0f;
                    if (ONE && r0 == 0) {
#pragma unroll
                        for (int j = 0; j < E; ++j) h[q][j] = now.h[ONE ? q : 0][ONE ? j >> 2 : 0][j & 3];
                    } else if (mine && r < p.rank16) {
                        constexpr int kAtOnce = ONE ? 1 : 8;   // splits, added in their order
                        const float* const src = p.h + (int64_t)t * p.rank16 + r;
                        const int64_t step = (int64_t)p.T * p.rank16;
                        for (int s0 = 0; s0 < p.splits; s0 += kAtOnce) {
                            floatx4_t v[kAtOnce][E / 4];
#pragma unroll
                            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                                for (int e = 0; e < E / 4; ++e)
                                    v[i][e] = *reinterpret_cast<const floatx4_t*>(src + min(s0 + i, p.splits - 1) * step + 4 * e);
#pragma unroll
                            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                                for (int j = 0; j < E; ++j) h[q][j] += s0 + i < p.splits ? v[i][j >> 2][j & 3] : 0.0f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < E; ++j) {   // other tokens' and other ranks' were not written
                        h[q][j] = mine && r + j < rank ? h[q][j] : 0.0f;
                        mx = fmaxf(mx, fabsf(h[q][j]));
                    }
                }
                if constexpr (F16) {
                    mx = fmaxf(mx, xor16_value(mx));
                    mx = fmaxf(mx, xor32_value(mx));
                    const int e = mx > 0.0f && mx < __builtin_inff() ? __builtin_amdgcn_frexp_expf(mx) - 15 : 0;
                    floatx4_t acc[4];
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt) acc[nt] = floatx4_t{};
#pragma unroll
                    for (int q = 0; q < CH; ++q) {
                        LoraHalves<E> x;
                        x.set(h[q], e);
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt) {
                            if constexpr (C == 32) {
                                acc[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv[q][nt], x.lo, acc[nt], 0, 0, 0);
                                acc[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv[q][nt], x.hi, acc[nt], 0, 0, 0);
                            } else {
                                acc[nt] = __builtin_amdgcn_mfma_f32_16x16x16f16(bv[q][nt], x.lo, acc[nt], 0, 0, 0);
                                acc[nt] = __builtin_amdgcn_mfma_f32_16x16x16f16(bv[q][nt], x.hi, acc[nt], 0, 0, 0);
                            }
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sum[nt][i] += __builtin_amdgcn_ldexpf(acc[nt][i], e);
                } else {
#pragma unroll
                    for (int q = 0; q < CH; ++q)
#pragma unroll
                        for (int j = 0; j < E; ++j)
#pragma unroll
                            for (int nt = 0; nt < 4; ++nt)
                                sum[nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[q][nt][j], h[q][j], sum[nt], 0, 0, 0);
                }
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                const int n = n0 + 16 * nt + 4 * grp;
                const int64_t at = (int64_t)t * p.N + n;
                const floatx4_t y = a < 0 ? now.base[nt] : now.base[nt] + scale * sum[nt];
                if (!mine) continue;
                if (p.vec && n < p.N) {
                    *reinterpret_cast<floatx4_t*>(p.y + at) = y;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < p.N) p.y[at + i] = y[i];
                }
            }
        }
    }
}

}  // namespace msnb
