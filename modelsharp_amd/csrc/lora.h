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

// The tile's tokens' adapters in lanes 0..15 (-1: none; -2: no token), one class after another.
struct LoraClasses {
    int mine;          // this lane's token's (lane % 16)
    uint32_t left;     // tokens whose class has not come yet
    __device__ __forceinline__ LoraClasses(const LoraArgs& p, int t0)
    {
        const int t = t0 + (threadIdx.x & 15);
        const int a = t < p.T ? p.which[t] : -2;
        mine = t < p.T && (unsigned)a >= (unsigned)p.adapters ? -1 : a;
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

template <typename T>
__device__ __forceinline__ float lora_rank(const LoraArgs& p, int a)
{
    return p.ranks ? min(max(p.ranks[a], 0), p.rank) : p.rank;
}

// E consecutive values from base + at as fp32, those from `n` on zero (base + at .. + n - 1 may
// be read); vec: whole 16- or 8-byte loads, then n is 0 or at least E where E divides the row.
template <int E, typename T>
__device__ __forceinline__ void lora_load(float (&x)[E], const T* base, int64_t at, int n, int vec)
{
    typedef T tv __attribute__((ext_vector_type(E)));
    if (vec && n >= E) {
        const tv v = *reinterpret_cast<const tv*>(base + at);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = i < n ? (float)base[at + i] : 0.0f;
    }
}

// grid: tiles * slots * splits; slot s takes the tile's classes s, s + slots, ... RT: rank tiles of
// 16 at a time. The four waves take every fourth step of 32 of the split's K.
template <typename T, int RT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs p, int slots)
{
    __shared__ floatx4_t sums[4][RT][kWave];
    const int sp = blockIdx.x % p.splits, rest = blockIdx.x / p.splits;
    const int slot = rest % slots, t0 = rest / slots * kLoraTokens;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, grp = lane >> 4, t = t0 + l16;
    const int steps = (p.K + 31) / 32, per = (steps + p.splits - 1) / p.splits;
    const int s0 = sp * per, s1 = min(steps, s0 + per);
    const float* const x = p.x + (int64_t)min(t, p.T - 1) * p.K;
    LoraClasses cls(p, t0);
    for (int c = 0; cls.left; ++c) {
        const int a = cls.next();
        if (c % slots != slot || a < 0) continue;
        const int rank = lora_rank<T>(p, a);
        const T* const A = static_cast<const T*>(p.a) + (int64_t)a * p.rank * p.K;
        for (int r0 = 0; r0 < rank; r0 += 16 * RT) {
            floatx4_t acc[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt] = floatx4_t{};
            for (int s = s0 + wave; s < s1; s += 4) {
                const int k = 32 * s + 8 * grp;
                float xv[8], av[RT][8];
                lora_load<4>(*reinterpret_cast<float(*)[4]>(xv), x, k, p.K - k, p.vec);
                lora_load<4>(*reinterpret_cast<float(*)[4]>(xv + 4), x, k + 4, p.K - k - 4, p.vec);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const int r = r0 + 16 * rt + l16;
                    lora_load<8>(av[rt], A, (int64_t)min(r, rank - 1) * p.K + k, r < rank ? p.K - k : 0, p.vec);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        acc[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[rt][j], xv[j], acc[rt], 0, 0, 0);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sums[wave][rt][lane] = acc[rt];
            __syncthreads();
            for (int rt = wave; rt < RT; rt += 4) {
                const floatx4_t v = (sums[0][rt][lane] + sums[1][rt][lane]) + (sums[2][rt][lane] + sums[3][rt][lane]);
                const int r = r0 + 16 * rt + 4 * grp;
                if (cls.mine == a && r < p.rank16)
                    *reinterpret_cast<floatx4_t*>(p.h + ((int64_t)sp * p.T + t) * p.rank16 + r) = v;
            }
            __syncthreads();
        }
    }
}

// grid: tiles * slots * ceil(N / 256); a wave takes 64 outputs of the tile's 16 tokens.
template <typename T>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs p, int slots)
{
    const int nb = (p.N + kLoraRows - 1) / kLoraRows;
    const int rest = blockIdx.x / nb, slot = rest % slots, t0 = rest / slots * kLoraTokens;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, grp = lane >> 4, t = t0 + l16;
    const int n0 = blockIdx.x % nb * kLoraRows + 64 * wave;
    LoraClasses cls(p, t0);
    for (int c = 0; cls.left; ++c) {
        const int a = cls.next();
        if (c % slots != slot || (a < 0 && p.base == p.y)) continue;
        const int rank = a < 0 ? 0 : lora_rank<T>(p, a);
        const float scale = a < 0 || !p.scales ? 1.0f : p.scales[a];
        const T* const B = static_cast<const T*>(p.b) + (int64_t)max(a, 0) * p.N * p.rank;
        floatx4_t acc[4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) acc[nt] = floatx4_t{};
        for (int r0 = 0; r0 < rank; r0 += 16) {
            const int r = r0 + 4 * grp;
            floatx4_t h{};
            if (cls.mine == a)
                for (int s = 0; s < p.splits; ++s)
                    h += *reinterpret_cast<const floatx4_t*>(p.h + ((int64_t)s * p.T + t) * p.rank16 + r);
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = r + j < rank ? h[j] : 0.0f;   // past it: 0 * x, NaN where x is not finite
            float bv[4][4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                const int n = min(n0 + 16 * nt + l16, p.N - 1);
                lora_load<4>(bv[nt], B, (int64_t)n * p.rank + r, rank - r, p.vec);
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[nt][j], h[j], acc[nt], 0, 0, 0);
        }
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            if (cls.mine != a) continue;
            const int n = n0 + 16 * nt + 4 * grp;
            const int64_t at = (int64_t)t * p.N + n;
            if (p.vec && n < p.N) {
                const floatx4_t b = p.base ? *reinterpret_cast<const floatx4_t*>(p.base + at) : floatx4_t{};
                *reinterpret_cast<floatx4_t*>(p.y + at) = a < 0 ? b : b + scale * acc[nt];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.N) {
                        const float b = p.base ? p.base[at + i] : 0.0f;
                        p.y[at + i] = a < 0 ? b : b + scale * acc[nt][i];
                    }
            }
        }
    }
}

}  // namespace msnb
