// lora.h — low-rank adapters of many requests beside a shared projection:
//
//   y[t] = base[t] + scale[a] B_a (A_a x[t]),   a = which[t]  (no adapter: y[t] = base[t])
//
// with A_a [rank, K] and B_a [N, rank]. Tokens are taken 16 at a time, in their order; the
// distinct adapters among the 16 are the tile's classes, and each class is a product on the fp32
// matrix cores of which the class's own columns are kept: no sorting, no copies, and every output
// has one writer, so that results do not depend on the order of anything.
//
//   lora_shrink_kernel,      h[split][t] = A_a x[t] over the split's part of K, zeros past the
//   lora_shrink_lds_kernel   adapter's rank (the second one: many tiles)
//   lora_expand_kernel       y[t] = base[t] + scale[a] (B_a (sum of the splits' h[t]))
//
// x and the sums are fp32; beside fp16 weights h is two fp16 halves (22 bits), as they are otherwise.
// 32 tokens, 16 adapters of rank 16, K = N = 3584: 6.0 and 5.9 us, two launches each of a few round
// trips to memory. 2048 tokens, rank 64, K = 4096, N = 11008: 19.5 us (1.7 TB/s of x, the fp32 matrix
// cores busy 40% of the cycles) and 44 us (4.1 TB/s of base and y).
#pragma once
#include "mfma_device.h"
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

// E consecutive values from base + at, of which n are there (VEC: all E, or none: then the last E,
// so that the load needs no branch). The others are zero without VEC, anything with it.
template <int E, bool VEC, typename T>
__device__ __forceinline__ auto lora_load(const T* base, int64_t at, int n)
{
    typedef T tv __attribute__((ext_vector_type(E)));
    if constexpr (VEC) {
        return *reinterpret_cast<const tv*>(base + (at + min(n - E, 0)));
    } else {
        tv x{};
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < n) x[i] = base[at + i];
        return x;
    }
}

// The first n of v's E values, zeros after them: by whole dwords, whatever the others hold.
template <int E, typename T>
__device__ __forceinline__ void lora_keep(T __attribute__((ext_vector_type(E))) & v, int n)
{
    typedef uint32_t dwords_t __attribute__((ext_vector_type(E * sizeof(T) / 4)));
    constexpr int P = 4 / sizeof(T);   // values of a dword
    dwords_t d = __builtin_bit_cast(dwords_t, v);
#pragma unroll
    for (int i = 0; i < E / P; ++i) d[i] &= n >= P * (i + 1) ? ~0u : n > P * i ? 0xffffu : 0u;
    v = __builtin_bit_cast(T __attribute__((ext_vector_type(E))), d);
}

// grid: tiles * rank groups * slots * splits; slot s takes the tile's classes s, s + slots, ... The
// waves take every WAVES'th step of 32 of the split's K, the next steps' loads in flight meanwhile,
// and meet in LDS. RT: rank tiles of 16 in a group.
template <typename T, int RT, int WAVES, bool VEC>
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
        const int rank = lora_rank(p, a);   // 0: nothing to add up, h is written as zeros
        const T* const A = static_cast<const T*>(p.a) + (int64_t)a * p.rank * p.K;
        struct Step {
            floatx4_t x[2];
            T __attribute__((ext_vector_type(8))) a[RT];
        };
        auto load = [&](int s, Step& v) {
            // rows of A past the rank stand for its last: their sums are not used
            const int k = 32 * s + 8 * grp;
            v.x[0] = lora_load<4, VEC>(x, k, p.K - k);
            v.x[1] = lora_load<4, VEC>(x, k + 4, p.K - k - 4);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                v.a[rt] = lora_load<8, VEC>(A, (int64_t)min(r0 + 16 * rt + l16, rank - 1) * p.K + k, p.K - k);
        };
        const bool any = r0 < rank;
        floatx4_t acc[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt] = floatx4_t{};
        auto add = [&](int s, Step& v) {
            if (VEC && 32 * s + 32 > p.K && 32 * s + 8 * grp >= p.K) {   // the last step's lanes past K
                v.x[0] = v.x[1] = floatx4_t{};
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) v.a[rt] = decltype(v.a[rt] + v.a[rt]){};
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    acc[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)v.a[rt][j], v.x[j >> 2][j & 3], acc[rt], 0, 0, 0);
        };
        constexpr int kRing = 3;
        Step ring[kRing];
        // every load is made, past the last step that one's again: behind a load under a condition the
        // compiler could only wait for all that is under way
        int s = s0 + wave;
        if (any && s < s1) {
#pragma unroll
            for (int n = 0; n + 1 < kRing; ++n) load(min(s + WAVES * n, s1 - 1), ring[n]);
            for (bool more = true; more;) {
#pragma unroll
                for (int n = 0; n < kRing; ++n) {
                    load(min(s + WAVES * (kRing - 1), s1 - 1), ring[(n + kRing - 1) % kRing]);
                    add(s, ring[n]);
                    s += WAVES;
                    if (!(more = s < s1)) break;
                }
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
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r + i < rank ? v[i] : 0.0f;
            if (cls.mine == a && r < p.rank16)
                *reinterpret_cast<floatx4_t*>(p.h + ((int64_t)sp * p.T + t) * p.rank16 + r) = v;
        }
        __syncthreads();
    }
}

// The same for many tiles: grid tiles * rank groups * slots * splits. A
// wave's steps go straight from memory to its own part of LDS, three under way, and no wave waits
// for another before the end. The products' operands want 16 rows side by side, and loaded that
// way every lane touches a line of its own, 64 cycles an instruction: with 2048 tokens, K = 4096
// and rank 64 that is 15.6 us by count, of the 24 that the launch took. Here 8 (fp16: 4) lanes take a row's part in a
// line, and the chunks of a row are turned by its number, so that the reads meet no bank twice.
constexpr int kLoraLdsWaves = 8, kLoraLdsRing = 3;
template <typename T, int RT>
constexpr int lora_lds_stage() { return 2048 + RT * 16 * 32 * (int)sizeof(T); }   // x, then A's rank tiles
template <typename T, int RT>
constexpr int lora_lds_bytes() { return kLoraLdsWaves * kLoraLdsRing * lora_lds_stage<T, RT>(); }
template <typename T, int RT>
__global__ __launch_bounds__(64 * kLoraLdsWaves) void lora_shrink_lds_kernel(LoraArgs p, int slots)
{
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int STAGE = lora_lds_stage<T, RT>(), LOADS = 2 + RT * (F16 ? 1 : 2);
    constexpr int AC = F16 ? 4 : 8;   // 16-byte chunks of a row of A's step
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int groups = (p.rank16 + 16 * RT - 1) / (16 * RT);
    const int sp = blockIdx.x % p.splits, rest = blockIdx.x / p.splits, slot = rest % slots;
    const int r0 = rest / slots % groups * (16 * RT), t0 = rest / slots / groups * kLoraTokens;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, grp = lane >> 4, t = t0 + l16;
    const int all = (p.K + 31) / 32, per = (all + p.splits - 1) / p.splits;
    const int first = sp * per, steps = min(all, first + per);
    uint8_t* const mine = lds + wave * kLoraLdsRing * STAGE;
    const uint32_t base = lds_address(mine);
    // what is past the last token, the adapter's rank or K reads as zero
    const __amdgpu_buffer_rsrc_t rx = buffer_rsrc(p.x + (int64_t)t0 * p.K, min(kLoraTokens, p.T - t0) * p.K * 4);
    int xoff[2], aoff[F16 ? 1 : 2];   // of step 0; and the first k of each
    const int xk = 4 * ((lane & 7) ^ (lane >> 3 & 7));
#pragma unroll
    for (int i = 0; i < 2; ++i) xoff[i] = ((8 * i + (lane >> 3)) * p.K + xk) * 4;
    const int arow = lane / AC, ak = F16 ? 8 * ((lane & 3) ^ (arow >> 1 & 3)) : xk;
#pragma unroll
    for (int i = 0; i < (F16 ? 1 : 2); ++i) aoff[i] = ((8 * i + arow) * p.K + ak) * (int)sizeof(T);
    LoraClasses cls(lora_adapter(p, t));
    for (int c = 0; cls.left; ++c) {
        const int a = cls.next();
        if (c % slots != slot || a < 0) continue;
        const int rank = __builtin_amdgcn_readfirstlane(lora_rank(p, a));
        const T* const A = static_cast<const T*>(p.a) + ((int64_t)a * p.rank + r0) * p.K;
        // (uniform, which the compiler does not see of a value read across lanes in a loop)
        const uint64_t at = (uint64_t)__builtin_amdgcn_readfirstlane((int)((uintptr_t)A >> 32)) << 32 |
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)(uintptr_t)A);
        const __amdgpu_buffer_rsrc_t ra =
            buffer_rsrc(reinterpret_cast<const void*>(at),
                        __builtin_amdgcn_readfirstlane(max(0, min(16 * RT, rank - r0)) * p.K * (int)sizeof(T)));
        auto issue = [&](int s, int slot) {   // past the last step: zeros, so that the waits' counts hold
            const uint32_t m0 = __builtin_amdgcn_readfirstlane(base) + slot * STAGE;
            const bool in = s < steps;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                lds_load16(rx, in && 32 * s + xk < p.K ? xoff[i] + 128 * s : kOOB, 0, m0 + 1024 * i);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < (F16 ? 1 : 2); ++i)
                    lds_load16(ra, in && 32 * s + ak < p.K ? aoff[i] + (16 * rt * p.K + 32 * s) * (int)sizeof(T) : kOOB, 0,
                               m0 + 2048 + 1024 * (rt * (F16 ? 1 : 2) + i));
        };
        floatx4_t acc[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt] = floatx4_t{};
        auto add = [&](int slot) {
            const uint8_t* const st = mine + slot * STAGE;
            floatx4_t x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                x[e] = *reinterpret_cast<const floatx4_t*>(st + l16 * 128 + ((2 * grp + e) ^ (l16 & 7)) * 16);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float av[8];
                const uint8_t* const ar = st + 2048 + rt * 16 * 32 * sizeof(T);
                if constexpr (F16) {
                    const auto v = *reinterpret_cast<const _Float16 __attribute__((ext_vector_type(8)))*>(
                        ar + l16 * 64 + (grp ^ (l16 >> 1 & 3)) * 16);
#pragma unroll
                    for (int j = 0; j < 8; ++j) av[j] = (float)v[j];
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const floatx4_t v =
                            *reinterpret_cast<const floatx4_t*>(ar + l16 * 128 + ((2 * grp + e) ^ (l16 & 7)) * 16);
#pragma unroll
                        for (int j = 0; j < 4; ++j) av[4 * e + j] = v[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    acc[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[j], x[j >> 2][j & 3], acc[rt], 0, 0, 0);
            }
        };
        if (r0 < rank) {
#pragma unroll
            for (int n = 0; n + 1 < kLoraLdsRing; ++n) issue(first + wave + kLoraLdsWaves * n, n);
            for (int s = first + wave, slot = 0; s < steps; s += kLoraLdsWaves) {
                const int free_slot = slot == 0 ? kLoraLdsRing - 1 : slot - 1;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // that slot's reads are done
                issue(s + kLoraLdsWaves * (kLoraLdsRing - 1), free_slot);
                wait_vmcnt<(kLoraLdsRing - 1) * LOADS>();
                add(slot);
                slot = slot + 1 == kLoraLdsRing ? 0 : slot + 1;
            }
            wait_vmcnt<0>();
        }
        __syncthreads();
        floatx4_t* const sums = reinterpret_cast<floatx4_t*>(lds);   // [wave][RT][lane]
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sums[(wave * RT + rt) * kWave + lane] = acc[rt];
        __syncthreads();
        if (wave < RT) {
            floatx4_t v = sums[wave * kWave + lane];
#pragma unroll
            for (int w = 1; w < kLoraLdsWaves; ++w) v += sums[(w * RT + wave) * kWave + lane];
            const int r = r0 + 16 * wave + 4 * grp;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r + i < rank ? v[i] : 0.0f;
            if (cls.mine == a && r < p.rank16)
                *reinterpret_cast<floatx4_t*>(p.h + ((int64_t)sp * p.T + t) * p.rank16 + r) = v;
        }
        __syncthreads();
    }
}

// grid: tiles of 16 `subs` tokens * slots * ceil(N / 256). For 16 tokens after 16:
//   the threads take h (4 ranks of a token each, the splits added in their order) to LDS: for fp16
//     weights as two halves of h 2^-e (kLowExp: 22 bits down to 2^-28 of the token's largest, then an
//     error of 2^-51 of that; e by token, so that any fp32 h fits);
//   each wave multiplies 64 rows of B_a, in its registers as long as the class does not change, with
//     each class's tokens, and leaves scale * sum in LDS;
//   the threads add it to the base and store, whole rows of 1 KB at a time.
// (A wave's sums lie 16 tokens by 16 outputs: stored from there, every instruction touches 16 lines,
// and the launch took 65 us in place of 44 at 2048 tokens of N = 11008.)
// R ranks at a time, in chunks of C; more come in further passes over the sums in LDS. ONE: h has
// one split, and the base and h of the next 16 tokens are on their way meanwhile. No load or store of
// that loop is under a condition, behind which the compiler could only wait for all that is under way:
// what is not wanted goes to an offset that the buffer does not have. VEC: B's ranks are read by
// fours or eights, base and y by fours; 0: value by value. (64 tokens of rank 64: eights 25.1 us, fours
// 28.1; 40 of rank 20: fours 12.7, value by value 29.9.)
// Memory bounds it: base and y once, 8 bytes an output against 2 ranks flops.
template <typename T, int C, int CH, bool ONE, int VEC>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs p, int slots, int subs)
{
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int E = C / 4, R = C * CH, LPT = R / 4;   // ranks of a lane's operand; lanes that take a token's h
    constexpr int HS = R + (F16 ? 8 : 4), YS = kLoraRows + 4;   // strides off the powers of two
    typedef T bvec_t __attribute__((ext_vector_type(E)));
    __shared__ floatx4_t ys[kLoraTokens * YS / 4];
    __shared__ floatx4_t hs[(F16 ? 2 * 2 : 4) * kLoraTokens * HS / 16];
    __shared__ int exps[kLoraTokens];
    T* const h0 = reinterpret_cast<T*>(hs);   // [token][HS], fp16: the high halves, then the low ones
    float* const yl = reinterpret_cast<float*>(ys);

    const int nb = (p.N + kLoraRows - 1) / kLoraRows;
    const int rest = blockIdx.x / nb, slot = rest % slots, t00 = rest / slots * (kLoraTokens * subs);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, grp = lane >> 4;
    const int n0 = blockIdx.x % nb * kLoraRows;
    const int ht = tid / LPT, hr = 4 * (tid % LPT);   // this thread's token and ranks of h (if ht < 16)
    bvec_t bv[CH][4];
    int held = -1;   // whose ranks 0 .. R - 1 those are

    struct Ahead {
        int adapter;
        floatx4_t base[4], h;
    };
    auto fetch = [&](int t0, Ahead& x) {
        x.adapter = lora_adapter(p, t0 + l16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // token 4 wave + i, outputs 4 lane ..
            const int t = min(t0 + 4 * wave + i, p.T - 1), n = n0 + 4 * lane;
            x.base[i] = p.base ? lora_load<4, (VEC > 0)>(p.base, (int64_t)t * p.N + n, p.N - n) : floatx4_t{};
        }
        if constexpr (ONE)
            x.h = *reinterpret_cast<const floatx4_t*>(p.h + (int64_t)min(t0 + min(ht, 15), p.T - 1) * p.rank16 +
                                                      min(hr, p.rank16 - 4));
    };
    Ahead next;
    fetch(t00, next);
#pragma unroll 1
    for (int sub = 0; sub < subs; ++sub) {
        const int t0 = t00 + kLoraTokens * sub;
        if (t0 >= p.T) return;
        const __amdgpu_buffer_rsrc_t rows = buffer_rsrc(p.y + (int64_t)t0 * p.N, 64 * p.N);   // these tokens' of y
        const Ahead now = next;
        if (subs > 1) fetch(min(t0 + kLoraTokens, p.T - 1), next);   // past the last: not used
        uint32_t done = 0, adds = 0;   // tokens of this workgroup's classes, and those with an adapter
        for (int r0 = 0; r0 < p.rank16; r0 += R) {
            if (ht < kLoraTokens) {
                floatx4_t h = now.h;
                const int r = r0 + hr;
                if (!ONE || r0 > 0) {
                    constexpr int kAtOnce = ONE ? 1 : 8;
                    const float* const src = p.h + (int64_t)min(t0 + ht, p.T - 1) * p.rank16 + min(r, p.rank16 - 4);
                    const int64_t step = (int64_t)p.T * p.rank16;
                    h = floatx4_t{};
                    for (int s0 = 0; s0 < p.splits; s0 += kAtOnce) {
                        floatx4_t v[kAtOnce];
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i)
                            v[i] = *reinterpret_cast<const floatx4_t*>(src + min(s0 + i, p.splits - 1) * step);
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) h[j] += s0 + i < p.splits ? v[i][j] : 0.0f;
                    }
                }
                if (r >= p.rank16) h = floatx4_t{};
                if constexpr (F16) {
                    float mx = fmaxf(fmaxf(fabsf(h[0]), fabsf(h[1])), fmaxf(fabsf(h[2]), fabsf(h[3])));
                    mx = fmaxf(mx, dpp_read<0xB1>(mx));
                    mx = fmaxf(mx, dpp_read<0x4E>(mx));
                    if constexpr (LPT >= 8) mx = fmaxf(mx, dpp_read<0x141>(mx));
                    if constexpr (LPT >= 16) mx = fmaxf(mx, dpp_read<0x140>(mx));
                    const int e = mx > 0.0f && mx < __builtin_inff() ? __builtin_amdgcn_frexp_expf(mx) - 15 : 0;
                    _Float16 __attribute__((ext_vector_type(4))) hi, lo;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float v = __builtin_amdgcn_ldexpf(h[j], -e);
                        hi[j] = (_Float16)v;
                        lo[j] = (_Float16)((v - (float)hi[j]) * (1 << kLowExp));
                    }
                    *reinterpret_cast<decltype(hi)*>(h0 + ht * HS + hr) = hi;
                    *reinterpret_cast<decltype(lo)*>(h0 + (kLoraTokens + ht) * HS + hr) = lo;
                    if (hr == 0) exps[ht] = e;
                } else {
                    *reinterpret_cast<floatx4_t*>(h0 + ht * HS + hr) = h;
                }
            }
            __syncthreads();
            LoraClasses cls(now.adapter);
            bvec_t hv[F16 ? 2 : 1][CH];   // this lane's token's
#pragma unroll
            for (int q = 0; q < CH; ++q)
#pragma unroll
                for (int k = 0; k < (F16 ? 2 : 1); ++k)
                    hv[k][q] = *reinterpret_cast<const bvec_t*>(h0 + (kLoraTokens * k + l16) * HS + C * q + E * grp);
            const int e = F16 ? exps[l16] : 0;
            for (int c = 0; cls.left; ++c) {
                const uint32_t before = cls.left;
                const int a = cls.next();
                if (c % slots != slot) continue;
                done |= before & ~cls.left;
                if (a < 0) continue;
                adds |= before & ~cls.left;
                const int rank = lora_rank(p, a);
                const float scale = p.scales ? p.scales[a] : 1.0f;
                const T* const B = static_cast<const T*>(p.b) + (int64_t)a * p.N * p.rank;
                if (held != a || p.rank16 > R) {
#pragma unroll
                    for (int q = 0; q < CH; ++q)
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt) {
                            const int n = min(n0 + 64 * wave + 16 * nt + l16, p.N - 1), r = r0 + C * q + E * grp;
                            const int64_t at = (int64_t)n * p.rank + r;
                            if constexpr (E == 8 && VEC == 4)
                                bv[q][nt] = __builtin_shufflevector(lora_load<4, true>(B, at, p.rank - r),
                                                                    lora_load<4, true>(B, at + 4, p.rank - r - 4), 0, 1, 2,
                                                                    3, 4, 5, 6, 7);
                            else
                                bv[q][nt] = lora_load<E, (VEC > 0)>(B, at, p.rank - r);
                        }
                    if (rank < r0 + R)   // columns past the adapter's own rank are not its values
#pragma unroll
                        for (int q = 0; q < CH; ++q)
#pragma unroll
                            for (int nt = 0; nt < 4; ++nt) lora_keep<E, T>(bv[q][nt], rank - (r0 + C * q + E * grp));
                    held = a;
                }
                floatx4_t acc[4], low[4];
#pragma unroll
                for (int nt = 0; nt < 4; ++nt) acc[nt] = low[nt] = floatx4_t{};
#pragma unroll
                for (int q = 0; q < CH; ++q)
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt) {
                        if constexpr (F16) {
#pragma unroll
                            for (int k = 1; k >= 0; --k) {
                                floatx4_t& sum = k ? low[nt] : acc[nt];
                                if constexpr (C == 32)
                                    sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv[q][nt], hv[k][q], sum, 0, 0, 0);
                                else
                                    sum = __builtin_amdgcn_mfma_f32_16x16x16f16(bv[q][nt], hv[k][q], sum, 0, 0, 0);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < E; ++j)
                                acc[nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[q][nt][j], hv[0][q][j], acc[nt], 0, 0, 0);
                        }
                    }
                if (cls.mine == a)
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt) {
                        floatx4_t* const y = reinterpret_cast<floatx4_t*>(yl + l16 * YS + 64 * wave + 16 * nt + 4 * grp);
                        floatx4_t v;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            v[i] = scale * (F16 ? __builtin_amdgcn_ldexpf(__builtin_fmaf(low[nt][i], kLow, acc[nt][i]), e)
                                                : acc[nt][i]);
                        *y = r0 == 0 ? v : *y + v;
                    }
            }
            __syncthreads();
        }
        if (p.base == p.y) done &= adds;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tok = 4 * wave + i, n = n0 + 4 * lane;
            const floatx4_t sum = *reinterpret_cast<const floatx4_t*>(yl + tok * YS + 4 * lane);
            const floatx4_t y = adds >> tok & 1 ? now.base[i] + sum : now.base[i];
            const bool mine = done >> tok & 1;
            if constexpr (VEC > 0) {
                const int off = mine && n < p.N ? (int)((uint32_t)(tok * p.N + n) * 4u) : kOOB;
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, y), rows, off, 0, 0);
            } else if (mine) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n + k < p.N) p.y[(int64_t)(t0 + tok) * p.N + n + k] = y[k];
            }
        }
    }
}

}  // namespace msnb
