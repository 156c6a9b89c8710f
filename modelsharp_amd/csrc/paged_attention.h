// paged_attention.h — attention of each request's new tokens over its keys and values in a paged
// cache (fp32 or fp16), causal, with an optional sliding window:
//
//   out[t, h] = sum_j w_j V[row_j, g],   w = softmax(scale q_t,h . K[row_j, g]),
//   j in [max(0, pos - window + 1), pos],  pos = past[r] + t - cu[r],  g = h / (H / kvH)
//
// The query heads of a kv head and the tokens of a request are rows of one matrix, row = token
// * group + head in group, so that a tile of K and V serves every row that reads it.
#pragma once
#include "serving.h"

namespace msnb {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
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

// Tile `idx` of the batch, the requests in order and each one's tiles from its last (the longest
// range of keys) to its first; false past the end. Every wave by itself, with a uniform idx.
template <int BM>
__device__ __forceinline__ bool paged_tile(const PagedAttnArgs& p, int idx, PagedTile& t)
{
    const PagedBatch& b = p.b;
    const int lane = threadIdx.x & (kWave - 1);
    for (int base = 0; base < b.requests; base += kWave) {
        const int i = min(base + lane, b.requests - 1);
        const int c0 = max(b.cu[i], 0), c1 = min(b.cu[i + 1], b.tokens);
        const int n = base + lane < b.requests ? max(c1 - c0, 0) : 0;
        const int tiles = (n * p.grp.div + BM - 1) / BM;
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
            t.past = min(max(__builtin_amdgcn_readfirstlane(b.past[t.r]), 0), 0x3fffffff);
            t.klast = min((int64_t)t.past + nl, (int64_t)b.max_pages * b.page.div) - 1;
            return true;
        }
        idx -= __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return false;
}

// Positions [lo, hi] that some row of the tile sees; split `sp` takes [klo, khi] of them, in
// whole steps of `step`. Empty where khi < klo.
struct PagedRange {
    int klo, khi;
};
__device__ __forceinline__ PagedRange paged_range(const PagedAttnArgs& p, int pos0, int pos1, int klast, int sp, int step)
{
    const int lo = p.window >= 0 ? max(0, pos0 - p.window + 1) : 0, hi = min(pos1, klast);
    const int first = lo / step, n = hi >= lo ? hi / step - first + 1 : 0;
    const int per = (n + p.splits - 1) / p.splits;
    const int a = sp * per, e = min(n, a + per);
    if (a >= e) return {0, -1};
    return {max(lo, (first + a) * step), min(hi, (first + e) * step - 1)};
}

__device__ __forceinline__ float* paged_part_ml(const PagedAttnArgs& p, int sp, int64_t row)
{
    return p.part + ((int64_t)sp * p.b.tokens * p.H + row) * 2;
}
__device__ __forceinline__ float* paged_part_o(const PagedAttnArgs& p, int sp, int64_t row)
{
    const int64_t n = (int64_t)p.b.tokens * p.H;
    return p.part + (int64_t)p.splits * n * 2 + (sp * n + row) * p.D;
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
__device__ __forceinline__ void paged_exact_row(const PagedAttnArgs& p, const PagedTile& t, int lr, int sp, PagedRange kr)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int row = t.row0 + lr, tok = p.grp.quot(row);
    const int g = blockIdx.x % p.kvH, head = g * p.grp.div + row - tok * p.grp.div;
    const int pos = t.past + tok;
    const int lo = max(kr.klo, p.window >= 0 ? max(0, pos - p.window + 1) : 0), hi = min(kr.khi, pos);
    const float* const q = p.q + (int64_t)(t.t0 + tok) * p.q_stride + (int64_t)head * p.D;
    const T* const kc = static_cast<const T*>(p.kc);
    const T* const vc = static_cast<const T*>(p.vc);
    auto score = [&](int rw) {
        const T* const k = kc + ((int64_t)rw * p.kvH + g) * p.D;
        float s = 0.0f;
        for (int d = 0; d < p.D; ++d) s = __builtin_fmaf(q[d], (float)k[d], s);
        return s * p.scale2;
    };
    float m = -__builtin_inff();
    bool seen = false, bad = false;
    for (int k = lo + lane; k <= hi; k += kWave) {
        const int rw = paged_row(p.b, t.r, k);
        if (rw < 0) continue;
        const float s = score(rw);
        seen = true;
        bad |= !(s < __builtin_inff());
        m = fmaxf(m, s);
    }
    m = row16_max_all(m);
    m = fmaxf(m, xor16_value(m));
    m = fmaxf(m, xor32_value(m));
    seen = __ballot(seen) != 0;
    bad = __ballot(bad) != 0;
    const bool all_low = seen && !bad && m == -__builtin_inff();
    float l = 0.0f;
    if (seen && !bad && !all_low)
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
    for (int c0 = 0; c0 < p.D; c0 += kWave) {
        const int c = min(c0 + lane, p.D - 1);
        float acc = bad || (all_low && p.splits == 1) ? __builtin_nanf("") : 0.0f;
        if (seen && !bad && !all_low)
            for (int k0 = lo; k0 <= hi; k0 += kWave) {
                const int k = k0 + lane, rw = k <= hi ? paged_row(p.b, t.r, k) : -1;
                const float w = rw >= 0 ? __builtin_amdgcn_exp2f(score(rw) - m) / l : 0.0f;
                for (int j = 0; j < min(kWave, hi - k0 + 1); ++j) {
                    const int rj = __builtin_amdgcn_readlane(rw, j);
                    const float wj = lane_value(w, j);
                    if (rj >= 0) acc = __builtin_fmaf(wj, (float)vc[((int64_t)rj * p.kvH + g) * p.D + c], acc);
                }
            }
        if (c0 + lane < p.D) o[c0 + lane] = acc;
    }
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

// Tiles of 16 rows: single tokens and short chunks. Four waves take every fourth step of 16 U
// keys each with their own running maximum and sums, and meet in LDS at the end.
//
// S^T = K Q^T (keys M, rows N) leaves lane l with the scores of row l % 16 at keys 4 (l / 16) + i,
// which is where the fp32 matrix product O^T += V^T P^T over four keys wants its weights: step i
// takes keys 4 g + i of the four lane groups g, and lane l gives V[key 4 (l / 16) + i] from its
// own 16-byte load. So neither the weights nor V pass through LDS, V's rows come in as whole
// lines, and the weights stay fp32. K in fp16 meets the queries as two halves, q = 2^e (qh + ql)
// (22 bits; e by row, so that any fp32 query fits), K in fp32 in fp32.
// The cache's bytes bound it: per 16 keys of fp16, D = 128, 8 KB against 1152 cycles of the
// matrix cores, 17 TB/s over the card.
template <typename T, int DP, int U>
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedAttnArgs p)
{
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int VEC = F16 && DP >= 128 ? 8 : 4;   // channels of one lane's load of V
    constexpr int NC = DP / (16 * VEC);             // loads of a V row's part
    constexpr int KS = DP / PagedElem<T>::kStep;    // loads of a K row's part
    constexpr int KV = F16 ? 8 : 4;                 // channels of one lane's load of K
    typedef typename PagedElem<T>::vec_t kvec_t;
    typedef T vvec_t __attribute__((ext_vector_type(VEC)));
    __shared__ float stat[2][4][16];
    __shared__ floatx4_t merge[4][4][kWave];
    __shared__ int flag;

    const int g = blockIdx.x % p.kvH, rest = blockIdx.x / p.kvH;
    const int sp = rest % p.splits;
    PagedTile t;
    if (!paged_tile<16>(p, rest / p.splits, t)) return;
    const int lane = threadIdx.x & 63, grp = lane >> 4, l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (threadIdx.x == 0) flag = 0;

    const int row = t.row0 + min(l16, t.rows - 1), tok = p.grp.quot(row);
    const int head = g * p.grp.div + row - tok * p.grp.div;
    const int pos = t.past + tok;
    const PagedRange kr = paged_range(p, t.past + p.grp.quot(t.row0), t.past + p.grp.quot(t.row0 + t.rows - 1), t.klast,
                                      sp, 16 * U);
    const int k_lo = max(kr.klo, p.window >= 0 ? max(0, pos - p.window + 1) : 0), k_hi = min(kr.khi, pos);

    // the queries, once
    const float* const q = p.q + (int64_t)(t.t0 + tok) * p.q_stride + (int64_t)head * p.D;
    kvec_t qh[KS], ql[F16 ? KS : 1];
    float fac = p.scale2;
    {
        float x[KS][KV];
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int c = KV * grp + PagedElem<T>::kStep * s;
#pragma unroll
            for (int i = 0; i < KV / 4; ++i) {
                const floatx4_t v = c < p.D ? floatx4_t(*reinterpret_cast<const f4u_t*>(q + c + 4 * i)) : floatx4_t{};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[s][4 * i + e] = v[e];
                    mx = fmaxf(mx, fabsf(v[e]));
                }
            }
        }
        if constexpr (F16) {
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
                    ql[s][i] = (_Float16)(v - (float)qh[s][i]);
                }
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < KV; ++i) qh[s][i] = x[s][i];
        }
    }

    const int64_t hs = (int64_t)p.kvH * p.D;   // a cache row
    const T* const kc = static_cast<const T*>(p.kc) + (int64_t)g * p.D;
    const T* const vc = static_cast<const T*>(p.vc) + (int64_t)g * p.D;
    const bool whole = (p.b.page.div & 15) == 0;   // 16 aligned keys lie in one page

    floatx4_t acc[NC][VEC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[c][j] = floatx4_t{};
    float m = -__builtin_inff(), l = 0.0f;

    for (int k0 = kr.klo / (16 * U) * (16 * U) + 16 * U * wave; k0 <= kr.khi; k0 += 64 * U) {
        // every load first; keys past the request's last read that one, pages that are not
        // there read the cache's first row, and both are masked
        kvec_t kx[U][KS];
        vvec_t vx[U][4][NC];
        bool there[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = k0 + 16 * u;
            int krow, vrow[4];
            if (whole) {
                const int st = min(key, t.klast & ~15);
                const int base = paged_row(p.b, t.r, st);
                krow = base < 0 ? 0 : base + min(key + l16, t.klast) - st;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vrow[i] = base < 0 ? 0 : base + min(key + 4 * grp + i, t.klast) - st;
                    there[u][i] = base >= 0;
                }
            } else {
                krow = max(paged_row(p.b, t.r, min(key + l16, t.klast)), 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vrow[i] = paged_row(p.b, t.r, min(key + 4 * grp + i, t.klast));
                    there[u][i] = vrow[i] >= 0;
                    vrow[i] = max(vrow[i], 0);
                }
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int c = KV * grp + PagedElem<T>::kStep * s;
                kx[u][s] = *reinterpret_cast<const kvec_t*>(kc + krow * hs + (c < p.D ? c : 0));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int ch = VEC * (l16 + 16 * c);
                    vx[u][i][c] = *reinterpret_cast<const vvec_t*>(vc + vrow[i] * hs + (ch < p.D ? ch : 0));
                }
        }
        float sc[U][4];
        float mt = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            floatx4_t s4{};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if constexpr (F16) {
                    s4 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kx[u][s], qh[s], s4, 0, 0, 0);
                    s4 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kx[u][s], ql[s], s4, 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[u][s][e], qh[s][e], s4, 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = k0 + 16 * u + 4 * grp + i;
                sc[u][i] = there[u][i] && key >= k_lo && key <= k_hi ? s4[i] * fac : -__builtin_inff();
                mt = fmaxf(mt, sc[u][i]);
            }
        }
        mt = fmaxf(mt, xor16_value(mt));
        mt = fmaxf(mt, xor32_value(mt));
        const float mn = fmaxf(m, mt), ms = mn == -__builtin_inff() ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        l *= al;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[u][i] = __builtin_amdgcn_exp2f(sc[u][i] - ms);
                l += sc[u][i];
            }
        if (__ballot(al != 1.0f))
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[c][j] *= al;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)vx[u][i][c][j], sc[u][i], acc[c][j], 0, 0, 0);
    }

    // the waves' sums meet: statistics, then four quads of channels at a time
    l += xor16_value(l);
    l += xor32_value(l);
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
    const float f = ll != 0.0f ? __builtin_amdgcn_exp2f(m - ms) / ll : 0.0f;
    const int64_t orow = (int64_t)(t.t0 + tok) * p.H + head;
    float* const o = p.splits > 1 ? paged_part_o(p, sp, orow) : p.out + orow * p.D;
    const bool mine = l16 < t.rows;
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
        paged_part_ml(p, sp, orow)[0] = mm;
        paged_part_ml(p, sp, orow)[1] = ll;
    }
    if (odd) flag = 1;
    __syncthreads();
    if (flag)
        for (int lr = wave; lr < t.rows; lr += 4) paged_exact_row<T>(p, t, lr, sp, kr);
}

// The splits' records of one output row, joined in the splits' order. A wave per row.
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs p)
{
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= (int64_t)p.b.tokens * p.H) return;
    const int tok = (int)(row / p.H);
    if (tok < p.b.cu[0] || tok >= p.b.cu[p.b.requests]) return;   // rows of no request stay as they were
    float m = -__builtin_inff();
    bool low = false;
    for (int s = 0; s < p.splits; ++s) {
        const float* const ml = paged_part_ml(p, s, row);
        if (ml[1] != 0.0f) {
            m = fmaxf(m, ml[0]);
            low = true;
        }
    }
    const bool all_low = low && m == -__builtin_inff();
    const float ms = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
        const float* const ml = paged_part_ml(p, s, row);
        if (ml[1] != 0.0f) l += ml[1] * __builtin_amdgcn_exp2f(ml[0] - ms);
    }
    for (int c = lane; c < p.D; c += 64) {
        float o = all_low ? __builtin_nanf("") : 0.0f;
        if (!all_low)
            for (int s = 0; s < p.splits; ++s) {
                const float* const ml = paged_part_ml(p, s, row);
                if (ml[1] != 0.0f && !(ml[0] == -__builtin_inff()))
                    o += (ml[1] * __builtin_amdgcn_exp2f(ml[0] - ms) / l) * paged_part_o(p, s, row)[c];
            }
        p.out[row * p.D + c] = o;
    }
}

}  // namespace msnb
