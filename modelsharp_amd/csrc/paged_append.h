// paged_append.h — norms of queries and keys for each head, the position rotation, and the append
// of the new keys and values to a paged cache, in one pass over the projections' rows:
//
//   n(x) = (x * inv) * gamma,  inv = 1 / sqrt(sum(x^2) / D + eps)          (per head)
//   y_j, y_j+h = n_j c - n_j+h s, n_j+h c + n_j s   (or the pairs 2j, 2j + 1)
//
// with c, s row min(position, cos_rows - 1) of the caches, as GroupQueryAttention has them.
// Every value is read once and written once, and nothing else is done: memory bounds a chunk (2048
// tokens of 28 + 4 + 4 heads of 128: 15.3 us, 4.7 TB/s; a library copy reaches 5.1), the chain cu ->
// past and table -> store a few tokens (8 tokens: 3.6 us).
#pragma once
#include "serving.h"

namespace msnb {

struct AppendPlace {
    int pos, row;   // position; row of the cache or of the contiguous outputs, -1: none
};

// Uniform over the wave.
__device__ __forceinline__ bool append_place(const AppendArgs& p, int t, AppendPlace& at)
{
    if (!p.b.cu) {
        at.pos = p.positions ? max(p.positions[t], 0) : 0;   // null: nothing turns
        at.row = t;
        return true;
    }
    const int r = paged_request(p.b, t);
    if (r >= p.b.requests) return false;   // a row behind the last request's
    const int i = t - p.b.cu[r];
    if (i < 0) return false;
    at.pos = (int)min((int64_t)max(p.b.past[r], 0) + i, (int64_t)kPagedPositions);
    at.row = at.pos < kPagedPositions ? paged_row(p.b, r, at.pos) : -1;
    return true;
}

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void append_store4(void* base, int64_t at, int f16, floatx4_t v)
{
    if (f16)
        *reinterpret_cast<half4_t*>(static_cast<_Float16*>(base) + at) =
            half4_t{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    else
        *reinterpret_cast<floatx4_t*>(static_cast<float*>(base) + at) = v;
}

// grid (tokens, ceil(head rows / (256 / GS))): GS lanes per head row of D = 8 * (lanes used), each
// holding the two groups of four channels that rotate into each other. Head rows are the
// token's H query heads, then its key heads, then its value heads (paged only).
template <int GS>
__global__ __launch_bounds__(256) void append_vec_kernel(AppendArgs p)
{
    const int t = blockIdx.x, lane = threadIdx.x & (GS - 1);
    const int slot = blockIdx.y * (256 / GS) + threadIdx.x / GS;
    const int slots = p.H + p.kvH * (p.b.cu ? 2 : 1);
    AppendPlace at;
    if (!append_place(p, t, at)) return;
    const int kind = slot < p.H ? 0 : slot < p.H + p.kvH ? 1 : 2;
    const int head = slot - (kind == 0 ? 0 : kind == 1 ? p.H : p.H + p.kvH);
    const bool live = slot < slots && lane < (p.D >> 3);
    const int quads = p.rot_half >> 2;   // lanes whose channels turn
    const bool turns = kind < 2 && lane < quads;
    const int c0 = lane < quads ? 4 * lane : 2 * p.rot_half + 8 * (lane - quads);
    const int c1 = lane < quads ? p.rot_half + 4 * lane : c0 + 4;
    const float* const row = kind == 0   ? p.q + t * p.q_stride + (int64_t)head * p.D
                             : kind == 1 ? p.k + t * p.k_stride + (int64_t)head * p.D
                                         : p.v + t * p.v_stride + (int64_t)head * p.D;
    floatx4_t a{}, b{};
    if (live) {
        a = *reinterpret_cast<const floatx4_t*>(row + c0);
        b = *reinterpret_cast<const floatx4_t*>(row + c1);
    }
    const float* const gamma = kind == 0 ? p.gq : kind == 1 ? p.gk : nullptr;
    floatx4_t ca{}, sa{}, cb{}, sb{}, ga{}, gb{};
    if (live && turns) {   // halves: channel j turns by angle j; pairs: channel j by angle j / 2
        const int64_t tr = (int64_t)min(at.pos, p.cos_rows - 1) * p.half;
        if (p.interleaved) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ca[i] = p.cos[tr + (c0 >> 1) + i];
                sa[i] = p.sin[tr + (c0 >> 1) + i];
                cb[i] = p.cos[tr + (c1 >> 1) + i];
                sb[i] = p.sin[tr + (c1 >> 1) + i];
            }
        } else {
            ca = *reinterpret_cast<const floatx4_t*>(p.cos + tr + c0);
            sa = *reinterpret_cast<const floatx4_t*>(p.sin + tr + c0);
        }
    }
    if (gamma) {   // differs between the waves of a workgroup only by kind
        if (live) {
            ga = *reinterpret_cast<const floatx4_t*>(gamma + c0);
            gb = *reinterpret_cast<const floatx4_t*>(gamma + c1);
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += a[i] * a[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += b[i] * b[i];
    ss = group_sum_all<GS>(ss);
    if (gamma) {
        const float inv = 1.0f / __builtin_sqrtf(ss / (float)p.D + p.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = (a[i] * inv) * ga[i];
            b[i] = (b[i] * inv) * gb[i];
        }
    }
    if (turns) {
        const floatx4_t x = a, y = b;
        if (p.interleaved) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[2 * i] = x[2 * i] * ca[i] - x[2 * i + 1] * sa[i];
                a[2 * i + 1] = x[2 * i + 1] * ca[i] + x[2 * i] * sa[i];
                b[2 * i] = y[2 * i] * cb[i] - y[2 * i + 1] * sb[i];
                b[2 * i + 1] = y[2 * i + 1] * cb[i] + y[2 * i] * sb[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = x[i] * ca[i] - y[i] * sa[i];
                b[i] = y[i] * ca[i] + x[i] * sa[i];
            }
        }
    }
    if (!live) return;
    if (kind == 0) {
        float* const o = p.q_out + ((int64_t)t * p.H + head) * p.D;
        *reinterpret_cast<floatx4_t*>(o + c0) = a;
        *reinterpret_cast<floatx4_t*>(o + c1) = b;
    } else if (at.row >= 0) {
        void* const base = kind == 1 ? p.k_out : p.v_out;
        const int64_t o = ((int64_t)at.row * p.kvH + head) * p.D;
        append_store4(base, o + c0, p.f16, a);
        append_store4(base, o + c1, p.f16, b);
    }
}

// Any head_dim up to kAppendMaxDim, any alignment: a wave per head row, staged in LDS (the
// outputs may be the inputs). grid (tokens, ceil(head rows / 4)).
__global__ __launch_bounds__(256) void append_any_kernel(AppendArgs p)
{
    __shared__ float rows[4][kAppendMaxDim];
    const int t = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int slot = blockIdx.y * 4 + wave;
    const int slots = p.H + p.kvH * (p.b.cu ? 2 : 1);
    AppendPlace at;
    if (slot >= slots || !append_place(p, t, at)) return;   // no barrier follows
    const int kind = slot < p.H ? 0 : slot < p.H + p.kvH ? 1 : 2;
    const int head = slot - (kind == 0 ? 0 : kind == 1 ? p.H : p.H + p.kvH);
    const float* const row = kind == 0   ? p.q + t * p.q_stride + (int64_t)head * p.D
                             : kind == 1 ? p.k + t * p.k_stride + (int64_t)head * p.D
                                         : p.v + t * p.v_stride + (int64_t)head * p.D;
    const float* const gamma = kind == 0 ? p.gq : kind == 1 ? p.gk : nullptr;
    float* const x = rows[wave];
    float ss = 0.0f;
    for (int d = lane; d < p.D; d += 64) {
        x[d] = row[d];
        ss += x[d] * x[d];
    }
    const float inv = 1.0f / __builtin_sqrtf(group_sum_all<64>(ss) / (float)p.D + p.eps);
    if (gamma)
        for (int d = lane; d < p.D; d += 64) x[d] = (x[d] * inv) * gamma[d];
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");   // the wave's LDS writes before its reads
    __builtin_amdgcn_wave_barrier();
    if (kind > 0 && at.row < 0) return;
    const int rot = kind < 2 ? 2 * p.rot_half : 0;
    const int64_t tr = (int64_t)min(at.pos, p.cos_rows - 1) * p.half;
    const int64_t o = kind == 0 ? ((int64_t)t * p.H + head) * p.D : ((int64_t)at.row * p.kvH + head) * p.D;
    for (int d = lane; d < p.D; d += 64) {
        float y = x[d];
        if (d < rot) {
            const int j = p.interleaved ? d >> 1 : d < p.rot_half ? d : d - p.rot_half;
            const int i0 = p.interleaved ? 2 * j : j, i1 = p.interleaved ? 2 * j + 1 : j + p.rot_half;
            const float c = p.cos[tr + j], s = p.sin[tr + j];
            y = d == i0 ? x[i0] * c - x[i1] * s : x[i1] * c + x[i0] * s;
        }
        if (kind == 0)
            p.q_out[o + d] = y;
        else if (p.f16)
            static_cast<_Float16*>(kind == 1 ? p.k_out : p.v_out)[o + d] = (_Float16)y;
        else
            static_cast<float*>(kind == 1 ? p.k_out : p.v_out)[o + d] = y;
    }
}

}  // namespace msnb
