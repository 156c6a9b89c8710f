// paged_plan.h — a step's lengths, pages and rows from what each request wants:
//
//   have = ceil(past / page), need = ceil((past + want) / page) - have
//   served: want > 0, the pages fit the table, the sum of want up to and with this request
//           fits the step's rows, and need is 0 or its sum fits the free pages
//   cu = sums of want over the served; page j of the step is the j-th from the top of the stack
//
// (sums over the requests whose pages fit the table, served or not, so that what waits is not passed by what comes
// behind it), and the step's end: lengths advance, the
// pages of requests that ended go back to the stack.
#pragma once
#include "serving_loop.h"

namespace msnb {

// a + b, at most 2^32 - 1: sums of lengths that make no sense stay ordered.
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b)
{
    const uint32_t s = a + b;
    return s < a ? ~0u : s;
}

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t sat_dpp(uint32_t x)
{
    return sat_add(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROW_MASK, 0xF, false));
}
// Inclusive saturating scan over the wave.
__device__ __forceinline__ uint32_t wave_scan_sat(uint32_t x)
{
    x = sat_dpp<0x111, 0xF>(x);   // row_shr:1
    x = sat_dpp<0x112, 0xF>(x);
    x = sat_dpp<0x114, 0xF>(x);
    x = sat_dpp<0x118, 0xF>(x);
    x = sat_dpp<0x142, 0xA>(x);   // row_bcast:15 -> rows 1, 3
    return sat_dpp<0x143, 0xC>(x);   // row_bcast:31 -> rows 2, 3
}

// Two sums over a workgroup of WAVES waves: what lies before this thread, and the whole. The
// scratch is used again behind the next barrier but one.
struct PairScan {
    uint32_t a, b;           // before this thread
    uint32_t all_a, all_b;
};
template <int WAVES>
__device__ __forceinline__ PairScan block_scan2(uint32_t a, uint32_t b, uint32_t (&scratch)[2][WAVES])
{
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    const uint32_t sa = wave_scan_sat(a), sb = wave_scan_sat(b);
    if (lane == kWave - 1) {
        scratch[0][wave] = sa;
        scratch[1][wave] = sb;
    }
    __syncthreads();
    // (exclusive by a lane's neighbour: a saturated sum cannot be taken back)
    uint32_t pa = __shfl_up(sa, 1), pb = __shfl_up(sb, 1);
    PairScan r{lane ? pa : 0, lane ? pb : 0, 0, 0};
    uint32_t ba = 0, bb = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) {
            ba = sat_add(ba, scratch[0][w]);
            bb = sat_add(bb, scratch[1][w]);
        }
        r.all_a = sat_add(r.all_a, scratch[0][w]);
        r.all_b = sat_add(r.all_b, scratch[1][w]);
    }
    r.a = sat_add(r.a, ba);
    r.b = sat_add(r.b, bb);
    return r;
}

// Every workgroup sums all requests for itself (8 bytes each, from L2), keeps both sums in LDS and
// writes its part of the tokens and of the new pages, each found by bisection: one launch, no
// workspace, no wait between workgroups. Bound by its chain of round trips and by the call: 4.2 us of kernel for 32
// requests of a token, 5.2 for 256 with chunks of 700 (11,000 rows), 8.1 the calls.
__global__ __launch_bounds__(256) void paged_plan_kernel(PlanArgs p)
{
    extern __shared__ uint32_t plan_lds[];
    uint32_t* const cu = plan_lds;                       // [requests + 1]
    uint32_t* const pg = plan_lds + p.requests + 1;      // pages of the step before each request
    __shared__ uint32_t scratch[2][2][4];
    const int tid = threadIdx.x, R = p.requests;
    const uint32_t count = min(max(*p.free_count, 0), p.num_pages);
    uint32_t asked = 0, wanted = 0, rows = 0, pages = 0;   // sums before this block of requests
    constexpr int kEach = 4;
    for (int base = 0; base < R; base += 256 * kEach) {
        uint32_t ask[kEach], need[kEach], sa = 0, sn = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = base + tid * kEach + i;
            const int w = r < R ? p.want[r] : 0, h = r < R ? max(p.past[r], 0) : 0;
            ask[i] = w;
            need[i] = h;
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int w = ask[i], h = need[i];
            const bool room = w > 0 && h <= kPagedPositions - w;
            const int end = room ? h + w : 0;
            const int have = p.page.quot(h) + (p.page.quot(h) * p.page.div < h);
            const int all = p.page.quot(end) + (p.page.quot(end) * p.page.div < end);
            const bool fits = room && all <= p.max_pages;
            ask[i] = fits ? w : 0;
            need[i] = fits ? all - have : 0;
            sa = sat_add(sa, ask[i]);
            sn = sat_add(sn, need[i]);
        }
        const PairScan s = block_scan2<4>(sa, sn, scratch[0]);
        uint32_t ca = sat_add(asked, s.a), cn = sat_add(wanted, s.b);
        uint32_t new_rows = 0, new_pages = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            ca = sat_add(ca, ask[i]);
            cn = sat_add(cn, need[i]);
            // (by a mask: of `if (!served) ask[i] = need[i] = 0` the compiler left the first element's zeros out)
            const uint32_t served = -(uint32_t)((ca <= (uint32_t)p.tokens) & ((need[i] == 0) | (cn <= count)));
            ask[i] &= served;
            need[i] &= served;
            new_rows += ask[i];
            new_pages += need[i];
        }
        const PairScan t = block_scan2<4>(new_rows, new_pages, scratch[1]);
        uint32_t cr = rows + t.a, cp = pages + t.b;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = base + tid * kEach + i;
            if (r < R) {
                cu[r] = cr;
                pg[r] = cp;
                if (blockIdx.x == 0) p.cu[r] = cr;
            }
            cr += ask[i];
            cp += need[i];
        }
        asked = sat_add(asked, s.all_a);
        wanted = sat_add(wanted, s.all_b);
        rows += t.all_a;
        pages += t.all_b;
    }
    if (tid == 0) {
        cu[R] = rows;
        pg[R] = pages;
        if (blockIdx.x == 0) {
            p.cu[R] = rows;
            *p.used = pages;
        }
    }
    __syncthreads();

    // the request that item `x` of the sums `at` belongs to: the last whose items begin at or before it
    auto find = [&](const uint32_t* at, uint32_t x) {
        int lo = 0, hi = R;   // at[lo] <= x < at[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (at[mid] <= x) lo = mid; else hi = mid;
        }
        return lo;
    };
    auto have_of = [&](int past) { return p.page.quot(past) + (p.page.quot(past) * p.page.div < past); };
    const int step = gridDim.x * 256, first = blockIdx.x * 256 + tid;
    for (int t = first; t < p.tokens; t += step) {
        int r = -1, pos = -1, slot = -1;
        if ((uint32_t)t < rows) {
            r = find(cu, t);
            const int past = max(p.past[r], 0);
            pos = past + t - (int)cu[r];
            const int col = p.page.quot(pos), have = have_of(past);
            const int e = col < have ? p.table[(int64_t)r * p.max_pages + col] : p.free[count - 1 - (pg[r] + col - have)];
            if ((unsigned)e < (unsigned)p.num_pages) slot = e * p.page.div + pos - col * p.page.div;
        }
        p.request[t] = r;
        p.position[t] = pos;
        p.slot[t] = slot;
    }
    for (uint32_t j = first; j < pages; j += step) {
        const int r = find(pg, j);
        p.table[(int64_t)r * p.max_pages + have_of(max(p.past[r], 0)) + (j - pg[r])] = p.free[count - 1 - j];
    }
}

// The step's end, by one workgroup (where a page goes depends on all before it, and a step returns few): requests
// in blocks of 1024; the table entries of those that ended, one after another, 1024 at a time. 5.2 us for 64
// requests that return 900 pages.
__global__ __launch_bounds__(1024) void paged_commit_kernel(CommitArgs p)
{
    constexpr int kBlock = 1024, kWaves = kBlock / kWave;
    __shared__ int ended[kBlock], first_col[kBlock];
    __shared__ uint32_t start[kBlock + 1];       // table entries before each of them
    __shared__ uint32_t scratch[2][2][kWaves];
    const int tid = threadIdx.x;
    const int count = min(max(*p.free_count, 0), p.num_pages);
    int top = count - min(max(*p.used, 0), count);
    for (int base = 0; base < p.requests; base += kBlock) {
        const int r = base + tid;
        int cols = 0, keep = 0;
        bool done = false;
        if (r < p.requests) {
            const int64_t end = (int64_t)max(p.past[r], 0) + max(p.cu[r + 1] - p.cu[r], 0);
            const int after = (int)min(end, (int64_t)kPagedPositions);
            done = p.done && p.done[r];
            p.past[r] = done ? 0 : after;
            keep = p.keep ? min(max(p.keep[r], 0), p.max_pages) : 0;
            cols = min(p.page.quot(after) + (p.page.quot(after) * p.page.div < after), p.max_pages);
        }
        const uint32_t mine = done && cols > keep ? cols - keep : 0;
        const PairScan s = block_scan2<kWaves>(mine ? 1 : 0, mine, scratch[0]);
        if (mine) {
            ended[s.a] = r;
            first_col[s.a] = keep;
            start[s.a] = s.b;
        }
        if (tid == 0) start[s.all_a] = s.all_b;
        __syncthreads();
        const int n = (int)s.all_a;
        int flip = 0;
        for (uint32_t f0 = 0; f0 < s.all_b; f0 += kBlock, flip ^= 1) {
            const uint32_t f = f0 + tid;
            int e = -1;
            if (f < s.all_b) {
                int lo = 0, hi = n;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (start[mid] <= f) lo = mid; else hi = mid;
                }
                int32_t* const at = p.table + (int64_t)ended[lo] * p.max_pages + first_col[lo] + (f - start[lo]);
                e = *at;
                *at = -1;
            }
            const bool page = (unsigned)e < (unsigned)p.num_pages;
            const PairScan q = block_scan2<kWaves>(page ? 1 : 0, 0, scratch[flip]);
            // (a page returned twice would run past the stack: dropped)
            if (page && (int64_t)top + q.a < p.num_pages) p.free[top + q.a] = e;
            top = (int)min((int64_t)top + q.all_a, (int64_t)p.num_pages);
        }
        __syncthreads();
    }
    if (tid == 0) *p.free_count = top;
}

}  // namespace msnb
