// Bookkeeping and stores of a step over a paged cache: pages, slots and
// positions from request lengths (paged_plan_body, paged_rows_body), and the
// rotary embedding with the store of k and v to the slots (paged_rope_body).
#pragma once
#include "../paged_args.h"
#include "common.h"

namespace ifr {

// Inclusive sum over a workgroup of up to 1024 threads; `total` is the
// workgroup's.  part: 16 entries of LDS, free again at the return.
IFR_DEV uint64_t block_scan(uint64_t v, uint64_t *part, uint64_t &total) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, nw = (int)(blockDim.x + 63) >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t u = __shfl_up(v, d, 64);
        if (lane >= d) v += u;
    }
    if (lane == 63) part[wave] = v;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
    for (int w = 0; w < nw; w++) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    __syncthreads();
    return before + v;
}

// Last index i < n with a[i] <= x (a[0] <= x, a non-decreasing).
IFR_DEV uint32_t last_at_most(const uint32_t *a, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n; // a[lo] <= x < a[hi]
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Position and slot of row `row`, which is request r's (rows from `start` to
// `end`; kv rows of the cache after the step, 0: not granted).
IFR_DEV void paged_row(const PagedPlanArgs &a, uint32_t row, uint32_t r, uint32_t start, uint32_t end, uint32_t kv) {
    uint32_t pos = PG_NO_ROW;
    uint64_t slot = ~0ull;
    if (kv && row < end) {
        pos = kv - (end - start) + (row - start);
        const uint32_t page = a.table[(size_t)r * a.max_pages + (pos >> a.lp)];
        if (page < a.n_pages) slot = ((uint64_t)page << a.lp) + (pos & ((1u << a.lp) - 1));
    }
    a.positions[row] = pos;
    a.slots[row] = slot;
}

// The requests of a step, by one workgroup: rounds of blockDim requests, the
// running sums carried between them.  (One workgroup: the free list and the
// table may be updated in place, and every request depends on the sums of
// those before it; a step has far fewer requests than rows.)  Bound by the
// latency of its chain: lengths, two scans, the popped pages, the rows.
__device__ inline void paged_plan_body(const PagedPlanArgs &a) {
    __shared__ uint64_t part[16];
    __shared__ uint32_t s_start[PG_PLAN_THREADS + 1], s_off[PG_PLAN_THREADS + 1], s_held[PG_PLAN_THREADS], s_kv[PG_PLAN_THREADS];
    const uint32_t tid = threadIdx.x, T = blockDim.x, lane = tid & 63, pm = (1u << a.lp) - 1;
    uint64_t top = min(*a.free_count, a.n_pages);
    const uint64_t cap = (uint64_t)a.max_pages << a.lp;

    // released requests' pages onto the stack: a wave per request, its valid
    // entries kept in order (s_off[i]: how many request i of the round has)
    for (uint32_t base = 0; base < a.n_requests; base += T) {
        const uint32_t r = base + tid;
        uint32_t held = 0;
        if (r < a.n_requests && a.new_len[r] == PG_RELEASE)
            held = (uint32_t)min((uint64_t)a.max_pages, ((uint64_t)a.ctx_len[r] + pm) >> a.lp);
        if (!__syncthreads_or(held != 0)) continue;
        s_held[tid] = held;
        s_off[tid] = 0;
        __syncthreads();
        auto each = [&](bool push) {
            for (uint32_t i = tid >> 6; i < T; i += T >> 6) {
                const uint32_t h = s_held[i];
                const uint32_t *row = a.table + (size_t)(base + i) * a.max_pages;
                uint32_t n = 0;
                for (uint32_t e = 0; e < h; e += 64) {
                    const uint32_t page = e + lane < h ? row[e + lane] : ~0u;
                    const uint64_t ok = __ballot(page < a.n_pages);
                    if (push && page < a.n_pages) {
                        const uint64_t to = top + s_start[i] + n + __popcll(ok & ((1ull << lane) - 1));
                        if (to < a.n_pages) a.free_pages[to] = page;
                    }
                    n += __popcll(ok);
                }
                if (!push && h && lane == 0) s_off[i] = n;
            }
        };
        each(false);
        __syncthreads();
        uint64_t total;
        const uint32_t cnt = s_off[tid];
        s_start[tid] = (uint32_t)(block_scan(cnt, part, total) - cnt);
        __syncthreads();
        each(true);
        __syncthreads();
        top = min(top + total, (uint64_t)a.n_pages);
    }
    __threadfence(); // the pushed pages, read below by other waves
    __syncthreads();

    uint64_t rows0 = 0, need0 = 0, taken = 0;
    for (uint32_t base = 0; base < a.n_requests; base += T) {
        const uint32_t r = base + tid, nr = min(T, a.n_requests - base);
        const bool in = r < a.n_requests;
        const uint32_t ctx = in ? a.ctx_len[r] : 0, nw = in ? a.new_len[r] : 0;
        const bool gone = nw == PG_RELEASE;
        const uint64_t n = gone ? 0 : nw;
        uint64_t total_rows, total_need;
        const uint64_t end = rows0 + block_scan(n, part, total_rows), start = end - n;
        const uint64_t sum = (uint64_t)ctx + n;
        const bool fits = in && !gone && sum <= cap && end <= a.n_rows;
        const uint32_t held = (uint32_t)(((uint64_t)ctx + pm) >> a.lp);
        const uint64_t need = fits ? ((sum + pm) >> a.lp) - held : 0;
        const uint64_t off = need0 + block_scan(need, part, total_need) - need;
        const bool ok = fits && (!need || off + need <= top);
        if (in) {
            a.row_start[r] = (uint32_t)min(start, (uint64_t)a.n_rows);
            a.kv_len[r] = ok ? (uint32_t)sum : 0u;
            if (a.ctx_len_out) a.ctx_len_out[r] = ok ? (uint32_t)sum : gone ? 0u : ctx;
        }
        // the round's new table entries, one per thread: entry i of the round
        // is request j's, the last one whose pages begin at or before i
        const uint64_t mine = ok ? need : 0;
        uint64_t fresh;
        const uint64_t upto = block_scan(mine, part, fresh);
        s_off[tid] = (uint32_t)(upto - mine);
        s_start[tid] = (uint32_t)min(start, (uint64_t)a.n_rows);
        s_held[tid] = held;
        s_kv[tid] = ok ? (uint32_t)sum : 0u;
        if (tid == nr - 1) s_start[nr] = (uint32_t)min(end, (uint64_t)a.n_rows);
        __syncthreads();
        for (uint64_t i = tid; i < fresh; i += T) {
            const uint32_t j = last_at_most(s_off, nr, (uint32_t)i);
            a.table[(size_t)(base + j) * a.max_pages + s_held[j] + (uint32_t)(i - s_off[j])] =
                a.free_pages[top - 1 - (taken + i)];
        }
        taken += fresh;
        rows0 += total_rows;
        need0 += total_need;
        if (a.rows_here) {
            __threadfence_block();
            __syncthreads();
            const uint32_t first = s_start[0], last = base + nr == a.n_requests ? a.n_rows : s_start[nr];
            for (uint32_t row = first + tid; row < last; row += T) {
                const uint32_t j = last_at_most(s_start, nr, row);
                paged_row(a, row, base + j, s_start[j], s_start[j + 1], s_kv[j]);
            }
        }
        __syncthreads();
    }
    if (!a.n_requests) // no request has any of the rows
        for (uint32_t row = tid; row < a.n_rows; row += T) paged_row(a, row, 0, 0, 0, 0);
    if (tid == 0) {
        a.row_start[a.n_requests] = (uint32_t)min(rows0, (uint64_t)a.n_rows);
        *a.free_count_out = (uint32_t)(top - taken);
    }
}

// The rows of a large step, 256 threads each with rows of its own.  A
// workgroup finds its first row's request by a 256-way search of row_start,
// and its rows' among the next 1024 requests' starts in LDS.
constexpr uint32_t PG_ROWS_PER = 512, PG_ROWS_WIN = 1024;

__device__ inline void paged_rows_body(const PagedPlanArgs &a) {
    __shared__ uint32_t s_start[PG_ROWS_WIN + 1], s_kv[PG_ROWS_WIN], s_n;
    const uint32_t tid = threadIdx.x, row0 = blockIdx.x * PG_ROWS_PER;
    // the last request that starts at or before row0 (requests without rows
    // share their start with the next: the last one of them has row0)
    uint32_t lo = 0, hi = a.n_requests;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 255) / 256, i = lo + tid * step;
        if (tid == 0) s_n = 0;
        __syncthreads();
        if (i < hi && a.row_start[i] <= row0) atomicAdd(&s_n, 1u);
        __syncthreads();
        const uint32_t k = s_n;
        __syncthreads();
        // the first k samples are at or before row0 (row_start[0] = 0 is)
        lo += (k - 1) * step;
        hi = min(hi, lo + step);
    }
    const uint32_t r0 = lo, nr = min(PG_ROWS_WIN, a.n_requests - r0);
    for (uint32_t i = tid; i < nr; i += 256) {
        s_start[i] = a.row_start[r0 + i];
        s_kv[i] = a.kv_len[r0 + i];
    }
    if (tid == 0) s_start[nr] = a.row_start[r0 + nr];
    __syncthreads();
    for (uint32_t row = row0 + tid; row < min(row0 + PG_ROWS_PER, a.n_rows); row += 256) {
        if (row < s_start[nr] || r0 + nr == a.n_requests) {
            const uint32_t j = last_at_most(s_start, nr, row);
            paged_row(a, row, r0 + j, s_start[j], s_start[j + 1], s_kv[j]);
        } else { // more requests than the window between this row and the workgroup's first
            const uint32_t r = last_at_most(a.row_start, a.n_requests, row);
            paged_row(a, row, r, a.row_start[r], a.row_start[r + 1], a.kv_len[r]);
        }
    }
}

// ------------------------------------------------------ RoPE and the store --
// Workgroup (x, part): rows x * rows_per .., its part of their 8-element
// items.  The angles' (cos, sin) of the rows go to LDS, one angle per thread:
// theta_j = 2^(-2j/hs log2(base)) and pos * theta_j / 2pi in 64 bits, reduced
// to a fraction of a turn there, cos and sin of it in f32 (at position 1e5 an
// f32 product would be off by 4e-3).  An item is four pairs of one head: eight
// contiguous elements, or four and the four half a head away (NeoX).  Memory
// bound: each element is read once and written once.
constexpr uint32_t PG_ROPE_LDS = 4 * 64; // (cos, sin) pairs: up to 4 rows of up to 64

__device__ inline void paged_rope_body(const PagedRopeArgs &a) {
    __shared__ float2 cs[PG_ROPE_LDS];
    __shared__ uint32_t s_pos[4];
    __shared__ uint64_t s_slot[4];
    const uint32_t tid = threadIdx.x, hh = a.hs / 2, cpi = a.hs / 8;
    const uint32_t row0 = blockIdx.x * a.rows_per, nrows = min(a.rows_per, a.n_rows - row0);
    if (tid < nrows) {
        s_pos[tid] = a.positions[row0 + tid];
        s_slot[tid] = a.slots[row0 + tid];
    }
    for (uint32_t i = tid; i < nrows * hh; i += PG_ROPE_THREADS) {
        const uint32_t m = i / hh, j = i % hh;
        float c = 1.0f, s = 0.0f;
        if (a.turn) {
            const double th = exp2(-(double)(2 * j) / (double)a.hs * a.log2_base);
            double t = (double)a.positions[row0 + m] * th * 0.15915494309189533577; // in turns
            t -= rint(t);
            sincospif((float)(2.0 * t), &s, &c);
        }
        cs[i] = make_float2(c, s);
    }
    __syncthreads();
    const uint32_t heads = (a.q ? a.n_heads : 0) + 2 * a.n_kv, per_row = heads * cpi;
    const uint32_t items = nrows * per_row;
    for (uint32_t it = blockIdx.y * PG_ROPE_THREADS + tid; it < items; it += a.parts * PG_ROPE_THREADS) {
        const uint32_t m = it / per_row, w = it % per_row, h = w / cpi, ci = w % cpi;
        if (s_pos[m] == PG_NO_ROW) continue;
        const uint32_t nq = heads - 2 * a.n_kv;
        const uint32_t what = h < nq ? 0u : h < nq + a.n_kv ? 1u : 2u; // q, k, v
        const uint32_t head = h - (what == 0 ? 0 : what == 1 ? nq : nq + a.n_kv);
        const bool pairs_apart = a.neox && what < 2;
        // the item's elements: e0 .. +4 and e1 .. +4 of the head
        const uint32_t e0 = pairs_apart ? 4 * ci : 8 * ci, e1 = pairs_apart ? e0 + hh : e0 + 4;
        const size_t row = row0 + m;
        const float *x = (what == 0 ? a.q + row * a.ld_q : what == 1 ? a.k + row * a.ld_k : a.v + row * a.ld_v) +
                         (size_t)head * a.hs;
        const float4 u = *(const float4 *)(x + e0), v = *(const float4 *)(x + e1);
        float y[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        if (what < 2 && a.turn) {
            const float2 *ang = cs + m * hh + 4 * ci;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = pairs_apart ? i : 2 * i, q = pairs_apart ? i + 4 : 2 * i + 1;
                const float x0 = y[p], x1 = y[q];
                y[p] = ang[i].x * x0 - ang[i].y * x1;
                y[q] = ang[i].y * x0 + ang[i].x * x1;
            }
        }
        char *dst;
        uint32_t f16;
        if (what == 0) {
            f16 = a.q_f16;
            dst = (char *)a.q_out + (row * a.ld_q_out + (size_t)head * a.hs) * (f16 ? 2 : 4);
        } else {
            const uint64_t slot = s_slot[m], page = slot >> a.lp;
            if (page >= a.n_pages) continue;
            f16 = a.kv_f16;
            const int64_t off = (int64_t)page * a.page_stride + (int64_t)(slot & ((1ull << a.lp) - 1)) * a.row_stride +
                                (int64_t)head * a.head_stride;
            dst = (char *)(what == 1 ? a.key : a.value) + off * (f16 ? 2 : 4);
        }
        if (f16) {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = (uint32_t)f32_to_f16(y[2 * i]) | (uint32_t)f32_to_f16(y[2 * i + 1]) << 16;
            if (pairs_apart) {
                *(uint2 *)(dst + 2 * e0) = make_uint2(o[0], o[1]);
                *(uint2 *)(dst + 2 * e1) = make_uint2(o[2], o[3]);
            } else {
                *(uint4 *)(dst + 2 * e0) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        } else {
            *(float4 *)(dst + 4 * e0) = make_float4(y[0], y[1], y[2], y[3]);
            *(float4 *)(dst + 4 * e1) = make_float4(y[4], y[5], y[6], y[7]);
        }
    }
}

} // namespace ifr
