// Bookkeeping and stores of a step over a paged cache: pages, slots and
// positions from request lengths (paged_plan_body, paged_rows_body), and the
// rotary embedding with the store of k and v to the slots (paged_rope_body).
#pragma once
#include "../paged_args.h"
#include "common.h"

namespace ifr {

// Sums that stay at the largest value instead of passing it (lengths come
// from the caller; sums past 2^32 - 1 only have to be seen to be too large).
IFR_DEV uint32_t add_sat(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// Inclusive saturating sum over the wave, by DPP: within rows of 16, then the
// rows' last lanes onto the rows behind them.
IFR_DEV uint32_t wave_scan(uint32_t v) {
    v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false)); // row_shr 1
    v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
    v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
    v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
    v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false)); // lane 15 of a row to the next, rows 1 and 3
    v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false)); // lane 31 to rows 2 and 3
    return v;
}
// Two inclusive saturating sums over a workgroup of up to 1024 threads, and
// its totals.  part: 32 entries of LDS, free again at the return.
IFR_DEV void block_scan2(uint32_t &x, uint32_t &y, uint32_t *part, uint32_t &total_x, uint32_t &total_y) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = (blockDim.x + 63) >> 6;
    x = wave_scan(x);
    y = wave_scan(y);
    if (lane == 63) {
        part[2 * wave] = x;
        part[2 * wave + 1] = y;
    }
    __syncthreads();
    // the waves' sums, one a lane, in every wave
    const uint32_t px = wave_scan(lane < nw ? part[2 * lane] : 0), py = wave_scan(lane < nw ? part[2 * lane + 1] : 0);
    total_x = __builtin_amdgcn_readlane(px, 63);
    total_y = __builtin_amdgcn_readlane(py, 63);
    const uint32_t w = __builtin_amdgcn_readfirstlane(wave);
    const uint32_t bx = w ? __builtin_amdgcn_readlane(px, w - 1) : 0, by = w ? __builtin_amdgcn_readlane(py, w - 1) : 0;
    x = add_sat(x, bx);
    y = add_sat(y, by);
    __syncthreads();
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

// The same for N consecutive x from x0, whose steps run side by side.
template <int N>
IFR_DEV void last_at_most_of(const uint32_t *a, uint32_t n, uint32_t x0, uint32_t (&at)[N]) {
#pragma unroll
    for (int z = 0; z < N; z++) at[z] = 0;
    for (uint32_t step = 1u << (31 - __builtin_clz(n)); step; step >>= 1) {
        uint32_t v[N];
#pragma unroll
        for (int z = 0; z < N; z++) v[z] = a[min(at[z] + step, n - 1)];
#pragma unroll
        for (int z = 0; z < N; z++)
            if (at[z] + step < n && v[z] <= x0 + z) at[z] += step;
    }
}

// Position and slot of row `row`, which is request r's (rows from `start` to
// `end`; kv rows of the cache after the step, 0: not granted).  page_of(i, first):
// the page with the request's rows from i << lp (first: this row is its first).
template <class F>
IFR_DEV void paged_row(const PagedPlanArgs &a, uint32_t row, uint32_t start, uint32_t end, uint32_t kv, F page_of) {
    uint32_t pos = PG_NO_ROW;
    uint64_t slot = ~0ull;
    if (kv && row < end) {
        pos = kv - (end - start) + (row - start);
        const uint32_t page = page_of(pos >> a.lp, !(pos & ((1u << a.lp) - 1)));
        if (page < a.n_pages) slot = ((uint64_t)page << a.lp) + (pos & ((1u << a.lp) - 1));
    }
    a.positions[row] = pos;
    a.slots[row] = slot;
}

// The requests of a step, by one workgroup: rounds of blockDim requests, the
// running sums carried between them.  (One workgroup: the free list and the
// table may be updated in place, and every request depends on the sums of
// those before it; a step has far fewer requests than rows.)  Bound by the
// latency of its chain: lengths, a scan, the popped pages with the pages of the
// rows.  The rows take their pages from where they come from (the request's
// last page, or the free list), not from the table entries written beside them.
// 32 decodes 4.1 us, 1021 requests of which a tenth are released 10 (a launch that
// does nothing: 3.3).
__device__ inline void paged_plan_body(const PagedPlanArgs &a) {
    __shared__ uint32_t part[32], s_fresh;
    __shared__ uint32_t s_start[PG_PLAN_THREADS + 1], s_off[PG_PLAN_THREADS], s_held[PG_PLAN_THREADS], s_kv[PG_PLAN_THREADS];
    const uint32_t tid = threadIdx.x, T = blockDim.x, pm = (1u << a.lp) - 1;
    const uint32_t cap = a.max_pages << a.lp; // at most 2^30
    // the first round's lengths, read once for both passes
    const uint32_t ctx0 = tid < a.n_requests ? a.ctx_len[tid] : 0, new0 = tid < a.n_requests ? a.new_len[tid] : 0;
    uint32_t top = min(*a.free_count, a.n_pages);

    // Released requests' pages onto the stack, those that are pages, in order:
    // the entries of a round's released requests one after another, four per
    // thread and pass.
    bool pushed = false;
    for (uint32_t base = 0; base < a.n_requests; base += T) {
        const uint32_t r = base + tid;
        uint32_t held = 0;
        if (r < a.n_requests && (base ? a.new_len[r] : new0) == PG_RELEASE)
            held = (uint32_t)min((uint64_t)a.max_pages, ((uint64_t)(base ? a.ctx_len[r] : ctx0) + pm) >> a.lp);
        if (!__syncthreads_or(held != 0)) continue;
        pushed = true;
        // those that hold pages in a list: where each one's entries begin, and which it is (s_off, free until below)
        uint32_t upto = held, listed = held != 0, total, n_listed, no;
        block_scan2(upto, listed, part, total, n_listed);
        if (held) {
            s_start[listed - 1] = upto - held;
            s_off[listed - 1] = r;
        }
        __syncthreads();
        constexpr int N = 4;
        for (uint32_t first = 0; first < total; first += N * T) {
            uint32_t page[N], count = 0, zero = 0, all;
            const uint32_t i0 = first + N * tid;
            uint32_t j = i0 < total ? last_at_most(s_start, n_listed, i0) : 0;
#pragma unroll
            for (int z = 0; z < N; z++) {
                page[z] = ~0u;
                if (i0 + z < total) {
                    // (each has an entry at least: the next entry is its own or the next one's first)
                    if (z && j + 1 < n_listed && s_start[j + 1] <= i0 + z) j++;
                    page[z] = a.table[(size_t)s_off[j] * a.max_pages + (i0 + z - s_start[j])];
                }
            }
#pragma unroll
            for (int z = 0; z < N; z++) count += page[z] < a.n_pages;
            uint32_t to = count;
            block_scan2(to, zero, part, all, no);
            to += top - count;
#pragma unroll
            for (int z = 0; z < N; z++)
                if (page[z] < a.n_pages) {
                    if (to < a.n_pages) a.free_pages[to] = page[z];
                    to++;
                }
            top = min(top + all, a.n_pages);
        }
        __syncthreads();
    }
    if (pushed) __syncthreads(); // read below by other waves of this workgroup

    // rows0: rows of the requests before the round; need0: pages that they need; taken: pages they got
    uint32_t rows0 = 0, need0 = 0, taken = 0;
    for (uint32_t base = 0; base < a.n_requests; base += T) {
        const uint32_t r = base + tid, nr = min(T, a.n_requests - base);
        const bool in = r < a.n_requests;
        const uint32_t ctx = !base ? ctx0 : in ? a.ctx_len[r] : 0, nw = !base ? new0 : in ? a.new_len[r] : 0;
        const bool gone = nw == PG_RELEASE;
        // (one row past n_rows is as good as any more: the sums then stay exact up to there)
        const uint32_t n = gone ? 0 : min(nw, a.n_rows + 1), sum = gone ? ctx : add_sat(ctx, nw);
        const uint32_t held = (uint32_t)(((uint64_t)ctx + pm) >> a.lp);
        const bool room = in && !gone && sum <= cap;
        const uint32_t need = room ? ((sum + pm) >> a.lp) - held : 0;
        // Rows and pages in one scan.  (A request whose rows end past n_rows counts for no pages, but all
        // behind it end there too, so nobody asks for the sums that it is in.)
        uint32_t end = n, off = need, total_rows, total_need;
        if (tid == 0) s_fresh = 0;
        block_scan2(end, off, part, total_rows, total_need);
        end = add_sat(end, rows0);
        off = add_sat(off, need0); // with its own
        const uint32_t start = min(end - n, a.n_rows); // (a saturated sum's too is past n_rows)
        const bool ok = room && end <= a.n_rows && (!need || off <= top);
        if (in) {
            a.row_start[r] = start;
            a.kv_len[r] = ok ? sum : 0u;
            if (a.ctx_len_out) a.ctx_len_out[r] = ok ? sum : gone ? 0u : ctx;
        }
        // Pages are granted up to the first request that they do not reach, so a granted request's pages begin
        // where the sum of needs does.
        off -= need;
        s_off[tid] = off;
        s_start[tid] = start;
        s_held[tid] = held;
        s_kv[tid] = ok ? sum : 0u;
        if (tid == nr - 1) s_start[nr] = min(end, a.n_rows);
        if (ok && need) atomicMax(&s_fresh, off + need);
        __syncthreads();
        const uint32_t fresh = max(s_fresh, taken);
        // where the rows are another launch's, their new pages' entries are too, from where each request's pages begin
        if (!a.rows_here && in) a.pops[r] = off;
        // the round's new table entries: popped page i is request j's, the last one whose pages begin at or before
        // i (one without new pages shares its place with the next)
        auto entry = [&](uint32_t i, uint32_t j) {
            a.table[(size_t)(base + j) * a.max_pages + s_held[j] + (i - s_off[j])] = a.free_pages[top - 1 - i];
        };
        if (!a.rows_here) {
        } else if (fresh - taken <= T) {
            if (taken + tid < fresh) entry(taken + tid, last_at_most(s_off, nr, taken + tid));
        } else {
            for (uint32_t i = taken + 4 * tid; i < fresh; i += 4 * T) {
                uint32_t j[4];
                last_at_most_of(s_off, nr, i, j);
#pragma unroll
                for (int z = 0; z < 4; z++)
                    if (i + z < fresh) entry(i + z, j[z]);
            }
        }
        if (a.rows_here) {
            const uint32_t first = s_start[0], last = base + nr == a.n_requests ? a.n_rows : s_start[nr];
#pragma unroll 2
            for (uint32_t row = first + tid; row < last; row += T) {
                const uint32_t j = last_at_most(s_start, nr, row);
                paged_row(a, row, s_start[j], s_start[j + 1], s_kv[j], [&](uint32_t i, bool) {
                    return i < s_held[j] ? a.table[(size_t)(base + j) * a.max_pages + i]
                                         : a.free_pages[top - 1 - (s_off[j] + i - s_held[j])];
                });
            }
        }
        taken = fresh;
        rows0 = add_sat(rows0, total_rows);
        need0 = add_sat(need0, total_need);
        __syncthreads();
    }
    if (!a.n_requests) // no request has any of the rows
        for (uint32_t row = tid; row < a.n_rows; row += T) paged_row(a, row, 0, 0, 0, [](uint32_t, bool) { return 0u; });
    if (tid == 0) {
        a.row_start[a.n_requests] = min(rows0, a.n_rows);
        *a.free_count_out = top - taken;
        if (!a.rows_here) a.pops[a.n_requests] = top;
    }
}

// The rows of a large step, 256 threads each with rows of their own, and the
// table entries of their new pages (every new page has a new row that is its
// first).  A workgroup finds its first row's request by a 256-way search of
// row_start, and its rows' among the next 1024 requests' starts in LDS: 58885
// rows of 1021 requests 5 us.
constexpr uint32_t PG_ROWS_PER = 512, PG_ROWS_WIN = 1024;

__device__ inline void paged_rows_body(const PagedPlanArgs &a) {
    __shared__ uint32_t s_start[PG_ROWS_WIN + 1], s_kv[PG_ROWS_WIN], s_pops[PG_ROWS_WIN], s_n;
    const uint32_t tid = threadIdx.x, row0 = blockIdx.x * PG_ROWS_PER;
    // the last request that starts at or before row0 (requests without rows
    // share their start with the next: the last one of them has row0)
    uint32_t lo = 0, hi = a.n_requests <= PG_ROWS_WIN ? 1 : a.n_requests; // (all in the window: from the first)
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
        s_pops[i] = a.pops[r0 + i];
    }
    if (tid == 0) s_start[nr] = a.row_start[r0 + nr];
    __syncthreads();
    const uint32_t top = a.pops[a.n_requests], pm = (1u << a.lp) - 1;
    auto fill = [&](uint32_t row, uint32_t r, uint32_t start, uint32_t end, uint32_t kv, uint32_t pops) {
        const uint32_t held = (kv - (end - start) + pm) >> a.lp; // (of a granted request)
        paged_row(a, row, start, end, kv, [&](uint32_t i, bool first) {
            uint32_t *entry = a.table + (size_t)r * a.max_pages + i;
            if (i < held) return *entry;
            const uint32_t page = a.free_pages[top - 1 - (pops + i - held)];
            if (first) *entry = page;
            return page;
        });
    };
    for (uint32_t row = row0 + tid; row < min(row0 + PG_ROWS_PER, a.n_rows); row += 256) {
        if (row < s_start[nr] || r0 + nr == a.n_requests) {
            const uint32_t j = last_at_most(s_start, nr, row);
            fill(row, r0 + j, s_start[j], s_start[j + 1], s_kv[j], s_pops[j]);
        } else { // more requests than the window between this row and the workgroup's first
            const uint32_t r = last_at_most(a.row_start, a.n_requests, row);
            fill(row, r, a.row_start[r], a.row_start[r + 1], a.kv_len[r], a.pops[r]);
        }
    }
}

// ------------------------------------------------------ RoPE and the store --
// Workgroup (row, part): the part's 8-element items of the row (one part where
// the rows fill the chip).  The row's angles' (cos, sin) go to LDS, one angle
// per thread: theta_j = 2^(-2j/hs log2(base)) and pos * theta_j / 2pi in 64
// bits, reduced to a fraction of a turn there, cos and sin of it in f32 (at
// position 1e5 an f32 product would be off by 4e-3).  An item is four pairs of
// one head: eight contiguous elements, or four and the four half a head away
// (NeoX).  Memory bound: each element is read once and written once.
// 8190 rows of 48 heads of 128, f32 to an f16 cache: 58 us, 5.2 TB/s (in
// workgroups of four rows, whose trigonometry fills their threads, 71: fewer of
// them overlap their loads); 32 rows 4.3 us, with one workgroup a row 4.9.
constexpr uint32_t PG_ROPE_LDS = 64; // (cos, sin) pairs of a row

__device__ inline void paged_rope_body(const PagedRopeArgs &a) {
    __shared__ float2 cs[PG_ROPE_LDS];
    const uint32_t tid = threadIdx.x, hh = a.hs / 2, cpi = a.hs / 8;
    const size_t row = blockIdx.x;
    const uint32_t pos = a.positions[row];
    if (pos == PG_NO_ROW) return;
    const uint64_t slot = a.slots[row], page = slot >> a.lp;
    if (tid < hh) {
        float c = 1.0f, s = 0.0f;
        if (a.turn) {
            const double th = exp2(-(double)(2 * tid) / (double)a.hs * a.log2_base);
            double t = (double)pos * th * 0.15915494309189533577; // in turns
            t -= rint(t);
            sincospif((float)(2.0 * t), &s, &c);
        }
        cs[tid] = make_float2(c, s);
    }
    __syncthreads();
    const uint32_t heads = (a.q ? a.n_heads : 0) + 2 * a.n_kv, items = heads * cpi;
    for (uint32_t it = blockIdx.y * PG_ROPE_THREADS + tid; it < items; it += a.parts * PG_ROPE_THREADS) {
        const uint32_t h = it / cpi, ci = it % cpi;
        const uint32_t nq = heads - 2 * a.n_kv;
        const uint32_t what = h < nq ? 0u : h < nq + a.n_kv ? 1u : 2u; // q, k, v
        const uint32_t head = h - (what == 0 ? 0 : what == 1 ? nq : nq + a.n_kv);
        const bool pairs_apart = a.neox && what < 2;
        // the item's elements: e0 .. +4 and e1 .. +4 of the head
        const uint32_t e0 = pairs_apart ? 4 * ci : 8 * ci, e1 = pairs_apart ? e0 + hh : e0 + 4;
        const float *x = (what == 0 ? a.q + row * a.ld_q : what == 1 ? a.k + row * a.ld_k : a.v + row * a.ld_v) +
                         (size_t)head * a.hs;
        const float4 u = *(const float4 *)(x + e0), v = *(const float4 *)(x + e1);
        float y[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        if (what < 2 && a.turn) {
            const float2 *ang = cs + 4 * ci;
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
