// Attention of several requests' new rows over a paged cache.
//
//   out = softmax_j(scale q . k_j) . v_j  over the rows j that the row at
//   position p sees: j <= p, and under a window w also j > p - w or j < sinks.
//
// Work is cut into tiles: the queries q0 .. q0 + QT - 1 of one request times
// the heads of one KV head (its G query heads, or a sub-group of them), so a
// K/V row read once serves all of them.  A tile's visible keys are key tiles
// of the cache (sinks first, then from the window's start to its last
// query), which up to n_splits workgroups share; with more than one, each
// leaves a partial (m, l, o) and paged_attn_merge joins them.
//
// Scores are kept in base-2 units (scale2 = scale log2 e).  The running
// reference r of a row (m of the partials) is a value near its maximum so far
// that the weights 2^(s - r) are taken against; -inf until a score above -inf
// came, and a row that ends there is 0.
#pragma once
#include "../paged_args.h"
#include "attention.h"

namespace ifr {

typedef float float4v __attribute__((ext_vector_type(4)));

// Operand types: q, cache and output f16; q and output f32 over an f16 cache
// (q and the softmax weights in two f16 parts each, 22 bits); all f32 (f32
// matrix products).
enum PaType : int { PA_H = 0, PA_M = 1, PA_S = 2 };

// A tile of a request's queries, the same for all lanes.
struct PaTile {
    uint32_t r, row0;   // request; packed row of the first query
    uint32_t nq;        // queries
    int32_t p0, plast;  // positions of the first and last query (p0 may be negative)
};
// Its key tiles of KT rows: `ns` from row 0 (sinks), then from tile `lo`; n in all.
struct PaKeys {
    uint32_t ns, lo, n;
};
// Weights are 2^(s - r + 7): the largest that the reference lets through, 2^15,
// is an f16 number still, and f16's smallest normal one is 2^-21 of a row's largest
// weight.  (The factor is in the sums and the weighted rows alike.)
constexpr float PA_UP = 7.0f;
template <int KT>
IFR_DEV PaKeys pa_keys(const PagedAttnArgs &a, const PaTile &t) {
    PaKeys k = {0, 0, 0};
    if (t.plast < 0) return k;
    const uint32_t first = a.window ? (uint32_t)max(t.p0 - (int32_t)a.window + 1, 0) : 0u;
    k.lo = first / KT;
    k.ns = min((min(a.sinks, first) + KT - 1) / KT, k.lo);
    k.n = k.ns + (uint32_t)t.plast / KT + 1 - k.lo;
    return k;
}
// Key tiles of each split of a tile with n: the launch's chunk, or more where
// its splits would not reach.
IFR_DEV uint32_t pa_chunk(const PagedAttnArgs &a, uint32_t n) { return max((n + a.n_splits - 1) / a.n_splits, a.chunk); }

// Entry i of a table that no kernel writes meanwhile, at an index that all
// lanes share: a scalar load, which the waits for the rows on their way do not
// order (a vector load here would wait for all of them).
IFR_DEV uint32_t pa_entry(const uint32_t *p, uint32_t i) {
    typedef const __attribute__((address_space(4))) uint32_t const_u32;
    return ((const_u32 *)(uintptr_t)p)[i];
}

// An address that all lanes share, in scalar registers.
IFR_DEV const char *pa_scalar(const char *p) {
    const uint64_t x = (uint64_t)p;
    return (const char *)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x));
}
// Rows and cache length of request r, whatever the buffers hold.
IFR_DEV void pa_request(const PagedAttnArgs &a, uint32_t r, uint32_t &row0, uint32_t &n, uint32_t &kv) {
    row0 = min(a.row_start[r], a.n_rows);
    n = min(max(a.row_start[r + 1], row0), a.n_rows) - row0;
    kv = min(a.kv_len[r], a.max_pages << a.lp);
}
// The same for a request that all lanes share (in scalar registers).
IFR_DEV void pa_request_uniform(const PagedAttnArgs &a, uint32_t r, uint32_t &row0, uint32_t &n, uint32_t &kv) {
    const uint32_t s0 = pa_entry(a.row_start, r), s1 = pa_entry(a.row_start, r + 1), len = pa_entry(a.kv_len, r);
    row0 = min(s0, a.n_rows);
    n = min(max(s1, row0), a.n_rows) - row0;
    kv = min(len, a.max_pages << a.lp);
}
// Queries [q0, q0 + QT) of request r's n rows from row0.
IFR_DEV PaTile pa_tile(const PagedAttnArgs &a, uint32_t r, uint32_t row0, uint32_t n, uint32_t kv, uint32_t q0) {
    PaTile t;
    t.r = r;
    t.row0 = row0 + q0;
    t.nq = min(a.QT, n - q0);
    // a request without rows in the cache (refused) sees nothing
    t.p0 = kv ? (int32_t)kv - (int32_t)n + (int32_t)q0 : -(1 << 30);
    t.plast = t.p0 + (int32_t)t.nq - 1;
    return t;
}
IFR_DEV uint32_t pa_wave_sum(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v; // inclusive; lane 63 has the sum
}
// The lane that has the `left`-th of the lanes' things (`mine` each), and how many the lanes before it have.
IFR_DEV bool pa_pick(uint32_t mine, uint32_t left, uint32_t &src, uint32_t &before) {
    const uint32_t sum = pa_wave_sum(mine);
    const uint64_t has = __ballot(sum > left);
    if (!has) return false;
    src = __builtin_amdgcn_readfirstlane((uint32_t)__ffsll((unsigned long long)has) - 1);
    before = __builtin_amdgcn_readlane(sum - mine, src);
    return true;
}
// The `at`-th tile of all requests; false if there are fewer.  Sorted and up to
// 64 requests, one a lane: the tiles in the order of their last positions (by 64),
// the farthest first, so that the workgroups with the most keys start first
// (nine requests' chunks 504 us, in the order of the requests 567).
// Else from the last request's last tile, 64 requests a step (16 of 4 rows over 300 6.6 us, sorted 7.1).
IFR_DEV bool pa_find(const PagedAttnArgs &a, bool sorted, uint32_t at, uint32_t &r, uint32_t &q0) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t src = 0, before = 0;
    if (a.n_requests == 1) {
        uint32_t row0, n, kv;
        pa_request_uniform(a, 0, row0, n, kv);
        const uint32_t nt = (n + a.QT - 1) / a.QT;
        r = 0;
        q0 = (nt - 1 - at) * a.QT;
        return at < nt;
    }
    if (sorted) {
        uint32_t row0, n = 0, kv = 0, nt = 0;
        if (lane < a.n_requests) {
            pa_request(a, lane, row0, n, kv);
            nt = (n + a.QT - 1) / a.QT;
        }
        // tiles of this lane's request whose last position is 64 x or more (x = 0: all)
        auto count = [&](uint32_t x) {
            const int32_t least = (int32_t)(64 * x);
            if (!x) return nt;
            if (!nt || (int32_t)kv <= least) return 0u;
            const int32_t up = least + 1 - (int32_t)kv + (int32_t)n; // tile c - 1 ends there if c QT reaches it
            const uint32_t c = up > (int32_t)a.QT ? ((uint32_t)up + a.QT - 1) / a.QT : 1u;
            return c < nt ? 1 + nt - c : 1u;
        };
        auto total = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane(pa_wave_sum(count(x)), 63); };
        if (total(0) <= at) return false;
        uint32_t lo = 0, hi = (a.max_pages << a.lp) / 64 + 1; // total(lo) > at >= total(hi)
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (total(mid) > at) lo = mid;
            else hi = mid;
        }
        const uint32_t more = count(hi), mine = count(lo) - more;
        if (!pa_pick(mine, at - total(hi), src, before)) return false;
        const uint32_t e = at - total(hi) - before + __builtin_amdgcn_readlane(more, src); // from the request's last tile
        r = src;
        q0 = (__builtin_amdgcn_readlane(nt, src) - 1 - e) * a.QT;
        return true;
    }
    uint32_t left = at;
    for (uint32_t top = a.n_requests; top;) {
        // lane 0 has the last request not yet counted
        uint32_t nt = 0;
        if (lane < top) {
            uint32_t row0, n, kv;
            pa_request(a, top - 1 - lane, row0, n, kv);
            nt = (n + a.QT - 1) / a.QT;
        }
        if (pa_pick(nt, left, src, before)) {
            r = top - 1 - src;
            q0 = (__builtin_amdgcn_readlane(nt, src) - 1 - (left - before)) * a.QT;
            return true;
        }
        left -= __builtin_amdgcn_readlane(pa_wave_sum(nt), 63);
        top -= min(top, 64u);
    }
    return false;
}

// Key tiles of each split of request r's tiles, where a workgroup serves them all: by its last tile's keys.  (Under
// a window an earlier tile may have one more, as its ends fall, and one more as the last has fewer rows.)
template <int KT>
IFR_DEV uint32_t pa_request_chunk(const PagedAttnArgs &a, uint32_t r, uint32_t row0, uint32_t n, uint32_t kv, uint32_t &keys) {
    keys = pa_keys<KT>(a, pa_tile(a, r, row0, n, kv, n ? (n - 1) / a.QT * a.QT : 0)).n;
    if (a.window && n > a.QT) keys += 2;
    return pa_chunk(a, keys);
}
// The `at`-th split of all requests, the longest first (whole chunks, then the
// requests' last parts by length): workgroups of unequal lengths, the long ones
// started last, had left the chip half empty at the end (64 decodes of 200 to
// 8192 rows 123 us, in the order of the requests 139).  In the
// order of splits and requests where each has a CU of its own (8 decodes of 200 7.0
// us, sorted 8.0; with two a CU the parts of a long sequence would share theirs, 16
// of 50 to 8000 69 us for 44), and for more than 64 requests.
template <int KT>
IFR_DEV bool pa_find_split(const PagedAttnArgs &a, uint32_t at, uint32_t &r, uint32_t &split) {
    const uint32_t R = a.n_requests, lane = threadIdx.x & 63;
    r = R == 1 ? 0 : at % R;
    split = R == 1 ? at : at / R;
    if (!a.sorted) return split < a.n_splits;
    uint32_t full = 0, rest = 0; // whole chunks; key tiles of the last part, and one (0: there is none)
    if (lane < R) {
        uint32_t row0, n, kv, keys;
        pa_request(a, lane, row0, n, kv);
        const uint32_t C = pa_request_chunk<KT>(a, lane, row0, n, kv, keys);
        full = n ? keys / C : 0;
        rest = n && (keys % C || !full) ? keys % C + 1 : 0;
    }
    uint32_t src = 0, before = 0;
    if (pa_pick(full, at, src, before)) {
        r = src;
        split = at - before;
        return true;
    }
    // the k-th largest of the last parts, bit by bit from the top (a comparison of each with all took 2.5 us of 64
    // requests' 14); equal ones in the order of the requests
    uint32_t k = at - (uint32_t)__builtin_amdgcn_readlane(pa_wave_sum(full), 63);
    uint64_t left = __ballot(rest);
    if ((uint32_t)__popcll(left) <= k) return false;
    uint32_t most = a.chunk + 1; // (a chunk is longer where the splits would not reach)
    while (__ballot(rest > most)) most *= 2;
    for (int bit = 31 - __builtin_clz(most); bit >= 0; bit--) {
        const uint64_t ones = left & __ballot(rest >> bit & 1u);
        const uint32_t c = (uint32_t)__popcll(ones);
        if (k < c) left = ones;
        else {
            k -= c;
            left &= ~ones;
        }
    }
    const uint32_t ahead = __builtin_amdgcn_mbcnt_hi((uint32_t)(left >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)left, 0));
    r = (uint32_t)__ffsll((unsigned long long)(left & __ballot(ahead == k))) - 1;
    split = __builtin_amdgcn_readlane(full, r);
    return true;
}

// max and sum over the four lanes of a row (lanes n, n + 16, n + 32, n + 48)
IFR_DEV float pa_max4(float v) {
    return attn_groups_reduce<128>(v, [](float x, float y) { return fmaxf(x, y); });
}
IFR_DEV float pa_sum4(float v) {
    return attn_groups_reduce<128>(v, [](float x, float y) { return x + y; });
}

// element i of an f32 or f16 array
template <bool F32>
IFR_DEV float pa_at(const void *p, size_t i) {
    if constexpr (F32) return ((const float *)p)[i];
    else return (float)((const _Float16 *)p)[i];
}

// x in two f16 parts: 22 bits of it (both parts rounded to nearest)
IFR_DEV void pa_split(float x, _Float16 &hi, _Float16 &lo) {
    hi = (_Float16)x;
    lo = (_Float16)(x - (float)hi);
}

// Asks the scheduler for LEAD operands' LDS reads (READS each), then a product and the
// next operand's reads in turn, N operands in all (PRODUCTS each).  Left to itself
// it keeps one read ahead, and every product waits out most of the LDS latency.
template <int LEAD, int N, int PRODUCTS, int READS>
IFR_DEV void pa_interleave() {
    __builtin_amdgcn_sched_group_barrier(0x100, LEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < N - LEAD; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, PRODUCTS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, LEAD * PRODUCTS, 0);
}

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
// two f32 to a pair of f16, to nearest
IFR_DEV uint32_t pa_pack(float x, float y) { return __builtin_bit_cast(uint32_t, half2v{(_Float16)x, (_Float16)y}); }
// acc + both halves of a pair
IFR_DEV float pa_add2(uint32_t h, float acc) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, h), half2v{(_Float16)1, (_Float16)1}, acc, false);
}
// x and y in two f16 parts each: the second is x - hi, formed and rounded in one
// mixed-precision multiply-add.  (The pair and the -1 are hidden from the
// compiler, which otherwise converts twice and back.)
IFR_DEV void pa_split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    hi = pa_pack(x, y);
    float minus = -1.0f;
    asm("" : "+v"(hi));
    asm("" : "+v"(minus));
    const half2v h = __builtin_bit_cast(half2v, hi);
    lo = __builtin_bit_cast(uint32_t, half2v{(_Float16)__builtin_fmaf((float)h[0], minus, x), (_Float16)__builtin_fmaf((float)h[1], minus, y)});
}

IFR_DEV bool pa_odd(float x) { return (__float_as_uint(x) & 0x7F800000u) == 0x7F800000u; } // infinite or NaN

// The power of two that a query row of largest value mx is scaled by before it
// is split: its largest value comes into [2^14, 2^15), so that the second
// parts of values down to 2^-17 of it are normal f16 numbers.  (A row below
// 2^-46 keeps a factor of 2^60, so that the scores' factor, its inverse, does not vanish.)
IFR_DEV int pa_q_exponent(float mx) { return mx > 0.0f && !pa_odd(mx) ? min(14 - ilogbf(mx), 60) : 0; }

// --------------------------------------------------------- 16-row kernel --
// One workgroup of four waves per (tile, KV head, sub-group of heads, split):
// the tile's up to 16 (query, head) rows are one side of every product, and
// the waves take the split's key tiles of 32 rows in turn.  K and V go from
// the cache straight into registers in the layout the matrix products read:
//   S^T = K Q^T   lane (n = lane % 16, g = lane / 16) loads 16 bytes of the rows n
//                 and 16 + n of the key tile at dims 32c + 8g;
//   O^T = V^T P^T lane loads dims 8n .. 8n + 7 of the rows 16u + 4g + e (a whole
//                 row per 16 lanes): the score accumulator holds exactly the
//                 weights of these rows for query row n, so P^T needs no
//                 exchange, and V^T's operand for output tile t is element t of
//                 the eight rows' loads, an 8 x 8 transpose of halves inside
//                 the lane (output row i of tile t is dim 8i + t).
// So there is no LDS and no barrier in the loop; the waves' states are joined
// through LDS once.  Rows whose page is no page read page 0 and are masked.
// Bound by memory where the keys are many: 64 decodes of 200 to 8192 rows, 8 KV
// heads of 128 in f16, 123 us, 4.8 TB/s; two of 106 K and 131 K 189 us, 5.1
// TB/s (a large copy: 4.8).  Both need the next key tile's loads in flight over
// the products, which is 8 waves a CU by the registers; with 12 waves, and 43
// registers spilled for them, the former is 205 us.  Short calls are a chain of trips to
// memory: one decode of 145 rows 5.5 us.
// Chunks of f32 caches run here too, in RB = 2 blocks of 16 rows, which halve
// what the caches behind the loads have to give (the products of one block need
// 11 TB/s of K and V); the queries are then read from LDS.  2048 rows over 4096,
// 32 heads of 128: 1555 us, 110 TFLOP/s (one block 1732; a library's f32 product
// 154), 12 heads 632 (835), 32 heads of 64 825 (961).
constexpr int PAD_WAVES = 4;
// 16-row blocks of a key tile: two, which the f16 products' eight keys a lane
// need; one for f32 rows of 128, whose two blocks do not fit the registers (54
// spilled: 1191 rows over 1869 of 32 heads 379 us, with one 249).
template <int HSP, int T>
constexpr int PAD_NU = T == PA_S && HSP == 128 ? 1 : 2;

template <int HSP, int T>
struct PaRegs {
    static constexpr int KC = T == PA_S ? HSP / 16 : HSP / 32; // 16-byte loads of a K row
    static constexpr int DV = HSP / 16;                        // dims of a V row per lane
    uint4 k[PAD_NU<HSP, T>][KC];
    uint32_t v[4 * PAD_NU<HSP, T>][T == PA_S ? DV : DV / 2];
};

template <int HSP, int T, int RB>
__device__ void pa_rows16_body(const PagedAttnArgs &a) {
    constexpr int ES = T == PA_S ? 4 : 2, KC = PaRegs<HSP, T>::KC, DV = HSP / 16, NU = PAD_NU<HSP, T>, PAD_KT = 16 * NU, ROWS = 16 * RB;
    constexpr int OP = HSP + 4;
    __shared__ __attribute__((aligned(16))) float og[PAD_WAVES][ROWS][OP];
    __shared__ float mg[PAD_WAVES][ROWS], lg[PAD_WAVES][ROWS];
    const uint32_t tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t b = blockIdx.x;
    const uint32_t kvh = b % a.n_kv;
    b /= a.n_kv;
    const uint32_t sub = b % a.n_sub;
    b /= a.n_sub;
    const uint32_t hs = a.hs, heads = min(a.heads_per, a.G - sub * a.heads_per);
    uint32_t r, q0 = 0, split = blockIdx.y, row0, nrows, kv, last_keys;
    if (a.search ? !pa_find(a, a.sorted, b, r, q0) : !pa_find_split<PAD_KT>(a, b, r, split)) return;
    pa_request_uniform(a, r, row0, nrows, kv);
    const uint32_t qend = a.search ? q0 + 1 : nrows, chunk = pa_request_chunk<PAD_KT>(a, r, row0, nrows, kv, last_keys);
    const uint32_t *tab = a.table + (size_t)r * a.max_pages;
    const uint32_t pm = (1u << a.lp) - 1;
    uint32_t head[RB]; // of this lane's rows n + 16 b
#pragma unroll
    for (int b = 0; b < RB; b++) head[b] = kvh * a.G + sub * a.heads_per + (n + 16 * b) % heads;

    for (; q0 < qend; q0 += a.QT) {
        const PaTile t = pa_tile(a, r, row0, nrows, kv, q0);
        const PaKeys keys = pa_keys<PAD_KT>(a, t);
        const uint32_t C = a.search ? pa_chunk(a, keys.n) : chunk, i0 = split * C, i1 = min(i0 + C, keys.n);
        const bool one = keys.n <= C; // (a tile without keys too: split 0 writes its zeros)
        if (i0 >= i1 && !(one && split == 0)) continue;
        // a row sees the keys k <= qpos with k > qlow or k < sinks
        bool row_ok[RB];
        int32_t qpos[RB], qlow[RB];
        const int32_t sinks = (int32_t)a.sinks;
        uint32_t gq[RB]; // packed row
#pragma unroll
        for (int b = 0; b < RB; b++) {
            const uint32_t qi = (n + 16 * b) / heads;
            row_ok[b] = qi < t.nq;
            qpos[b] = row_ok[b] ? t.p0 + (int32_t)qi : -1;
            qlow[b] = a.window ? qpos[b] - (int32_t)a.window : -1;
            gq[b] = t.row0 + (row_ok[b] ? qi : 0);
        }

        float4v o[RB][DV];
        float m[RB], l[RB];

        auto tile_of = [&](uint32_t i) { return i < keys.ns ? i : keys.lo + i - keys.ns; };
        // page of the 16 rows from 16 * b16
        auto page_of = [&](uint32_t b16) {
            return pa_entry(tab, min(b16 >> (a.lp - 4), a.max_pages - 1));
        };
        PaRegs<HSP, T> x;
        const uint32_t dk = T == PA_S ? 4 * g : 8 * g, dv = DV * n;
        auto base_of = [&](const void *p, uint32_t page, uint32_t row) {
            return (const char *)p + ((int64_t)(page < a.n_pages ? page : 0u) * a.page_stride +
                                      (int64_t)(row & pm) * a.row_stride + (int64_t)kvh * a.head_stride) * ES;
        };
        auto load_k = [&](uint32_t kt, uint32_t pg0, uint32_t pg1) {
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const char *p = base_of(a.key, u ? pg1 : pg0, kt * PAD_KT + 16 * u);
                const uint32_t off = n * (uint32_t)a.row_stride;
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const uint32_t d = (T == PA_S ? 16 : 32) * c + dk;
                    x.k[u][c] = *(const uint4 *)(p + (size_t)(off + (HSP == 128 && hs == 128 ? d : min(d, hs - (T == PA_S ? 4 : 8)))) * ES);
                }
            }
        };
        auto load_v = [&](uint32_t kt, uint32_t pg0, uint32_t pg1) {
#pragma unroll
            for (int u = 0; u < NU; u++) {
                const char *p = base_of(a.value, u ? pg1 : pg0, kt * PAD_KT + 16 * u);
                const uint32_t d = min(dv, hs - DV);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const char *s = p + (size_t)((4 * g + e) * (uint32_t)a.row_stride + d) * ES;
                    uint32_t *w = x.v[4 * u + e];
                    constexpr int W = sizeof(x.v[0]) / 4; // 2, 4 or 8 words
                    if constexpr (W == 2) {
                        const uint2 y = *(const uint2 *)s;
                        w[0] = y.x; w[1] = y.y;
                    } else {
#pragma unroll
                        for (int z = 0; z < W; z += 4) {
                            const uint4 y = *(const uint4 *)(s + 4 * z);
                            w[z] = y.x; w[z + 1] = y.y; w[z + 2] = y.z; w[z + 3] = y.w;
                        }
                    }
                }
            }
        };

        // the first tile's rows on their way before anything else is waited for
        uint32_t kt = 0, pg0 = 0, pg1 = 0, kn = 0, pn0 = 0, pn1 = 0;
        if (i0 + wave < i1) {
            kt = tile_of(i0 + wave);
            kn = tile_of(min(i0 + wave + PAD_WAVES, i1 - 1));
            pg0 = page_of(NU * kt);
            pg1 = page_of(NU * kt + 1);
            pn0 = page_of(NU * kn);
            pn1 = page_of(NU * kn + 1);
            load_k(kt, pg0, pg1);
            load_v(kt, pg0, pg1);
        }
        __builtin_amdgcn_sched_barrier(0);

        // q: dims 32c + 8g .. of row n (f32 cache: 16c + 4g ..)
        half8v qh[T == PA_S ? 1 : KC], ql[T == PA_M ? KC : 1];
        float4v qf[T == PA_S && RB == 1 ? KC : 1];
        float rs = a.scale2; // of the row's raw scores
#pragma unroll
        for (int b = 0; b < RB; b++) {
            static_assert(RB == 1 || T == PA_S, "rows of f32 only in larger tiles");
            const char *qp = (const char *)a.q + ((size_t)gq[b] * a.ld_q + (size_t)head[b] * hs) * (T == PA_H ? 2 : 4);
            if constexpr (T == PA_H) {
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const uint32_t d = 32 * c + 8 * g;
                    const bool ok = row_ok[b] && d < hs;
                    uint4 x = *(const uint4 *)(qp + 2 * (ok ? d : 0));
                    if (!ok) x = make_uint4(0, 0, 0, 0);
                    qh[c] = __builtin_bit_cast(half8v, x);
                }
            } else if constexpr (T == PA_M) {
                // scaled by a power of two that puts the row's largest value in [2^14, 2^15)
                float x[KC][8], mx = 0.0f;
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const uint32_t d = 32 * c + 8 * g;
                    const bool ok = row_ok[b] && d < hs;
                    const float4 u = *(const float4 *)(qp + 4 * (ok ? d : 0)), w = *(const float4 *)(qp + 4 * (ok ? d : 0) + 16);
                    const float y[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[c][e] = ok ? y[e] : 0.0f;
                        mx = fmaxf(mx, fabsf(x[c][e]));
                    }
                }
                mx = pa_max4(mx);
                const int ex = pa_q_exponent(mx);
                rs = ldexpf(rs, -ex);
#pragma unroll
                for (int c = 0; c < KC; c++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        _Float16 hi, lo;
                        pa_split(ldexpf(x[c][e], ex), hi, lo);
                        qh[c][e] = hi;
                        ql[c][e] = lo;
                    }
            } else {
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const uint32_t d = 16 * c + 4 * g;
                    const bool ok = row_ok[b] && d < hs;
                    const float4 x = *(const float4 *)(qp + 4 * (ok ? d : 0));
                    const float4v y = ok ? float4v{x.x, x.y, x.z, x.w} : float4v{0, 0, 0, 0};
                    if constexpr (RB == 1) qf[c] = y;
                    else if (wave == 0) *(float4v *)&og[0][n + 16 * b][d] = y; // (two blocks' q do not fit the registers)
                }
            }
        }
        if constexpr (RB > 1) __syncthreads();

        auto clear = [&]() {
#pragma unroll
            for (int b = 0; b < RB; b++) {
#pragma unroll
                for (int d = 0; d < DV; d++) o[b][d] = float4v{0, 0, 0, 0};
                m[b] = -INFINITY;
                l[b] = 0.0f;
            }
        };
        clear();
            for (uint32_t i = i0 + wave; i < i1; i += PAD_WAVES) {
                const uint32_t k0 = kt * PAD_KT;
                if (hs != HSP) { // (uniform) dims past the head size: zero, as q's are (0 x inf is not)
#pragma unroll
                    for (int u = 0; u < NU; u++)
#pragma unroll
                        for (int c = 0; c < KC; c++)
                            if ((T == PA_S ? 16 : 32) * c + dk >= hs) x.k[u][c] = make_uint4(0, 0, 0, 0);
                }
                float4v s[RB][NU];
#pragma unroll
                for (int b = 0; b < RB; b++)
#pragma unroll
                    for (int u = 0; u < NU; u++) s[b][u] = float4v{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < NU; u++)
#pragma unroll
                    for (int c = 0; c < KC; c++) {
                        // (all reads of the queries at once would spill 74 registers)
                        if (RB > 1 && HSP == 128 && c) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int b = 0; b < RB; b++) {
                            if constexpr (T == PA_S) {
                                const float4v kf = __builtin_bit_cast(float4v, x.k[u][c]);
                                float4v q;
                                if constexpr (RB == 1) q = qf[c];
                                else q = *(const float4v *)&og[0][n + 16 * b][16 * c + dk];
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    s[b][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], q[e], s[b][u], 0, 0, 0);
                            } else {
                                const half8v kh = __builtin_bit_cast(half8v, x.k[u][c]);
                                s[b][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[c], s[b][u], 0, 0, 0);
                                if constexpr (T == PA_M)
                                    s[b][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[c], s[b][u], 0, 0, 0);
                            }
                        }
                    }
                const bool bad0 = pg0 >= a.n_pages, bad1 = NU == 2 && pg1 >= a.n_pages;
                // the next tile's K (past the last: the last again, unused)
                load_k(kn, pn0, pn1);
                // (uniform) keys past a row's position, or on no page; keys before a row's window
                const bool past = (int32_t)(k0 + PAD_KT - 1) > t.p0 || bad0 || bad1;
                const bool behind = a.window && (int64_t)k0 <= (int64_t)t.plast - a.window;
#pragma unroll
                for (int b = 0; b < RB; b++)
#pragma unroll
                    for (int u = 0; u < NU; u++) s[b][u] *= rs;
                if (past) {
#pragma unroll
                    for (int u = 0; u < NU; u++) {
                        const bool gone = u ? bad1 : bad0;
                        const int32_t first = (int32_t)(k0 + 16 * u + 4 * g), thi = (gone ? -1 : t.plast) - first;
#pragma unroll
                        for (int b = 0; b < RB; b++) {
                            const int32_t hi = (gone ? -1 : qpos[b]) - first;
#pragma unroll
                            for (int e = 0; e < 4; e++) s[b][u][e] = e <= hi ? s[b][u][e] : -INFINITY;
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            // rows of V that are on no page or past the last position have no part in the sums,
                            // whatever was left in their memory
#pragma unroll
                            for (int z = 0; z < (int)(sizeof(x.v[0]) / 4); z++) x.v[4 * u + e][z] = e <= thi ? x.v[4 * u + e][z] : 0u;
                        }
                    }
                }
                if (behind) {
                    const int32_t sk = sinks - (int32_t)(k0 + 4 * g);
#pragma unroll
                    for (int b = 0; b < RB; b++) {
                        const int32_t lo = qlow[b] - (int32_t)(k0 + 4 * g);
#pragma unroll
                        for (int u = 0; u < NU; u++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                s[b][u][e] = (16 * u + e > lo) | (16 * u + e < sk) ? s[b][u][e] : -INFINITY;
                    }
                }
                float p[RB][4 * NU];
#pragma unroll
                for (int b = 0; b < RB; b++) {
                    float mt = -INFINITY;
#pragma unroll
                    for (int u = 0; u < NU; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) mt = fmaxf(mt, s[b][u][e]);
                    mt = pa_max4(mt);
                    // the reference moves only where a row's maximum passes it by more than 8: most tiles rescale nothing
                    if (__ballot(mt > m[b] + 8.0f)) {
                        const float mn = fmaxf(m[b], mt), al = mn == -INFINITY ? 0.0f : softmax_exp2(m[b] - mn);
                        m[b] = mn;
                        l[b] *= al;
#pragma unroll
                        for (int d = 0; d < DV; d++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[b][d][e] *= al;
                    }
                    const float mr = m[b] == -INFINITY ? 0.0f : m[b] - PA_UP;
#pragma unroll
                    for (int u = 0; u < NU; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            p[b][4 * u + e] = softmax_exp2(s[b][u][e] - mr);
                            l[b] += p[b][4 * u + e];
                        }
                }
                if constexpr (T == PA_S) {
#pragma unroll
                    for (int j = 0; j < 4 * NU; j++)
#pragma unroll
                        for (int d = 0; d < DV; d++)
#pragma unroll
                            for (int b = 0; b < RB; b++)
                                o[b][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.v[j][d]), p[b][j], o[b][d], 0, 0, 0);
                } else {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        if constexpr (T == PA_M) pa_split2(p[0][j], p[0][j + 1], hi[j / 2], lo[j / 2]);
                        else hi[j / 2] = pa_pack(p[0][j], p[0][j + 1]);
                    }
                    const half8v ph = __builtin_bit_cast(half8v, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                    half8v pl;
                    if constexpr (T == PA_M) pl = __builtin_bit_cast(half8v, make_uint4(lo[0], lo[1], lo[2], lo[3]));
#pragma unroll
                    for (int d = 0; d < DV; d++) {
                        // halves d of the eight rows' loads: the low or high half of word d / 2
                        uint4 w;
                        const uint32_t sel = (d & 1) ? 0x07060302u : 0x05040100u;
                        w.x = __builtin_amdgcn_perm(x.v[1][d / 2], x.v[0][d / 2], sel);
                        w.y = __builtin_amdgcn_perm(x.v[3][d / 2], x.v[2][d / 2], sel);
                        w.z = __builtin_amdgcn_perm(x.v[5][d / 2], x.v[4][d / 2], sel);
                        w.w = __builtin_amdgcn_perm(x.v[7][d / 2], x.v[6][d / 2], sel);
                        const half8v vt = __builtin_bit_cast(half8v, w);
                        o[0][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, ph, o[0][d], 0, 0, 0);
                        if constexpr (T == PA_M) o[0][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, pl, o[0][d], 0, 0, 0);
                    }
                }
                kt = kn;
                load_v(kt, pn0, pn1);
                pg0 = pn0;
                pg1 = pn1;
                kn = tile_of(min(i + 2 * PAD_WAVES, i1 - 1));
                pn0 = page_of(NU * kn);
                pn1 = page_of(NU * kn + 1);
            }
        // A weight of 0 times an infinity or NaN in a row of V that a query does not see is NaN (and the two parts
        // of a weight may make one of an infinity): where a sum is not finite though its weights are, the wave does
        // its keys again, one by one on the vector units, each row with those that it sees.
#pragma unroll
        for (int b = 0; b < RB; b++) {
            l[b] = pa_sum4(l[b]);
            bool odd = false;
#pragma unroll
            for (int d = 0; d < DV; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) odd |= pa_odd(o[b][d][e]);
            if (__ballot(odd && row_ok[b] && !pa_odd(l[b]))) {
#pragma unroll
                for (int d = 0; d < DV; d++) o[b][d] = float4v{0, 0, 0, 0};
                m[b] = -INFINITY;
                l[b] = 0.0f;
                for (uint32_t i = i0 + wave; i < i1; i += PAD_WAVES)
                    for (uint32_t z = 0; z < PAD_KT; z++) {
                        const uint32_t key = tile_of(i) * PAD_KT + z, page = page_of(key / 16);
                        if (page >= a.n_pages || (int32_t)key > t.plast) continue;
                        const size_t koff = (size_t)((int64_t)page * a.page_stride + (int64_t)(key & pm) * a.row_stride + (int64_t)kvh * a.head_stride);
                        float d4 = 0.0f;
                        for (uint32_t d = 4 * DV * g; d < min(4 * DV * (g + 1), hs); d++)
                            d4 = fmaf(pa_at<T != PA_H>(a.q, (size_t)gq[b] * a.ld_q + (size_t)head[b] * hs + d), pa_at<T == PA_S>(a.key, koff + d), d4);
                        const float s1 = pa_sum4(d4) * a.scale2;
                        if (!((int32_t)key <= qpos[b] & ((int32_t)key > qlow[b] | (int32_t)key < sinks))) continue;
                        const float mn = fmaxf(m[b], s1), mr = mn == -INFINITY ? 0.0f : mn;
                        const float al = m[b] == -INFINITY ? 0.0f : softmax_exp2(m[b] - mr), p = softmax_exp2(s1 - mr + PA_UP);
                        m[b] = mn;
                        // (0 x inf: a sum that was infinite stays so, or was NaN)
                        l[b] = l[b] * al + p;
#pragma unroll
                        for (int e = 0; e < 4; e++)
#pragma unroll
                            for (int d = 0; d < DV; d++) {
                                const uint32_t dim = DV * (4 * g + e) + d;
                                o[b][d][e] = (al == 0.0f ? 0.0f : o[b][d][e] * al) + p * pa_at<T == PA_S>(a.value, koff + min(dim, hs - 1));
                            }
                    }
            }
        }

        // the waves' states through LDS
        if constexpr (RB > 1) __syncthreads(); // (over the queries)
#pragma unroll
        for (int b = 0; b < RB; b++) {
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int d = 0; d < DV; d++) og[wave][n + 16 * b][DV * (4 * g + e) + d] = o[b][d][e];
            if (g == 0) {
                mg[wave][n + 16 * b] = m[b];
                lg[wave][n + 16 * b] = l[b];
            }
        }
        __syncthreads();
        const uint32_t rows = t.nq * heads, quads = hs / 4;
        for (uint32_t it = tid; it < rows * quads; it += 64 * PAD_WAVES) {
            const uint32_t rr = it / quads, d = 4 * (it % quads);
            float M = -INFINITY, L = 0.0f, O[4] = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < PAD_WAVES; w++) M = fmaxf(M, mg[w][rr]);
            const float mr = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < PAD_WAVES; w++) {
                const float wt = softmax_exp2(mg[w][rr] - mr);
                const float4 y = *(const float4 *)&og[w][rr][d];
                L = fmaf(lg[w][rr], wt, L);
                O[0] = fmaf(y.x, wt, O[0]);
                O[1] = fmaf(y.y, wt, O[1]);
                O[2] = fmaf(y.z, wt, O[2]);
                O[3] = fmaf(y.w, wt, O[3]);
            }
            const size_t orow = t.row0 + rr / heads, ohead = kvh * a.G + sub * a.heads_per + rr % heads;
            if (one) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                char *dst = (char *)a.out + (orow * a.ld_out + ohead * hs + d) * (T == PA_H ? 2 : 4);
                // a row that saw nothing has O = 0
                const float y[4] = {O[0] * inv, O[1] * inv, O[2] * inv, O[3] * inv};
                if constexpr (T == PA_H)
                    *(uint2 *)dst = make_uint2((uint32_t)f32_to_f16(y[0]) | (uint32_t)f32_to_f16(y[1]) << 16,
                                               (uint32_t)f32_to_f16(y[2]) | (uint32_t)f32_to_f16(y[3]) << 16);
                else *(float4 *)dst = make_float4(y[0], y[1], y[2], y[3]);
            } else {
                const size_t at = (orow * ((size_t)a.n_kv * a.G) + ohead) * a.n_splits + split;
                *(float4 *)(a.part_o + at * hs + d) = make_float4(O[0], O[1], O[2], O[3]);
                if (d == 0) *(float2 *)(a.part_ml + at * 2) = make_float2(M, L);
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------ tile kernel --
// Chunks: a workgroup of four waves per (tile, KV head, split), 32 of the
// tile's (query, head) rows per wave, one per lane pair (lanes l and l + 32).
// Per key tile of 64 rows, staged in LDS (two buffers of K and of V):
//   S^T = K Q^T      (Q^T stays in registers; v_mfma_f32_32x32x16_f16)
//   running softmax per row in registers: a lane holds 16 of its row's 32
//   scores per 32-key block
//   O^T += V^T P^T   with P^T straight from the score accumulator: the product
//   runs over the keys in the order the accumulator holds them
// K and V go from the cache straight into LDS (no registers in between), as
// rows of the tile whose 16-byte chunks are exchanged by an exclusive or with
// the row, so that the operand reads fall on distinct banks; V^T's operands
// are read with the transposing LDS load (lane i of 16 gets column i of four
// rows of 16).  Wave w brings the tile's rows 16w .. 16w + 15, which lie on
// one page.  Bound by the operand reads from LDS (128 KB a key tile and
// workgroup, 1024 cycles, as long as its products), the softmax beside them
// and power: 5720 rows of nine requests over 306 to 8000, 32 heads of 128, 492
// GFLOP in 504 us, 0.98 PFLOP/s with the matrix pipes 42-47% busy (a library's
// f16 product of 8192^3: 1.14).  Scores one key tile ahead of the softmax, in
// three forms, measured 1 to 4% slower (the clock falls from 2.0 to 1.7 GHz);
// one buffer of V and three workgroups a CU 592 us.  f32 rows, whose products
// are done twice and whose weights are split on the vector units: 517 over 1021,
// 32 heads of 64, 23 us, and the merge 8.
constexpr int PAT_WAVES = 4, PAT_KT = 64;

template <int HSP, int T>
__device__ void pa_tile_body(const PagedAttnArgs &a) {
    constexpr int KC = HSP / 16, DT = HSP / 32, KB = PAT_KT / 32;
    constexpr uint32_t RB = 2 * HSP, TB = PAT_KT * RB, CPR = HSP / 8; // bytes of a row and a tile; 16-byte chunks of a row
    constexpr uint32_t LPI = 1024 / RB;                                 // rows one load instruction brings
    __shared__ __attribute__((aligned(1024))) char ks[2 * TB], vs[2 * TB];
    // 16-row blocks of a tile that are on no page, a bit each: tile i's word is
    // i % 3, set while i - 1 is worked on, cleared while i + 1 is, a barrier from either
    __shared__ uint32_t s_flags[3];
    const uint32_t tid = threadIdx.x, lane = tid & 63, li = lane & 31, hl = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t kvh = blockIdx.x % a.n_kv, split = blockIdx.y;
    uint32_t r, q0, row0, nrows, kv;
    if (!pa_find(a, a.sorted, blockIdx.x / a.n_kv, r, q0)) return;
    pa_request_uniform(a, r, row0, nrows, kv);
    const PaTile t = pa_tile(a, r, row0, nrows, kv, q0);
    const PaKeys keys = pa_keys<PAT_KT>(a, t);
    const uint32_t C = pa_chunk(a, keys.n), i0 = split * C, i1 = min(i0 + C, keys.n);
    const bool one = keys.n <= C;
    if (i0 >= i1 && !(one && split == 0)) return;
    const uint32_t hs = a.hs, G = a.G, pm = (1u << a.lp) - 1;
    const uint32_t rr = wave * 32 + li, qi = rr / G, head = kvh * G + rr % G;
    const bool row_ok = qi < t.nq;
    // a row sees the keys k <= qpos with k > qlow or k < sinks
    const int32_t qpos = row_ok ? t.p0 + (int32_t)qi : -1, sinks = (int32_t)a.sinks;
    const int32_t qlow = a.window ? qpos - (int32_t)a.window : -1;
    const size_t gq = t.row0 + (row_ok ? qi : 0);
    const uint32_t *tab = a.table + (size_t)r * a.max_pages;

    // Chunk c of row y of a tile lies at chunk c ^ kx(y) (V: vx(y)) of the row.
    // K's operand reads take the same chunk of 16 consecutive rows, V's four
    // chunks (64 bytes) of four rows.
    auto kx = [](uint32_t y) { return HSP == 128 ? y & 15 : (y >> 1) & 7; };
    auto vx = [](uint32_t y) { return HSP == 128 ? 4 * (y & 3) : 4 * ((y >> 1) & 1); };
    auto tile_of = [&](uint32_t i) {
        i = min(i, i1 - 1);
        return i < keys.ns ? i : keys.lo + i - keys.ns;
    };
    // the page of this wave's rows of tile kt
    auto page_of = [&](uint32_t kt) {
        return pa_entry(tab, min((kt * 4 + wave) >> (a.lp - 4), a.max_pages - 1));
    };
    // this lane's bytes of a load instruction, from its 16 rows' first (chunks past the head size: the last one,
    // which meets q's zeros or outputs that nobody stores)
    uint32_t k_off[16 / LPI], v_off[16 / LPI];
#pragma unroll
    for (uint32_t i = 0; i < 16 / LPI; i++) {
        const uint32_t y = i * LPI + lane / CPR, c = lane % CPR;
        k_off[i] = 2 * (y * (uint32_t)a.row_stride + 8 * min(c ^ kx(y), hs / 8 - 1));
        v_off[i] = 2 * (y * (uint32_t)a.row_stride + 8 * min(c ^ vx(y), hs / 8 - 1));
    }
    // this wave's 16 rows of tile kt into buffer b
    const int64_t head_off = 2 * (int64_t)kvh * a.head_stride;
    auto bring = [&](uint32_t b, uint32_t kt, uint32_t page) {
        const int64_t off = 2 * ((int64_t)(page < a.n_pages ? page : 0u) * a.page_stride +
                                 (int64_t)((kt * PAT_KT + 16 * wave) & pm) * a.row_stride) + head_off;
        const char *pk = pa_scalar((const char *)a.key + off), *pv = pa_scalar((const char *)a.value + off);
        const uint32_t lds = b * TB + 16 * wave * RB;
#pragma unroll
        for (uint32_t i = 0; i < 16 / LPI; i++) lds_dma16(pk, k_off[i], lds_addr(ks) + lds + i * 1024);
#pragma unroll
        for (uint32_t i = 0; i < 16 / LPI; i++) lds_dma16(pv, v_off[i], lds_addr(vs) + lds + i * 1024);
    };
    if (tid < 3) s_flags[tid] = 0;
    // The first tile on its way before the queries are read.  Tiles i and i + 1, and the latter's page:
    uint32_t flag = 0, kt = 0, kt1 = 0, pg = 0, pg1 = 0;
    if (i0 < i1) {
        kt = tile_of(i0);
        kt1 = tile_of(i0 + 1);
        pg = page_of(kt);
        pg1 = page_of(kt1);
        bring(0, kt, pg);
    }

    half8v qh[KC], ql[T == PA_M ? KC : 1];
    float rs = a.scale2;
    {
        const char *qp = (const char *)a.q + (gq * a.ld_q + (size_t)head * hs) * (T == PA_H ? 2 : 4);
        if constexpr (T == PA_H) {
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const uint32_t d = 16 * c + 8 * hl;
                const bool ok = row_ok && d < hs;
                uint4 x = *(const uint4 *)(qp + 2 * (ok ? d : 0));
                if (!ok) x = make_uint4(0, 0, 0, 0);
                qh[c] = __builtin_bit_cast(half8v, x);
            }
        } else {
            float x[KC][8], mx = 0.0f;
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const uint32_t d = 16 * c + 8 * hl;
                const bool ok = row_ok && d < hs;
                const float4 u = *(const float4 *)(qp + 4 * (ok ? d : 0)), w = *(const float4 *)(qp + 4 * (ok ? d : 0) + 16);
                const float y[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[c][e] = ok ? y[e] : 0.0f;
                    mx = fmaxf(mx, fabsf(x[c][e]));
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const int ex = pa_q_exponent(mx);
            rs = ldexpf(rs, -ex);
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    _Float16 hi, lo;
                    pa_split(ldexpf(x[c][e], ex), hi, lo);
                    qh[c][e] = hi;
                    ql[c][e] = lo;
                }
        }
    }

    uint32_t k_at[KC], v_at[DT]; // byte offsets of this lane's operands in a tile
#pragma unroll
    for (int c = 0; c < KC; c++) k_at[c] = li * RB + 16 * ((2 * c + hl) ^ kx(li));
    {
        const uint32_t y = (lane >> 2) & 3, col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
        for (int d = 0; d < DT; d++)
            v_at[d] = (4 * hl + y) * RB + 16 * ((4 * d + col / 8) ^ vx(4 * hl + y)) + 2 * (col % 8);
    }
    auto scores = [&](uint32_t b, float16v (&s)[KB]) {
#pragma unroll
        for (int u = 0; u < KB; u++)
#pragma unroll
            for (int e = 0; e < 16; e++) s[u][e] = 0.0f;
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int u = 0; u < KB; u++) {
                const half8v av = *(const half8v *)(ks + b * TB + 32 * u * RB + k_at[c]);
                s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, qh[c], s[u], 0, 0, 0);
                if constexpr (T == PA_M) s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, ql[c], s[u], 0, 0, 0);
            }
    };
    // V^T operand of 16 keys: block u, half cc, dims 32 d ..
    auto v_of = [&](uint32_t b, int u, int cc, int d) {
        typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) fp16x4 lds_fp16x4;
        const char *p = vs + b * TB + (32 * u + 16 * cc) * RB + v_at[d];
        const fp16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_fp16x4 *)(fp16x4 *)p);
        const fp16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_fp16x4 *)(fp16x4 *)(p + 8 * RB));
        return __builtin_bit_cast(half8v, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    float16v o[DT];
    float m, l;
    auto clear = [&]() {
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
    };
    clear();

    auto step = [&](uint32_t i, const uint32_t b) { // tile i, in buffer b
        float16v s[KB];
        const uint32_t k0 = kt * PAT_KT, nf = flag == 2 ? 0 : flag + 1;
        // (past the last tile: the last again, unused)
        bring(b ^ 1u, kt1, pg1);
        const uint32_t kt2 = tile_of(i + 2), pg2 = page_of(kt2);
        const uint32_t f = __builtin_amdgcn_readfirstlane(s_flags[flag]);
        if (pg1 >= a.n_pages && lane == 0) atomicOr(&s_flags[nf], 1u << wave);
        scores(b, s);
        // the operand reads run four ahead of the products that take them
        pa_interleave<4, KB * KC, T == PA_M ? 2 : 1, 1>();
        // (uniform) keys past a row's position, or on no page; keys before a row's window
        const bool past = f || (int32_t)(k0 + PAT_KT - 1) > t.p0;
        const bool behind = a.window && (int64_t)k0 <= (int64_t)t.plast - a.window;
        if (past) {
#pragma unroll
            for (int z = 0; z < 4; z++) { // 16 rows on one page
                const int32_t hi = (f >> z & 1u ? -1 : qpos) - (int32_t)(k0 + 16 * z + 4 * hl);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    s[z / 2][8 * (z % 2) + e] = 8 * (e / 4) + e % 4 <= hi ? s[z / 2][8 * (z % 2) + e] : -INFINITY;
            }
        }
        if (behind) {
            const int32_t lo = qlow - (int32_t)(k0 + 4 * hl), sk = sinks - (int32_t)(k0 + 4 * hl);
#pragma unroll
            for (int u = 0; u < KB; u++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int32_t at = 32 * u + 8 * (e / 4) + e % 4;
                    s[u][e] = (at > lo) | (at < sk) ? s[u][e] : -INFINITY;
                }
        }
        if (f || (int32_t)(k0 + PAT_KT - 1) > t.plast) {
            // rows of V that are on no page or past the tile's last position have no part in the sums, whatever
            // was left in their memory (the same in all waves)
            for (uint32_t z = tid; z < PAT_KT * CPR; z += 64 * PAT_WAVES) {
                const uint32_t at = z / CPR;
                if ((f >> (at / 16) & 1u) || (int32_t)(k0 + at) > t.plast)
                    *(uint4 *)(vs + b * TB + 16 * z) = make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
        }
        float mt = -INFINITY;
#pragma unroll
        for (int u = 0; u < KB; u++)
#pragma unroll
            for (int e = 0; e < 16; e++) mt = fmaxf(mt, s[u][e]);
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * rs;
        if (__ballot(mt > m + 8.0f)) {
            const float mn = fmaxf(m, mt), al = mn == -INFINITY ? 0.0f : softmax_exp2(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= al;
        }
        const float mr = m == -INFINITY ? 0.0f : m - PA_UP;
        half8v ph[KB][2], pl[T == PA_M ? KB : 1][2];
#pragma unroll
        for (int u = 0; u < KB; u++)
#pragma unroll
            for (int cc = 0; cc < 2; cc++) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float p0 = softmax_exp2(fmaf(s[u][8 * cc + e], rs, -mr)), p1 = softmax_exp2(fmaf(s[u][8 * cc + e + 1], rs, -mr));
                    if constexpr (T == PA_M) {
                        pa_split2(p0, p1, hi[e / 2], lo[e / 2]);
                        l += p0 + p1;
                    } else {
                        // summed as they are multiplied: rounded
                        hi[e / 2] = pa_pack(p0, p1);
                        l = pa_add2(hi[e / 2], l);
                    }
                }
                ph[u][cc] = __builtin_bit_cast(half8v, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                if constexpr (T == PA_M) pl[u][cc] = __builtin_bit_cast(half8v, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
#pragma unroll
        for (int u = 0; u < KB; u++)
#pragma unroll
            for (int cc = 0; cc < 2; cc++)
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const half8v av = v_of(b, u, cc, d);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, ph[u][cc], o[d], 0, 0, 0);
                    if constexpr (T == PA_M) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, pl[u][cc], o[d], 0, 0, 0);
                }
        pa_interleave<4, KB * 2 * DT, T == PA_M ? 2 : 1, 2>();
        if (tid == 0) s_flags[nf == 2 ? 0 : nf + 1] = 0;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the rows brought above
        __syncthreads();
        flag = nf;
        kt = kt1;
        kt1 = kt2;
        pg1 = pg2;
    };
    if (i0 < i1) {
        __syncthreads(); // the flags are cleared
        if (pg >= a.n_pages && lane == 0) atomicOr(&s_flags[0], 1u << wave);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        for (uint32_t i = i0; i < i1; i += 2) {
            step(i, 0);
            if (i + 1 < i1) step(i + 1, 1);
        }
    }
    // A weight of 0 times an infinity or NaN in a row of V that a query does not see is NaN (and the two parts of a
    // weight may make one of an infinity): where a sum is not finite though its weights are, the wave does its rows
    // again, key by key on the vector units, each row with the keys that it sees.
    l += __shfl_xor(l, 32, 64);
    bool odd = false;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) odd |= pa_odd(o[d][e]);
    if (__ballot(odd && row_ok && !pa_odd(l))) {
        clear();
        for (uint32_t i = i0; i < i1; i++)
            for (uint32_t z = 0; z < PAT_KT; z++) {
                const uint32_t key = tile_of(i) * PAT_KT + z;
                if ((int32_t)key > t.plast) break;
                const uint32_t page = __builtin_amdgcn_readfirstlane(tab[key >> a.lp]);
                if (page >= a.n_pages) continue;
                const size_t koff = (size_t)((int64_t)page * a.page_stride + (int64_t)(key & pm) * a.row_stride + (int64_t)kvh * a.head_stride);
                float d2 = 0.0f;
                for (uint32_t d = hl; d < hs; d += 2)
                    d2 = fmaf(pa_at<T == PA_M>(a.q, gq * a.ld_q + (size_t)head * hs + d), pa_at<false>(a.key, koff + d), d2);
                const float s1 = (d2 + __shfl_xor(d2, 32, 64)) * a.scale2;
                if (!((int32_t)key <= qpos & ((int32_t)key > qlow | (int32_t)key < sinks))) continue;
                const float mn = fmaxf(m, s1), mr = mn == -INFINITY ? 0.0f : mn;
                const float al = m == -INFINITY ? 0.0f : softmax_exp2(m - mr), p = softmax_exp2(s1 - mr + PA_UP);
                m = mn;
                l = l * al + p;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const uint32_t dim = 32 * d + 8 * (e / 4) + 4 * hl + e % 4;
                        o[d][e] = (al == 0.0f ? 0.0f : o[d][e] * al) + p * pa_at<false>(a.value, koff + min(dim, hs - 1));
                    }
            }
    }
    if (!row_ok) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const size_t at = (gq * ((size_t)a.n_kv * G) + head) * a.n_splits + split;
    const size_t off = gq * a.ld_out + (size_t)head * hs;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const uint32_t dim = 32 * d + 2 * e + 4 * hl;
            if (dim >= hs) continue;
            const float y[4] = {o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
            if (!one) *(float4 *)(a.part_o + at * hs + dim) = make_float4(y[0], y[1], y[2], y[3]);
            else if constexpr (T == PA_H)
                *(uint2 *)((uint16_t *)a.out + off + dim) =
                    make_uint2((uint32_t)f32_to_f16(y[0] * inv) | (uint32_t)f32_to_f16(y[1] * inv) << 16,
                               (uint32_t)f32_to_f16(y[2] * inv) | (uint32_t)f32_to_f16(y[3] * inv) << 16);
            else *(float4 *)((float *)a.out + off + dim) = make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        }
    if (!one && hl == 0) *(float2 *)(a.part_ml + at * 2) = make_float2(m, l);
}

// Joins the splits of tiles of the 16-row kernel (RPW 1) or of the tile
// kernel (KT 64, RPW 4): grid as its x, and per y four waves of RPW rows of the
// tile each.  A lane has the dims 2 lane, 2 lane + 1 (64 dims: one) of every
// row, and one split's (m, l) of 64 at a time; the rows' loads go out together.
// Bound by the latency of its chain (request, (m, l) with the first partials,
// output) and then by the partials' bytes.  Only splits that the tile has are
// read; a tile of one split is written already.  8 decodes in up to 24 splits:
// 4 us.  (A launch of its own: the kernel boundary orders the partials, and the
// one-sequence decode's merge by the last workgroup to arrive measured slower.)
template <int HSP, int T, int KT, int RPW>
__device__ void pa_merge_body(const PagedAttnArgs &a) {
    constexpr int E = HSP / 64, U = RPW == 1 ? 16 : 4; // U: partials of a row on their way
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t b = blockIdx.x;
    const uint32_t kvh = b % a.n_kv;
    b /= a.n_kv;
    const uint32_t sub = b % a.n_sub;
    b /= a.n_sub;
    const uint32_t hs = a.hs, heads = min(a.heads_per, a.G - sub * a.heads_per);
    uint32_t r = b, q0 = 0, row0, nrows, kv;
    if (a.search && !pa_find(a, false, b, r, q0)) return;
    pa_request_uniform(a, r, row0, nrows, kv);
    uint32_t last_keys;
    const uint32_t qend = a.search ? q0 + 1 : nrows, chunk = pa_request_chunk<KT>(a, r, row0, nrows, kv, last_keys);
    const uint32_t d = E * lane, dl = min(d, hs - E);
    for (; q0 < qend; q0 += a.QT) {
        const PaTile t = pa_tile(a, r, row0, nrows, kv, q0);
        const uint32_t n = pa_keys<KT>(a, t).n, C = a.search ? pa_chunk(a, n) : chunk;
        if (n <= C) continue;
        const uint32_t S = (n + C - 1) / C, rows = t.nq * heads;
        for (uint32_t first = RPW * (4 * blockIdx.y + wave); first < rows; first += RPW * 4 * gridDim.y) {
            size_t at[RPW];   // the row's first partial
            size_t out[RPW];
            float M[RPW], L[RPW], O[RPW][E];
#pragma unroll
            for (int k = 0; k < RPW; k++) {
                const uint32_t rr = min(first + k, rows - 1); // (past the last row: it again)
                const size_t orow = t.row0 + rr / heads, ohead = kvh * a.G + sub * a.heads_per + rr % heads;
                at[k] = (orow * ((size_t)a.n_kv * a.G) + ohead) * a.n_splits;
                out[k] = orow * a.ld_out + ohead * hs + d;
                M[k] = -INFINITY;
                L[k] = 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++) O[k][e] = 0.0f;
            }
            for (uint32_t s0 = 0; s0 < S; s0 += 64) {
                const uint32_t nb = min(S - s0, 64u);
                float2 ml[RPW];
                float v[RPW][U][E];
                auto load = [&](uint32_t s) { // (past the last: it again, unused)
#pragma unroll
                    for (int k = 0; k < RPW; k++)
#pragma unroll
                        for (int z = 0; z < U; z++) {
                            const float *p = a.part_o + (at[k] + s0 + min(s + z, nb - 1)) * hs + dl;
#pragma unroll
                            for (int e = 0; e < E; e++) v[k][z][e] = p[e];
                        }
                };
#pragma unroll
                for (int k = 0; k < RPW; k++) {
                    ml[k] = *(const float2 *)(a.part_ml + (at[k] + s0 + min(lane, nb - 1)) * 2);
                    if (lane >= nb) ml[k] = make_float2(-INFINITY, 0.0f);
                }
                load(0);
                float w[RPW]; // of this lane's split
#pragma unroll
                for (int k = 0; k < RPW; k++) {
                    const float mn = fmaxf(M[k], wave_max(ml[k].x)), mr = mn == -INFINITY ? 0.0f : mn;
                    const float sc = M[k] == -INFINITY ? 0.0f : softmax_exp2(M[k] - mr);
                    w[k] = softmax_exp2(ml[k].x - mr);
                    L[k] = L[k] * sc + wave_sum(w[k] * ml[k].y);
#pragma unroll
                    for (int e = 0; e < E; e++) O[k][e] *= sc;
                    M[k] = mn;
                }
                for (uint32_t s = 0; s < nb; s += U) {
                    float x[RPW][U][E];
#pragma unroll
                    for (int k = 0; k < RPW; k++)
#pragma unroll
                        for (int z = 0; z < U; z++)
#pragma unroll
                            for (int e = 0; e < E; e++) x[k][z][e] = v[k][z][e];
                    if (s + U < nb) load(s + U);
#pragma unroll
                    for (int z = 0; z < U; z++) {
                        if (s + z >= nb) break;
#pragma unroll
                        for (int k = 0; k < RPW; k++) {
                            const float wt = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w[k]), s + z));
#pragma unroll
                            for (int e = 0; e < E; e++) O[k][e] = fmaf(x[k][z][e], wt, O[k][e]);
                        }
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < RPW; k++) {
                if (first + k >= rows || d >= hs) continue;
                const float inv = L[k] == 0.0f ? 0.0f : 1.0f / L[k];
#pragma unroll
                for (int e = 0; e < E; e++) {
                    if constexpr (T == PA_H) ((uint16_t *)a.out)[out[k] + e] = f32_to_f16(O[k][e] * inv);
                    else ((float *)a.out)[out[k] + e] = O[k][e] * inv;
                }
            }
        }
    }
}

} // namespace ifr
