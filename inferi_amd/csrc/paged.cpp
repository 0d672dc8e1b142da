// Host side of the paged-cache operators (include/inferi_hip.h "several
// requests, a paged cache"): the checks of arguments, the launch shapes and
// the splits of the attention over the sequence.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "ctx.h"
#include "paged_args.h"

using namespace ifr;

namespace {

constexpr uint32_t MAX_CONTEXT = 1u << 30;          // max_pages * page_size, as max_pos
constexpr uint64_t PART_BYTES_MAX = 512ull << 20;   // partials of one attention call
constexpr uint64_t MAX_GRID = 1ull << 24;           // workgroups of 256 threads a launch takes

// How the attention splits a call's keys over workgroups (measured on 256 CUs, times in
// us): of `base` tiles over up to n key tiles each, the key tiles of a part.

// Tiles of 16 rows, n key tiles of 32; four waves take turns at them. A part costs a
// workgroup's fixed 5 us, its partials and the second launch 4 more, so up to 16 stay
// whole (one decode at 300 keys 6.2, in two 9.1). From half as many tiles as CUs the
// memory is busy with 32 each (16 / 32 / 64 decodes of 1000, 32 heads over 8 of 128:
// 16.5 / 29.5 / 53.9, in parts of 8 19.2 / 38.6 / 62.8); fewer tiles take parts down to
// 8 (8 decodes of 300 to 1000 keys of an f32 cache 13.6, of 4 16.1, of 16 15.6), as many
// as there are places for (two a CU: one over 16000 keys 19 to 21, in more 30; two over
// 64000 108, in 784 parts 117, in 1008 119). Beyond 64 the longest sequences remain
// alone at the end (64 decodes at 200 to 8192 126, parts of 32 140, of 128 131).
uint64_t split16(uint64_t base, uint64_t n, uint32_t n_cu) {
    if (n <= 16) return n;
    const uint64_t places = 2 * n_cu;
    return std::max<uint64_t>(2 * base >= n_cu ? 32 : 8, std::min<uint64_t>(64, (n * base + places - 1) / places));
}

// Tiles of 128 rows, n key tiles of 64. A key tile takes a workgroup 1.15 us alone on its
// CU, two that share one 1.4 times as long; the join takes 8 us and 10 ns a workgroup for
// its partials of 128. The number of parts that costs least by that, of those that all have
// places (`base` counts up to a tile a request too many). As chosen / another, us: 1024
// rows of 32 heads of 128 over 4096, window 1024, 1 part 30 / 2 parts 43; 512 over 2000
// 4 parts 41 / 1 part 54; 512 over 30000 4 parts 276 / 1 part 562; 2048 of 12 heads over
// 4096 2 parts 95 / 1 part 117; 517 of 32 heads of 64 over 1021, f32 over f16, 4 parts 32
// / 5 parts, not all with places, 34. Parts for 512 workgroups whatever n: 1024 rows over
// none 36 (1 part: 27). At most 512 key tiles, whatever that costs: 9 requests of 1 to
// 512 rows over 0 to 120000 keys 1497, 1024 1655, no bound 2229.
uint64_t split128(uint64_t base, uint64_t n, uint32_t hs, uint32_t n_cu) {
    uint64_t best = n;
    double least = 0.0;
    for (uint64_t parts = 1; parts <= n; parts++) {
        const uint64_t chunk = (n + parts - 1) / parts, groups = base * parts;
        if (parts > 1 && (chunk < 4 || 8 * groups > 17 * n_cu)) break;
        const double cus = (double)groups / n_cu; // workgroups a CU
        const double step = cus <= 1.0 ? 1.0 : cus <= 2.0 ? 1.0 + 0.4 * (cus - 1.0) : 1.4 * cus / 2.0;
        const double us = 1.15 * step * (double)chunk + (parts > 1 ? 8.0 + 0.01 * (double)groups * hs / 128 : 0.0);
        if (parts == 1 || us < least) {
            least = us;
            best = chunk;
        }
    }
    return std::min<uint64_t>(best, 512);
}

uint32_t log2_of(uint32_t v) { return 31u - (uint32_t)__builtin_clz(v); }
bool pow2(uint32_t v) { return v && !(v & (v - 1)); }

// Makes the context's device current for a call that may allocate or launch,
// and the caller's again at its end.
struct DeviceGuard {
    int before = -1;
    explicit DeviceGuard(int device) {
        int now = 0;
        if (hipGetDevice(&now) == hipSuccess && now != device && hipSetDevice(device) == hipSuccess) before = now;
    }
    ~DeviceGuard() {
        if (before >= 0) hipSetDevice(before);
    }
};

ifr_status check_pages(ifr_ctx *c, const char *who, uint32_t page_size, uint32_t n_pages, uint32_t max_pages) {
    if (!pow2(page_size) || page_size < 16 || page_size > MAX_CONTEXT)
        return c->fail(IFR_EINVAL, "%s: page_size %u (a power of two from 16)", who, page_size);
    if (!n_pages || n_pages == IFR_NO_PAGE) return c->fail(IFR_EINVAL, "%s: n_pages %u", who, n_pages);
    if (!max_pages || (uint64_t)max_pages * page_size > MAX_CONTEXT)
        return c->fail(IFR_EINVAL, "%s: max_pages %u of %u rows (at most 2^30 rows)", who, max_pages, page_size);
    return IFR_OK;
}

// The cache's arguments, with the dense strides filled in.
ifr_status check_cache(ifr_ctx *c, const char *who, ifr_paged_cache &k) {
    if (!k.key || !k.value) return c->fail(IFR_EINVAL, "%s: null cache", who);
    if (k.dtype != IFR_F16 && k.dtype != IFR_F32) return c->fail(IFR_EINVAL, "%s: cache dtype F16 or F32", who);
    if (ifr_status st = check_pages(c, who, k.page_size, k.n_pages, k.max_pages)) return st;
    if (!k.head_size || k.head_size % 8 || k.head_size > 128)
        return c->fail(IFR_EUNSUPPORTED, "%s: head_size %u (a multiple of 8, at most 128)", who, k.head_size);
    if (!k.n_kv_heads || k.n_kv_heads > 65535) return c->fail(IFR_EINVAL, "%s: n_kv_heads %u", who, k.n_kv_heads);
    const int64_t unit = k.dtype == IFR_F16 ? 8 : 4, most = 1 << 25;
    if (!k.head_stride) k.head_stride = k.head_size;
    if (!k.row_stride) k.row_stride = (int64_t)k.n_kv_heads * k.head_size;
    if (!k.page_stride) k.page_stride = (int64_t)k.page_size * k.row_stride;
    if (k.head_stride < 0 || k.row_stride < 0 || k.page_stride < 0 || k.head_stride % unit || k.row_stride % unit ||
        k.page_stride % unit || k.row_stride > most || k.page_stride > (1ll << 56) / std::max<int64_t>(k.n_pages, 1) ||
        k.head_stride > (1ll << 56) / k.n_kv_heads)
        return c->fail(IFR_EINVAL, "%s: cache strides (whole 16 bytes, rows at most 2^25 elements apart)", who);
    if ((uintptr_t)k.key % 16 || (uintptr_t)k.value % 16) return c->fail(IFR_EINVAL, "%s: cache not 16-byte aligned", who);
    return IFR_OK;
}

// One kernel of the attention and, where its tiles' keys go to several
// workgroups, the kernel that joins them.  tiles: at most; key_rows: of a key
// tile; least, most: key tiles of a split (more only where a tile has more than
// `most` of them for all its splits); want: workgroups that fill the chip.
ifr_status launch_attention(ifr_ctx *c, PagedAttnArgs &a, const char *name, const char *merge, uint64_t tiles,
                            uint32_t key_rows, uint32_t max_kv) {
    const uint64_t base = tiles * a.n_sub * a.n_kv;
    if (!base) return IFR_OK;
    if (base >= MAX_GRID) return c->fail(IFR_EUNSUPPORTED, "paged_attention: %llu workgroups", (unsigned long long)base);
    uint64_t keys = max_kv; // rows that a tile reads, at most
    if (a.window) keys = std::min<uint64_t>(keys, (uint64_t)a.window + a.sinks + a.QT + 2 * key_rows);
    const uint64_t key_tiles = (keys + key_rows - 1) / key_rows;
    const uint64_t heads = (uint64_t)a.n_kv * a.G, row_bytes = (uint64_t)a.n_rows * heads * (a.hs + 2) * 4;
    // (key tiles of 16, of f32 rows of 128: as many keys)
    const uint64_t chunk = key_rows == 64   ? split128(base, key_tiles, a.hs, c->n_cu)
                           : key_rows == 32 ? split16(base, key_tiles, c->n_cu)
                                            : 2 * split16(base, (key_tiles + 1) / 2, c->n_cu);
    uint64_t splits = std::max<uint64_t>(1, std::min((key_tiles + chunk - 1) / chunk, PART_BYTES_MAX / row_bytes));
    splits = std::min(splits, (MAX_GRID - 1) / base);
    a.chunk = (uint32_t)chunk;
    a.n_splits = (uint32_t)splits;
    if (splits > 1) {
        if (ifr_status st = c->ensure_scratch(row_bytes * splits)) return st;
        a.part_o = (float *)c->scratch;
        a.part_ml = a.part_o + (uint64_t)a.n_rows * heads * splits * a.hs;
    }
    a.sorted = a.n_requests > 1 && a.n_requests <= 64 && base * splits > (uint32_t)c->n_cu;
    // (without a search a workgroup finds its split with its request)
    const dim3 grid = a.search ? dim3((uint32_t)base, a.n_splits) : dim3((uint32_t)(base * splits));
    ifr_status st = c->launch(name, grid, dim3(256), 0, a);
    if (st || splits == 1) return st;
    // four waves a workgroup, of one row of a tile each (of four for the larger tiles)
    const uint32_t rows = key_rows == 64 ? 16 : 4;
    return c->launch(merge, dim3((uint32_t)base, (a.QT * a.heads_per + rows - 1) / rows), dim3(256), 0, a);
}

bool bad_ld(int64_t ld, int64_t least, int64_t unit) { return ld < least || ld % unit || ld > (1ll << 40); }

} // namespace

extern "C" {

IFR_API ifr_status ifr_paged_plan(ifr_ctx *c, const ifr_paged_plan_args *p) {
    if (!c) return IFR_EINVAL;
    if (!p) return c->fail(IFR_EINVAL, "paged_plan: null arguments");
    if (ifr_status st = check_pages(c, "paged_plan", p->page_size, p->n_pages, p->max_pages)) return st;
    if (!p->free_count || !p->free_count_out || !p->free_pages || !p->row_start)
        return c->fail(IFR_EINVAL, "paged_plan: null pointer");
    if (p->n_requests && (!p->ctx_len || !p->new_len || !p->block_table || !p->kv_len))
        return c->fail(IFR_EINVAL, "paged_plan: null pointer");
    if (p->n_rows && (!p->positions || !p->slots)) return c->fail(IFR_EINVAL, "paged_plan: null pointer");
    if (p->n_rows > MAX_CONTEXT || p->n_requests > MAX_CONTEXT)
        return c->fail(IFR_EINVAL, "paged_plan: %u rows of %u requests", p->n_rows, p->n_requests);
    if ((uint64_t)std::min(p->n_requests, PG_PLAN_THREADS) * p->max_pages >= (1ull << 31))
        return c->fail(IFR_EINVAL, "paged_plan: a table of %u x %u entries", p->n_requests, p->max_pages);
    DeviceGuard dev(c->device);
    PagedPlanArgs a{};
    a.ctx_len = p->ctx_len;
    a.new_len = p->new_len;
    a.free_pages = p->free_pages;
    a.free_count = p->free_count;
    a.free_count_out = p->free_count_out;
    a.table = p->block_table;
    a.ctx_len_out = p->ctx_len_out;
    a.row_start = p->row_start;
    a.kv_len = p->kv_len;
    a.positions = p->positions;
    a.slots = p->slots;
    a.n_requests = p->n_requests;
    a.n_rows = p->n_rows;
    a.n_pages = p->n_pages;
    a.lp = log2_of(p->page_size);
    a.max_pages = p->max_pages;
    // (us by the plan's workgroup / by a second launch: 2048 rows 4.8 / 6.9, 3074 6.0 / 7.0, 4611 6.9 / 7.0, 7170 8.6 / 7.2)
    a.rows_here = p->n_rows <= 4096 || !p->n_requests;
    if (!a.rows_here) {
        if (ifr_status st = c->ensure_scratch(((size_t)p->n_requests + 1) * 4)) return st;
        a.pops = (uint32_t *)c->scratch;
    }
    const uint32_t widest = std::max(p->n_requests, a.rows_here ? p->n_rows : 0u);
    const uint32_t threads = widest <= 64 ? 64 : widest <= 256 ? 256 : PG_PLAN_THREADS;
    ifr_status st = c->launch("paged_plan_k", dim3(1), dim3(threads), 0, a);
    if (st || a.rows_here) return st;
    return c->launch("paged_rows_k", dim3((p->n_rows + 511) / 512), dim3(256), 0, a);
}

IFR_API ifr_status ifr_paged_rope_store(ifr_ctx *c, const ifr_paged_cache *cache, const ifr_paged_rope_args *p) {
    if (!c) return IFR_EINVAL;
    if (!cache || !p) return c->fail(IFR_EINVAL, "paged_rope_store: null arguments");
    ifr_paged_cache k = *cache;
    k.max_pages = 1; // the table is not read
    if (ifr_status st = check_cache(c, "paged_rope_store", k)) return st;
    if (!p->n_rows) return IFR_OK;
    const uint32_t hs = k.head_size;
    if (p->variant != IFR_ROPE_ORIGINAL && p->variant != IFR_ROPE_NEOX)
        return c->fail(IFR_EINVAL, "paged_rope_store: bad variant");
    if (!(p->base_freq >= 0.0f) || std::isinf(p->base_freq))
        return c->fail(IFR_EINVAL, "paged_rope_store: base_freq (0, or positive and finite)");
    if (!p->k || !p->v || !p->positions || !p->slots) return c->fail(IFR_EINVAL, "paged_rope_store: null pointer");
    if (!p->q != !p->q_out) return c->fail(IFR_EINVAL, "paged_rope_store: q and q_out, or neither");
    if (p->q && (!p->n_heads || p->n_heads > 65535)) return c->fail(IFR_EINVAL, "paged_rope_store: n_heads %u", p->n_heads);
    if (p->q && p->q_dtype != IFR_F16 && p->q_dtype != IFR_F32)
        return c->fail(IFR_EINVAL, "paged_rope_store: q_dtype F16 or F32");
    if (p->n_rows > MAX_CONTEXT) return c->fail(IFR_EINVAL, "paged_rope_store: n_rows %u", p->n_rows);
    const int64_t qd = (int64_t)p->n_heads * hs, kd = (int64_t)k.n_kv_heads * hs;
    PagedRopeArgs a{};
    a.ld_q = p->ld_q ? p->ld_q : qd;
    a.ld_k = p->ld_k ? p->ld_k : kd;
    a.ld_v = p->ld_v ? p->ld_v : kd;
    a.ld_q_out = p->ld_q_out ? p->ld_q_out : qd;
    if ((p->q && (bad_ld(a.ld_q, qd, 4) || bad_ld(a.ld_q_out, qd, 8))) || bad_ld(a.ld_k, kd, 4) || bad_ld(a.ld_v, kd, 4))
        return c->fail(IFR_EINVAL, "paged_rope_store: leading dimensions");
    if ((uintptr_t)p->q % 16 || (uintptr_t)p->k % 16 || (uintptr_t)p->v % 16 || (uintptr_t)p->q_out % 16)
        return c->fail(IFR_EINVAL, "paged_rope_store: rows must be 16-byte aligned");
    if (p->q && (const void *)p->q == p->q_out && (p->q_dtype != IFR_F32 || a.ld_q != a.ld_q_out))
        return c->fail(IFR_EINVAL, "paged_rope_store: q_out may be q only in f32 with its ld");
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.positions = p->positions;
    a.slots = p->slots;
    a.q_out = p->q_out;
    a.key = k.key;
    a.value = k.value;
    a.page_stride = k.page_stride;
    a.row_stride = k.row_stride;
    a.head_stride = k.head_stride;
    a.turn = p->base_freq > 0.0f;
    a.log2_base = a.turn ? std::log2((double)p->base_freq) : 0.0;
    a.n_rows = p->n_rows;
    a.n_heads = p->n_heads;
    a.n_kv = k.n_kv_heads;
    a.hs = hs;
    a.n_pages = k.n_pages;
    a.lp = log2_of(k.page_size);
    a.neox = p->variant == IFR_ROPE_NEOX;
    a.q_f16 = p->q_dtype == IFR_F16;
    a.kv_f16 = k.dtype == IFR_F16;
    // a workgroup a row, or several that share it while that leaves CUs without one
    const uint32_t items = ((p->q ? p->n_heads : 0) + 2 * k.n_kv_heads) * (hs / 8);
    a.parts = std::max(1u, std::min((items + PG_ROPE_THREADS - 1) / PG_ROPE_THREADS, (uint32_t)c->n_cu * 2 / p->n_rows));
    if (p->n_rows >= MAX_GRID) return c->fail(IFR_EUNSUPPORTED, "paged_rope_store: %u rows", p->n_rows);
    DeviceGuard dev(c->device);
    return c->launch("paged_rope_k", dim3(p->n_rows, a.parts), dim3(PG_ROPE_THREADS), 0, a);
}

IFR_API ifr_status ifr_paged_attention(ifr_ctx *c, const ifr_paged_cache *cache, const ifr_paged_attn_args *p) {
    if (!c) return IFR_EINVAL;
    if (!cache || !p) return c->fail(IFR_EINVAL, "paged_attention: null arguments");
    ifr_paged_cache k = *cache;
    if (ifr_status st = check_cache(c, "paged_attention", k)) return st;
    if (!p->n_requests || !p->n_rows) return IFR_OK;
    const uint32_t hs = k.head_size;
    if (!k.block_table || !p->row_start || !p->kv_len || !p->q || !p->out)
        return c->fail(IFR_EINVAL, "paged_attention: null pointer");
    if (!p->n_heads || p->n_heads > 65535 || p->n_heads % k.n_kv_heads)
        return c->fail(IFR_EINVAL, "paged_attention: %u heads over %u KV heads", p->n_heads, k.n_kv_heads);
    if (p->q_dtype != IFR_F16 && p->q_dtype != IFR_F32)
        return c->fail(IFR_EINVAL, "paged_attention: q_dtype F16 or F32");
    if (p->q_dtype == IFR_F16 && k.dtype == IFR_F32)
        return c->fail(IFR_EUNSUPPORTED, "paged_attention: f16 queries over an f32 cache");
    if (p->n_rows > MAX_CONTEXT || p->n_requests > MAX_CONTEXT)
        return c->fail(IFR_EINVAL, "paged_attention: %u rows of %u requests", p->n_rows, p->n_requests);
    if (!(p->scale == 0.0f || (p->scale >= 0x1p-60f && p->scale <= 0x1p14f)))
        return c->fail(IFR_EINVAL, "paged_attention: scale (0, or 2^-60 to 2^14)");
    const int64_t qd = (int64_t)p->n_heads * hs;
    PagedAttnArgs a{};
    a.ld_q = p->ld_q ? p->ld_q : qd;
    a.ld_out = p->ld_out ? p->ld_out : qd;
    if (bad_ld(a.ld_q, qd, 8) || bad_ld(a.ld_out, qd, 8)) return c->fail(IFR_EINVAL, "paged_attention: ld_q, ld_out");
    if ((uintptr_t)p->q % 16 || (uintptr_t)p->out % 16)
        return c->fail(IFR_EINVAL, "paged_attention: q and out must be 16-byte aligned");
    if (p->q == p->out && a.ld_q != a.ld_out) return c->fail(IFR_EINVAL, "paged_attention: out may be q only with its ld");
    const uint32_t cap = k.max_pages * k.page_size;
    a.q = p->q;
    a.out = p->out;
    a.key = k.key;
    a.value = k.value;
    a.table = k.block_table;
    a.row_start = p->row_start;
    a.kv_len = p->kv_len;
    a.page_stride = k.page_stride;
    a.row_stride = k.row_stride;
    a.head_stride = k.head_stride;
    a.n_pages = k.n_pages;
    a.lp = log2_of(k.page_size);
    a.max_pages = k.max_pages;
    a.n_kv = k.n_kv_heads;
    a.hs = hs;
    a.G = p->n_heads / k.n_kv_heads;
    a.n_requests = p->n_requests;
    a.n_rows = p->n_rows;
    a.window = p->window >= cap ? 0 : p->window;
    a.sinks = a.window ? std::min(p->n_sinks, cap) : 0;
    const float scale = p->scale > 0.0f ? p->scale : 1.0f / std::sqrt((float)hs);
    a.scale2 = scale * 1.44269504088896341f;
    const char *type = p->q_dtype == IFR_F16 ? "f16" : k.dtype == IFR_F16 ? "mixed" : "f32";
    const uint32_t hsp = hs <= 64 ? 64 : 128;
    const uint32_t max_new = p->max_new ? std::min(p->max_new, p->n_rows) : p->n_rows;
    const uint32_t max_kv = p->max_kv ? std::min(p->max_kv, cap) : cap;

    // Steps of up to `few` new rows a request (two tiles of 16 (query, head) rows for
    // heads of 64 and less, one for larger ones) run in such tiles, longer ones, with the
    // decodes among them, in tiles of 128, which read K and V once for more rows. Two
    // tiles' worth, us in tiles of 16 and of 128: heads of 128, 16 requests over 2000
    // keys 48.8 / 40.9, 64 over 500 44.1 / 33.2, one over 30000 50 / 56; heads of 64, 64
    // over 1000 25.6 / 26.1 and, with f32 rows, 25.8 / 30.4. Three tiles' worth: 12 rows
    // of 4 requests over 9000 71.6 / 45.7. f32 caches, whose products run at a sixteenth of
    // the rate, run in tiles of 16 and, with more rows, of 32 (device/paged_attn.h); groups
    // of more than 64 heads (fewer than two rows of 128) always in tiles of 16.
    const uint32_t QT16 = std::max(16 / a.G, 1u), few = (hsp == 64 ? 2 : 1) * QT16;
    DeviceGuard dev(c->device);
    char name[64], merge[64];
    if (k.dtype == IFR_F32 || a.G > 64 || max_new <= few) {
        // a group of more than 16 heads is cut into sub-groups of 16
        a.heads_per = std::min(a.G, 16u);
        a.n_sub = (a.G + 15) / 16;
        a.search = max_new > QT16;
        const uint32_t rows = a.search && k.dtype == IFR_F32 ? 32 : 16;
        a.QT = std::max(rows / a.heads_per, 1u);
        const uint64_t tiles = a.search ? p->n_rows / a.QT + std::min(p->n_requests, p->n_rows) : p->n_requests;
        snprintf(name, sizeof name, "paged_rows%u_%s_h%u", rows, type, hsp);
        snprintf(merge, sizeof merge, "paged_merge16_%s_h%u", type, hsp);
        return launch_attention(c, a, name, merge, tiles, k.dtype == IFR_F32 && hsp == 128 ? 16 : 32, max_kv);
    }
    a.heads_per = a.G;
    a.n_sub = 1;
    a.QT = 128 / a.G;
    a.search = 1;
    const uint64_t tiles = p->n_rows / a.QT + std::min(p->n_requests, p->n_rows);
    snprintf(name, sizeof name, "paged_tile_%s_h%u", type, hsp);
    snprintf(merge, sizeof merge, "paged_merge128_%s_h%u", type, hsp);
    return launch_attention(c, a, name, merge, tiles, 64, max_kv);
}

} // extern "C"
