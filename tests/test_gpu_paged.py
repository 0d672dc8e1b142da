"""Paged-cache operators against their plain forms: the plan of a step's pages,
slots and positions, rotary embedding with the store, and attention.

Tolerances.  store: the angle's cos and sin are f32 values off by at most two
steps (2^-22 of 1) and each turned value is two products and a sum, so it is
within 2^-21 of |x0| + |x1| before its one rounding to the output's type.
attention, with f32 results (f16 or f32 cache): a score is a sum of hs
products; its error is at most hs * 2^-23 of sum |q_d k_d| scale (f32 sums) plus
2^-22 of the same (q in two halves of 22 bits), and an error e of the scores
moves a weight by a factor within e; the weights and the sum of them carry 2^-21
each and the sums of n weighted rows n * 2^-24 at the worst.  The bound taken is
(hs * 2^-23 + 2^-21) * max_j sum_d |q_d k_jd| * scale * 2 + n * 2^-24 + 2^-20, times max |v|.
attention with f16 results: the weights are rounded to f16, 2^-11 of each (2^-25 absolutely for
those below 2^-14 of the largest, at most n of them), so 2^-11 + n * 2^-25 of max |v| more, and the
result's own rounding, 2^-11 of it.
"""

import shutil

import numpy as np
import pytest

import inferi_amd as I
from tests.paged import NO, NP, Paged, attn_ref, plan_ref, rope_ref, run_plan

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ plan --

def _plan_case(rng, n, page, most, spare, release, n_rows=None, max_new=40, bad=False):
    ctx_len = [int(rng.integers(0, most * page)) if rng.random() < 0.8 else 0 for _ in range(n)]
    new_len = [int(min(rng.integers(0, max_new + 1), most * page - c)) for c in ctx_len]
    held = [-(-c // page) for c in ctx_len]
    need = sum(-(-(c + v) // page) - h for c, v, h in zip(ctx_len, new_len, held))
    n_pages = sum(held) + max(need + spare, 1)
    order = rng.permutation(n_pages).astype(np.uint32)
    table = np.full((n, most), NO, np.uint32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        at += h
    free = np.concatenate([order[at:], np.full(at, NO, np.uint32)])
    count = n_pages - at
    if release:
        for r in range(n):
            if rng.random() < release:
                new_len[r] = NO
    if bad and n > 1:
        table[0, 0] = n_pages
        table[1, :1] = NO
    rows = sum(v for v in new_len if v != NO)
    return ctx_len, new_len, free, count, table, page, n_pages, rows if n_rows is None else n_rows(rows)


@pytest.mark.parametrize("n,page,most,spare,release,bad", [
    (1, 16, 1, 0, 0.0, False), (1, 64, 40, 3, 0.0, False), (3, 16, 9, -2, 0.0, False), (32, 16, 30, 0, 0.0, False),
    (63, 32, 20, 5, 0.3, False), (64, 16, 12, -20, 0.3, False), (65, 16, 70, -3, 0.2, True), (257, 16, 8, 0, 0.1, False),
    (1023, 16, 9, 4, 0.05, True), (1024, 32, 5, -100, 0.2, False), (1025, 16, 5, 2, 0.1, False), (3000, 16, 4, -60, 0.4, True),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_against_plain(ctx, n, page, most, spare, release, bad, in_place):
    rng = np.random.default_rng(n * 7 + page + most)
    case = _plan_case(rng, n, page, most, spare, release, bad=bad)
    got, ref = run_plan(ctx, *case, in_place=in_place), plan_ref(*case)
    for k in ref:
        np.testing.assert_array_equal(got[k], ref[k], err_msg=k)


@pytest.mark.parametrize("n,rows", [(20, lambda r: r // 2), (20, lambda r: r + 700), (700, lambda r: r + 3000),
                                    (700, lambda r: r - 1), (40, lambda r: 0), (1500, lambda r: r // 3)])
def test_plan_rows_short_and_spare(ctx, n, rows):
    """Fewer rows than the requests bring (those past the end are refused), and more (they are no rows)."""
    case = _plan_case(np.random.default_rng(n), n, 16, 30, 10, 0.1, n_rows=rows, max_new=20)
    got, ref = run_plan(ctx, *case), plan_ref(*case)
    for k in ref:
        np.testing.assert_array_equal(got[k], ref[k], err_msg=k)


@pytest.mark.parametrize("n,page,spare,release", [(40, 16, 0, 0.0), (300, 64, -40, 0.1), (1100, 16, -900, 0.05), (2100, 32, 7, 0.2)])
def test_plan_of_many_rows(ctx, n, page, spare, release):
    """Steps whose rows are a launch of their own, some with too few pages for the last requests."""
    case = _plan_case(np.random.default_rng(n), n, page, 60, spare, release, max_new=600)
    assert case[-1] > 8192
    got, ref = run_plan(ctx, *case), plan_ref(*case)
    for k in ref:
        np.testing.assert_array_equal(got[k], ref[k], err_msg=k)


def test_plan_long_prompts_and_no_requests(ctx):
    page, most = 16, 4096
    free = np.random.default_rng(5).permutation(5000).astype(np.uint32)
    # 50,000 new rows of one request behind requests without rows; one longer than its table row holds
    case = ([3, 0, 0, 65000, 17], [0, 0, 50001, 600, 5000], free, 4800, np.full((5, most), NO, np.uint32), page, 5000, 55601)
    case[4][0, 0], case[4][4, :2] = 4999, (4998, 4997)
    got, ref = run_plan(ctx, *case), plan_ref(*case)
    for k in ref:
        np.testing.assert_array_equal(got[k], ref[k], err_msg=k)
    assert got["kv_len"].tolist() == [3, 0, 50001, 0, 5017]
    for rows in (0, 5, 3000):
        case = ([], [], free[:9], 4, np.zeros((0, 1), np.uint32), 16, 9, rows)
        got = run_plan(ctx, *case)
        assert got["row_start"].tolist() == [0] and got["free_count_out"].tolist() == [4]
        assert (got["positions"] == NO).all() and got["slots"].size == rows


def test_plan_values_past_32_bits(ctx):
    """Lengths whose sums pass 32 bits are refused, and the requests beside them are not."""
    page, most = 64, 4
    table = np.full((4, most), NO, np.uint32)
    case = ([0, 0xFFFFFFF0, 5, 0], [3, 0x40, 0xFFFFFFFE, 2], np.arange(9, dtype=np.uint32), 0xFFFFFFFF, table, page, 9, 40)
    got, ref = run_plan(ctx, *case), plan_ref(*case)
    assert got["kv_len"].tolist()[:3] == [3, 0, 0]
    for k in ref:
        np.testing.assert_array_equal(got[k], ref[k], err_msg=k)


# ----------------------------------------------------------------- store --

@pytest.mark.parametrize("hs,heads,kvh,neox,q_dtype,dtype,layout,rows", [
    (64, 14, 2, True, I.F16, I.F16, "dense", 1), (128, 32, 8, False, I.F16, I.F16, "dense", 33),
    (128, 12, 2, True, I.F32, I.F32, "gap", 7), (80, 5, 5, True, I.F32, I.F16, "heads", 19), (8, 3, 1, False, I.F16, I.F32, "gap", 5),
    (24, 2, 2, True, I.F16, I.F16, "gap", 64), (96, 6, 3, False, I.F32, I.F32, "heads", 11), (128, 8, 2, False, I.F16, I.F16, "gap", 1100),
    (104, 4, 1, True, I.F16, I.F16, "dense", 1027),
])
def test_rope_store_against_plain(ctx, hs, heads, kvh, neox, q_dtype, dtype, layout, rows):
    rng = np.random.default_rng(rows * hs)
    page, n_pages = 16, rows // 16 + 5
    cache = Paged(ctx, rng, dtype, n_pages, page, kvh, hs, layout, fill=0.25).upload()
    wide = (heads + 2 * kvh) * hs + 4
    x = rng.standard_normal((rows, wide)).astype(np.float32)
    pos = rng.integers(0, 200000, rows).astype(np.uint32)
    slots = rng.permutation(n_pages * page)[:rows].astype(np.uint64)
    if rows > 4:
        pos[2] = NO                       # not in the step
        slots[3] = I.NO_SLOT              # stores nothing
        slots[4] = n_pages * page         # past the cache
    ld_out = heads * hs + 8
    q_out = ctx.upload(np.full(rows * ld_out, 7, NP[q_dtype]))
    dx, dp, ds = ctx.upload(x), ctx.upload(pos), ctx.upload(slots)
    base = 500000.0
    ctx.paged_rope_store(cache.args(None, 1), I.PagedRope(
        n_rows=rows, n_heads=heads, variant=I.ROPE_NEOX if neox else I.ROPE_ORIGINAL, base_freq=base, q=dx.ptr,
        k=dx.ptr + 4 * heads * hs, v=dx.ptr + 4 * (heads + kvh) * hs, ld_q=wide, ld_k=wide, ld_v=wide,
        positions=dp.ptr, slots=ds.ptr, q_out=q_out.ptr, q_dtype=q_dtype, ld_q_out=ld_out))
    got = q_out.download(NP[q_dtype]).reshape(rows, ld_out)
    k, v = cache.dk.download(NP[dtype]), cache.dv.download(NP[dtype])
    y = x[:, :(heads + 2 * kvh) * hs].reshape(rows, heads + 2 * kvh, hs).astype(np.float64)
    turned = rope_ref(y[:, :heads + kvh], pos, base, neox)
    half = np.roll(np.abs(y[:, :heads + kvh]), hs // 2, -1) if neox else np.abs(y[:, :heads + kvh])[..., np.arange(hs) ^ 1]
    tol = (np.abs(y[:, :heads + kvh]) + half) * 2.0 ** -21
    step = lambda t: np.finfo(NP[t]).eps / 2  # noqa: E731
    live = pos != NO
    err = np.abs(got[:, :heads * hs].reshape(rows, heads, hs).astype(np.float64) - turned[:, :heads])
    assert (err <= tol[:, :heads] + step(q_dtype) * np.abs(turned[:, :heads]) + 1e-7)[live].all()
    assert (got[~live] == 7).all() and (got[:, heads * hs:] == 7).all()
    want_k, want_v, tol_k = (np.full(cache.k.size, 0.25) for _ in range(3))
    tol_k[:] = 0
    for i in range(rows):
        if live[i] and slots[i] < n_pages * page:
            at = cache.index(int(slots[i]) // page, int(slots[i]) % page)
            want_k[at], want_v[at] = turned[i, heads:], y[i, heads + kvh:].astype(NP[dtype])
            tol_k[at] = tol[i, heads:] + step(dtype) * np.abs(turned[i, heads:]) + 1e-7
    assert (np.abs(k - want_k) <= tol_k).all()
    np.testing.assert_array_equal(v, want_v.astype(NP[dtype]))
    for b in (q_out, dx, dp, ds):
        b.free()
    cache.free()


def test_rope_store_in_place_without_turn_and_without_q(ctx):
    rng = np.random.default_rng(3)
    rows, heads, kvh, hs = 9, 4, 2, 64
    cache = Paged(ctx, rng, I.F32, 2, 16, kvh, hs, fill=0.0).upload()
    q, k, v = (rng.standard_normal((rows, h, hs)).astype(np.float32) for h in (heads, kvh, kvh))
    dq, dk, dv = ctx.upload(q), ctx.upload(k), ctx.upload(v)
    pos, slots = ctx.upload(np.arange(rows, dtype=np.uint32) + 5), ctx.upload(np.arange(rows, dtype=np.uint64) + 3)
    args = dict(n_rows=rows, n_heads=heads, variant=I.ROPE_NEOX, base_freq=1e4, q=dq.ptr, k=dk.ptr, v=dv.ptr,
                positions=pos.ptr, slots=slots.ptr, q_out=dq.ptr, q_dtype=I.F32)
    ctx.paged_rope_store(cache.args(None, 1), I.PagedRope(**args))
    ref = rope_ref(q.astype(np.float64), np.arange(rows) + 5, 1e4, True)
    assert np.abs(dq.download().reshape(q.shape) - ref).max() < 4 * 2.0 ** -20
    # base 0 turns nothing; no q
    ctx.paged_rope_store(cache.args(None, 1), I.PagedRope(**{**args, "base_freq": 0.0, "q": None, "q_out": None}))
    np.testing.assert_array_equal(cache.dk.download().reshape(32, kvh, hs)[3:3 + rows], k)
    np.testing.assert_array_equal(cache.dv.download().reshape(32, kvh, hs)[3:3 + rows], v)
    for b in (dq, dk, dv, pos, slots):
        b.free()
    cache.free()


# ------------------------------------------------------------- attention --

TYPES = {"f16": (I.F16, I.F16), "mixed": (I.F32, I.F16), "f32": (I.F32, I.F32)}


def attn_case(ctx, rng, kind, heads, kvh, hs, page, lens, window=0, sinks=0, layout="dense", fill=np.nan, tail=0,
              bad_pages=(), scale=0.0, max_new=None, max_kv=None, q_std=2.0, edit=None, ld_pad=0, in_place=False):
    """Runs one call over requests (rows in the cache before, new rows) and returns (got, reference, bound per row and
    head).  `fill` stands wherever no row of a request was written; bad_pages: (request, index in its table)."""
    qt, kt = TYPES[kind]
    n = len(lens)
    total = [c + m for c, m in lens]
    most = max(-(-t // page) for t in total) + 2 if max(total) else 2
    n_pages = sum(-(-t // page) for t in total) + 2
    cache = Paged(ctx, rng, kt, n_pages, page, kvh, hs, layout, fill)
    order = list(rng.permutation(n_pages))
    table = np.full((n, most), NO, np.uint32)
    keys, vals = [], []
    for r, t in enumerate(total):
        k, v = (rng.standard_normal((t, kvh, hs)).astype(NP[kt]) for _ in range(2))
        if edit:
            edit(r, k, v)
        for i in range(-(-t // page)):
            table[r, i] = order.pop()
        for i in range(t):
            cache.put(int(table[r, i // page]), i % page, k[i], v[i])
        keys.append(k)
        vals.append(v)
    for r, i in bad_pages:
        table[r, i] = NO if i % 2 else n_pages
    cache.upload()
    rows = sum(m for _, m in lens)
    ld = heads * hs + ld_pad
    q = (rng.standard_normal((rows + tail, ld)) * q_std).astype(NP[qt])
    dq = ctx.upload(q)
    dout = dq if in_place else ctx.upload(np.full(q.size, 7, NP[qt]))
    start = np.concatenate([[0], np.cumsum([m for _, m in lens])]).astype(np.uint32)
    dt, dstart, dkv = ctx.upload(table), ctx.upload(start), ctx.upload(np.array(total, np.uint32))
    I.PagedAttention.launch(ctx, cache.args(dt, most), I.PagedAttentionParams(
        n_requests=n, n_rows=rows + tail, n_heads=heads, q_dtype=qt, window=window, n_sinks=sinks, scale=scale,
        max_new=max(m for _, m in lens) if max_new is None else max_new, max_kv=max(total) if max_kv is None else max_kv,
        row_start=dstart.ptr, kv_len=dkv.ptr, q=dq.ptr, out=dout.ptr, ld_q=ld, ld_out=ld))
    got = dout.download(NP[qt]).reshape(rows + tail, ld)
    if not in_place:
        assert (got[rows:] == 7).all() and (got[:, heads * hs:] == 7).all(), "rows or columns of nobody were written"
    got = got[:rows, :heads * hs].reshape(rows, heads, hs).astype(np.float64)
    ref, tol = np.zeros((rows, heads, hs)), np.zeros((rows, heads, 1))
    sc = scale or 1.0 / np.sqrt(hs)
    with np.errstate(invalid="ignore", over="ignore"):
        for r, (c, m) in enumerate(lens):
            if not m:
                continue
            there = np.ones(total[r], bool)
            for rr, i in bad_pages:
                if rr == r:
                    there[i * page:(i + 1) * page] = False
            x = q[start[r]:start[r] + m, :heads * hs].reshape(m, heads, hs)
            ref[start[r]:start[r] + m] = attn_ref(x, keys[r], vals[r], np.arange(c, c + m), window, sinks, scale, there)
            kk = np.repeat(np.abs(keys[r]).astype(np.float64), heads // kvh, 1)
            finite = np.where(np.isfinite(kk), kk, 0)
            mass = np.einsum("ihd,jhd->ihj", np.abs(x.astype(np.float64)), finite).max(-1) * sc
            vm = np.abs(np.where(np.isfinite(vals[r]), vals[r], 0)).max() if total[r] else 0
            b = (hs * 2.0 ** -23 + 2.0 ** -21) * mass * 2 + total[r] * 2.0 ** -24 + 2.0 ** -20
            if kind == "f16":
                b = b + 2.0 ** -11 + total[r] * 2.0 ** -25
            tol[start[r]:start[r] + m, :, 0] = b * float(vm)
    if kind == "f16":
        tol = tol + 2.0 ** -11 * np.abs(np.where(np.isfinite(ref), ref, 0)) + 2.0 ** -24
    for x in {id(x): x for x in (dq, dout, dt, dstart, dkv)}.values():
        x.free()
    cache.free()
    return got, ref, tol


def check(got, ref, tol):
    odd = ~np.isfinite(ref)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(ref))
    np.testing.assert_array_equal(got[odd & ~np.isnan(ref)], ref[odd & ~np.isnan(ref)])
    err = np.where(odd, 0, np.abs(got - np.where(odd, got, ref)))
    worst = np.nanmax(err / np.broadcast_to(tol, err.shape))
    assert worst <= 1.0, f"off by {worst:.2f} of the bound"


KINDS = ["f16", "mixed", "f32"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hs", [(32, 4, 64), (32, 8, 128), (14, 2, 64), (12, 2, 128), (5, 5, 80), (6, 2, 8),
                                          (40, 2, 96), (17, 1, 128), (64, 2, 40), (3, 1, 104)])
def test_decode_heads_and_sizes(ctx, kind, heads, kvh, hs):
    """One row per request at lengths around the tiles' and pages' ends."""
    rng = np.random.default_rng(heads * hs)
    lens = [(c, 1) for c in (0, 1, 15, 16, 30, 31, 32, 33, 63, 127, 128, 144, 300)]
    check(*attn_case(ctx, rng, kind, heads, kvh, hs, 16, lens, tail=3))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("layout", ["dense", "gap", "heads"])
def test_chunks_pages_and_layouts(ctx, kind, page, layout):
    """Prompt chunks, decodes, requests without rows and first tokens in one call."""
    rng = np.random.default_rng(page)
    lens = [(0, 1), (0, 70), (37, 1), (5, 0), (100, 33), (0, 2), (257, 5), (63, 129)]
    check(*attn_case(ctx, rng, kind, 8, 2, 64, page, lens, layout=layout, tail=2, ld_pad=8))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hs", [(4, 4, 128), (6, 2, 64), (7, 1, 128), (64, 1, 64), (72, 1, 32), (130, 1, 16)])
def test_chunks_groups(ctx, kind, heads, kvh, hs):
    rng = np.random.default_rng(heads)
    check(*attn_case(ctx, rng, kind, heads, kvh, hs, 32, [(50, 40), (0, 131), (200, 3), (90, 17)]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (7, 1), (32, 0), (33, 40), (64, 4), (100, 300), (129, 65), (1000, 4)])
def test_window_and_sinks(ctx, kind, window, sinks):
    rng = np.random.default_rng(window)
    lens = [(0, 1), (31, 1), (300, 1), (333, 3), (150, 100), (0, 200), (500, 1), (64, 64)]
    check(*attn_case(ctx, rng, kind, 8, 2, 128 if window % 2 else 64, 16, lens, window=window, sinks=sinks))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [0, 3000])
def test_long_decode_in_splits(ctx, kind, window):
    rng = np.random.default_rng(9)
    check(*attn_case(ctx, rng, kind, 8, 2, 128, 64, [(9000, 1), (17, 1), (4099, 1)], window=window, sinks=4 if window else 0))
    check(*attn_case(ctx, rng, kind, 4, 1, 64, 128, [(20001, 2)], window=window, sinks=70 if window else 0))


@pytest.mark.parametrize("kind", KINDS)
def test_long_chunk_over_a_long_context(ctx, kind):
    """Few tiles over many keys, and a chunk that is its own context."""
    rng = np.random.default_rng(10)
    check(*attn_case(ctx, rng, kind, 8, 2, 128, 64, [(5000, 70)]))
    check(*attn_case(ctx, rng, kind, 4, 2, 64, 16, [(0, 700), (3000, 1)]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [0, 40])
def test_what_is_masked_may_be_anything(ctx, kind, window):
    """Infinities and NaN in rows that a query does not see (later rows of its chunk, rows behind its window, rows past
    the last, pages that are none) have no part in its result; those it sees have."""
    rng = np.random.default_rng(11)
    lens = [(70, 20), (45, 1), (0, 33), (200, 150), (90, 3)]

    def edit(r, k, v):
        if r == 0:
            k[85, :, 3], v[85, :, 5] = np.nan, np.nan   # seen from position 85 on
            v[80, 0, 2], v[88, :, 7] = np.inf, -np.inf
        if r == 1:
            k[3], v[4] = np.nan, np.inf                  # behind the window of 40
        if r == 3:
            v[300, 1, 0] = np.inf
            v[40, :, 1] = np.nan
        if r == 4:
            v[91, 0, 0], k[92, 1] = np.nan, np.inf

    got, ref, tol = attn_case(ctx, rng, kind, 8, 2, 64, 16, lens, window=window, sinks=2 if window else 0, edit=edit,
                              bad_pages=[(2, 1), (3, 2)])
    check(got, ref, tol)
    assert np.isfinite(got[:10]).all() and np.isnan(got[19]).any()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_see_nothing_are_zero(ctx, kind):
    rng = np.random.default_rng(12)
    # every page of request 1 is none
    got, ref, tol = attn_case(ctx, rng, kind, 4, 2, 64, 16, [(10, 3), (20, 30), (3, 1)], bad_pages=[(1, 0), (1, 1), (1, 2), (1, 3)])
    check(got, ref, tol)
    assert (got[3:33] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_refused_requests_and_short_caches(ctx, kind):
    """kv_len 0 (a refused request) and kv_len below the new rows (first rows before the cache): zeros."""
    rng = np.random.default_rng(13)
    qt, kt = TYPES[kind]
    heads, kvh, hs, page = 8, 2, 64, 16
    cache = Paged(ctx, rng, kt, 6, page, kvh, hs)
    k, v = (rng.standard_normal((40, kvh, hs)).astype(NP[kt]) for _ in range(2))
    for i in range(40):
        cache.put(i // page, i % page, k[i], v[i])
    cache.upload()
    n = [5, 30, 4, 200, 40]
    kv = [0, 10, 0, 0, 40]
    rows = sum(n)
    q = rng.standard_normal((rows, heads, hs)).astype(NP[qt])
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
    table = ctx.upload(np.tile(np.arange(3, dtype=np.uint32), (5, 1)))
    dq, dout = ctx.upload(q), ctx.upload(np.full(q.shape, 7, NP[qt]))
    ds, dk = ctx.upload(start), ctx.upload(np.array(kv, np.uint32))
    I.PagedAttention.launch(ctx, cache.args(table, 3), I.PagedAttentionParams(
        n_requests=5, n_rows=rows, n_heads=heads, q_dtype=qt, max_new=200, max_kv=40, row_start=ds.ptr, kv_len=dk.ptr,
        q=dq.ptr, out=dout.ptr))
    got = dout.download(NP[qt]).reshape(q.shape).astype(np.float64)
    for r in range(5):
        ref = attn_ref(q[start[r]:start[r + 1]], k[:kv[r]], v[:kv[r]], np.arange(kv[r] - n[r], kv[r]))
        assert np.abs(got[start[r]:start[r + 1]] - ref).max() < (4e-3 if kind == "f16" else 2e-5)
        assert (got[start[r]:start[r + 1]][:max(n[r] - kv[r], 0)] == 0).all()
    for b in (table, dq, dout, ds, dk):
        b.free()
    cache.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("max_new,max_kv", [(1, 1), (0, 0), (3, 64), (500, 100000)])
def test_bounds_only_size_the_launch(ctx, kind, max_new, max_kv):
    rng = np.random.default_rng(14)
    check(*attn_case(ctx, rng, kind, 8, 2, 64, 16, [(100, 1), (500, 9), (0, 60), (1500, 1)], max_new=max_new, max_kv=max_kv))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("max_kv", [1, 300, 0])
def test_unequal_decodes_past_the_bound(ctx, kind, max_kv):
    """Decodes of very unequal lengths, most or all longer than the caller said: up to 64 and more requests."""
    rng = np.random.default_rng(19)
    for n in (2, 40, 64, 70):
        lens = [(int(c), 1) for c in np.exp(rng.uniform(0, np.log(2500), n))]
        lens[n // 2] = (6000, 1)
        check(*attn_case(ctx, rng, kind, 4, 2, 64, 16, lens, max_kv=max_kv))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 3, 33, 64, 130])
def test_equal_decodes(ctx, kind, n):
    """Decodes of the same length, around the lengths where they are split, with requests that have no rows between."""
    rng = np.random.default_rng(22)
    for c in (510, 511, 512, 544, 1023, 1024, 1100):
        lens = [(7, 0) if i % 13 == 5 else (c, 1) for i in range(n)]
        check(*attn_case(ctx, rng, kind, 4, 2, 64, 32, lens))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("requests", [1, 5, 66])
def test_windows_with_more_rows_than_the_bound(ctx, kind, requests):
    """Rows past max_new under a window of some whole chunks of keys: a request's earlier tiles reach over more key
    tiles than its last one."""
    rng = np.random.default_rng(20)
    for window in (225, 240, 256, 481, 490, 497, 505, 512, 520):
        lens = [(1000 + 13 * i, 9 + i % 40) if i < 5 else (3, 1) for i in range(requests)]
        check(*attn_case(ctx, rng, kind, 4, 2, 64, 16, lens, window=window, sinks=window % 5, max_new=1))


@pytest.mark.parametrize("kind", KINDS)
def test_values_far_from_one(ctx, kind):
    """Large scores (one row carries all), tiny and huge query rows, a scale of the caller's."""
    rng = np.random.default_rng(15)
    check(*attn_case(ctx, rng, kind, 4, 2, 128, 32, [(200, 40), (90, 1)], q_std=60.0))
    check(*attn_case(ctx, rng, kind, 4, 2, 128, 32, [(200, 40), (90, 1)], q_std=1e-4))
    check(*attn_case(ctx, rng, kind, 4, 2, 64, 32, [(200, 40), (90, 1)], scale=0.7))
    if kind != "f16":
        check(*attn_case(ctx, rng, kind, 4, 2, 64, 32, [(200, 3), (90, 1)], q_std=1e-30))
        check(*attn_case(ctx, rng, kind, 4, 2, 64, 32, [(200, 3), (90, 1)], q_std=1e6, scale=1e-6))


@pytest.mark.parametrize("kind", KINDS)
def test_output_in_place_of_the_queries(ctx, kind):
    rng = np.random.default_rng(16)
    check(*attn_case(ctx, rng, kind, 8, 2, 64, 16, [(100, 1), (3000, 1), (40, 150), (0, 3)], in_place=True))


@pytest.mark.parametrize("kind", KINDS)
def test_two_calls_give_the_same_bits(ctx, kind):
    lens = [(3000, 1), (100, 200), (40, 1)]
    a = attn_case(ctx, np.random.default_rng(17), kind, 8, 2, 128, 16, lens)[0]
    b = attn_case(ctx, np.random.default_rng(17), kind, 8, 2, 128, 16, lens)[0]
    np.testing.assert_array_equal(a, b)


def test_offsets_past_32_bits(ctx):
    """Pages beyond 4 GiB of a cache (and slots there): the last pages of 5 GiB of keys hold the rows."""
    rng = np.random.default_rng(18)
    kvh, hs, page = 8, 128, 16
    n_pages = (5 << 30) // (page * kvh * hs * 2)
    key, val = ctx.alloc(n_pages * page * kvh * hs * 2), ctx.alloc(n_pages * page * kvh * hs * 2)
    rows = 40
    table = np.array([[n_pages - 1, n_pages - 3, n_pages - 2]], np.uint32)
    pos = np.arange(rows)
    slots = table[0, pos // page].astype(np.uint64) * page + (pos % page).astype(np.uint64)
    q, k, v = (rng.standard_normal((rows, h, hs)).astype(np.float32) for h in (32, kvh, kvh))
    bufs = [ctx.upload(a) for a in (q, k, v, pos.astype(np.uint32), slots, table, np.array([0, rows], np.uint32),
                                    np.array([rows], np.uint32))]
    dq, dk, dv, dp, ds, dt, dstart, dkv = bufs
    cache = I.PagedCache(key=key.ptr, value=val.ptr, block_table=dt.ptr, dtype=I.F16, n_pages=n_pages, page_size=page,
                         max_pages=3, n_kv_heads=kvh, head_size=hs)
    ctx.paged_rope_store(cache, I.PagedRope(n_rows=rows, n_heads=32, variant=0, base_freq=0.0, q=dq.ptr, k=dk.ptr, v=dv.ptr,
                                            positions=dp.ptr, slots=ds.ptr, q_out=dq.ptr, q_dtype=I.F32))
    out = ctx.alloc(q.nbytes)
    I.PagedAttention.launch(ctx, cache, I.PagedAttentionParams(n_requests=1, n_rows=rows, n_heads=32, q_dtype=I.F32, max_new=rows,
                                                               max_kv=rows, row_start=dstart.ptr, kv_len=dkv.ptr, q=dq.ptr,
                                                               out=out.ptr))
    ref = attn_ref(q, k.astype(np.float16), v.astype(np.float16), pos)
    assert np.abs(out.download().reshape(q.shape) - ref).max() < 2e-5
    for b in bufs + [key, val, out]:
        b.free()


# ------------------------------------------------- the operators together --

@pytest.mark.parametrize("kind,window", [("f16", 0), ("mixed", 0), ("f32", 0), ("f16", 50), ("mixed", 50)])
def test_serving_steps(ctx, kind, window):
    """Prompts in chunks, decode steps, a release and a request in its place, all bookkeeping left on the device: plan,
    store and attention of every step against attention over each request's whole history."""
    rng = np.random.default_rng(20)
    qt, kt = TYPES[kind]
    heads, kvh, hs, page, most, n_pages = 8, 2, 64, 16, 20, 40
    cache = Paged(ctx, rng, kt, n_pages, page, kvh, hs).upload()
    n = 4
    u = lambda a, t=np.uint32: ctx.upload(np.asarray(a, t))  # noqa: E731
    free = u(rng.permutation(n_pages))
    count, lens, table = u([n_pages]), u([0] * n), u(np.full((n, most), NO))
    steps = [[70, 33, 0, 5], [50, 1, 9, 1], [1, 1, 1, 1], [1, NO, 1, 1], [1, 120, 1, 40], [1, 1, 1, 1], [250, 1, 1, 1], [1, 1, 1, 1]]
    hist = [([], []) for _ in range(n)]
    for new in steps:
        rows = sum(v for v in new if v != NO) + 2  # two rows of nobody
        x = rng.standard_normal((rows, heads + 2 * kvh, hs)).astype(np.float32)
        b = {"new_len": u(new), "row_start": u([0] * (n + 1)), "kv_len": u([0] * n), "positions": u([0] * rows), "slots": u([0] * rows, np.uint64)}
        ctx.paged_plan(I.PagedPlan(n_requests=n, n_rows=rows, n_pages=n_pages, page_size=page, max_pages=most, ctx_len=lens.ptr,
                                   ctx_len_out=lens.ptr, free_pages=free.ptr, free_count=count.ptr, free_count_out=count.ptr,
                                   block_table=table.ptr, **{k: v.ptr for k, v in b.items()}))
        args = cache.args(table, most)
        dx, wide = ctx.upload(x), (heads + 2 * kvh) * hs
        q, out = ctx.alloc(rows * heads * hs * 4), ctx.upload(np.full((rows, heads, hs), 7, NP[qt]))
        ctx.paged_rope_store(args, I.PagedRope(
            n_rows=rows, n_heads=heads, variant=I.ROPE_NEOX, base_freq=1e4, q=dx.ptr, k=dx.ptr + 4 * heads * hs,
            v=dx.ptr + 4 * (heads + kvh) * hs, ld_q=wide, ld_k=wide, ld_v=wide, positions=b["positions"].ptr,
            slots=b["slots"].ptr, q_out=q.ptr, q_dtype=qt))
        I.PagedAttention.launch(ctx, args, I.PagedAttentionParams(
            n_requests=n, n_rows=rows, n_heads=heads, q_dtype=qt, max_new=max(v for v in new if v != NO), window=window,
            n_sinks=3 if window else 0, row_start=b["row_start"].ptr, kv_len=b["kv_len"].ptr, q=q.ptr, out=out.ptr))
        got = out.download(NP[qt]).reshape(rows, heads, hs).astype(np.float64)
        kv, start = b["kv_len"].download(np.uint32), b["row_start"].download(np.uint32)
        assert (got[start[-1]:] == 7).all()
        for r, v in enumerate(new):
            if v == NO:
                hist[r] = ([], [])
                assert kv[r] == 0
                continue
            c = len(hist[r][0])
            mine = x[start[r]:start[r] + v].astype(np.float64)
            if kv[r] == 0 and v:
                assert new == steps[6] and r == 0, "only the prompt that the pages do not hold is refused"
                assert (got[start[r]:start[r] + v] == 0).all()
                continue
            assert kv[r] == c + v
            turned = rope_ref(mine[:, :heads + kvh], np.arange(c, c + v), 1e4, True)
            hist[r][0].extend(turned[:, heads:].astype(NP[kt]))
            hist[r][1].extend(mine[:, heads + kvh:].astype(NP[kt]))
            if not v:
                continue
            ref = attn_ref(turned[:, :heads].astype(NP[qt]), np.array(hist[r][0]), np.array(hist[r][1]), np.arange(c, c + v), window,
                           3 if window else 0)
            # rows of f16 caches may be one rounding apart from the plain ones: 2^-11 of scores up to 12 and of values up to 5
            lim = 2e-5 if kind == "f32" else 12 * 5 * 2.0 ** -11
            assert np.abs(got[start[r]:start[r] + v] - ref).max() < lim
        for y in (*b.values(), dx, q, out):
            y.free()
    assert lens.download(np.uint32).tolist() == [len(h[0]) for h in hist]
    used = sum(-(-len(h[0]) // page) for h in hist)
    left = int(count.download(np.uint32)[0])
    assert left == n_pages - used
    # no page is lost or held twice
    t = table.download(np.uint32).reshape(n, most)
    held = [int(t[r, i]) for r in range(n) for i in range(-(-len(hist[r][0]) // page))]
    assert sorted(held + free.download(np.uint32)[:left].tolist()) == list(range(n_pages))
    for y in (free, count, lens, table):
        y.free()
    cache.free()


def test_code_object_without_the_paged_one_beside_it(tmp_path):
    """A code object of the caller's in a directory of its own: the paged kernels then come from the library's."""
    path = tmp_path / "kernels.hsaco"
    shutil.copy(I.HSACO_PATH, path)
    other = I.LlmContext(0, str(path))
    a, b = other.upload(np.arange(8, dtype=np.float32)), other.upload(np.ones(8, np.float32))
    other.add_assign(a, b, 8)
    np.testing.assert_array_equal(a.download(), np.arange(8) + 1)
    check(*attn_case(other, np.random.default_rng(21), "f16", 4, 2, 64, 16, [(20, 1), (0, 40)]))
    a.free()
    b.free()
    other.close()
