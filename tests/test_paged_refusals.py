"""What the paged operators refuse, checked on the CPU: the host side built by
g++ around a context without kernels (tests/paged_host.cpp).  Arguments that
pass every check end in EUNSUPPORTED, "not in the code object"."""

import ctypes as C
import os
import shutil
import subprocess

import pytest

import inferi_amd as I

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
EINVAL, EUNSUPPORTED = 1, 2
A = 1 << 20  # an aligned address that nothing follows


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx or not os.path.exists(os.path.join(ROCM, "include", "hip")):
        pytest.skip("no g++ or no HIP headers")
    out = str(tmp_path_factory.mktemp("paged") / "libpaged_host.so")
    subprocess.run([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include",
                    os.path.join(ROOT, "tests", "paged_host.cpp"), os.path.join(ROOT, "inferi_amd", "csrc", "paged.cpp"),
                    f"-L{ROCM}/lib", "-lamdhip64", f"-Wl,-rpath,{ROCM}/lib", "-o", out], check=True)
    lib = C.CDLL(out)
    lib.paged_host_ctx.restype = C.c_void_p
    lib.paged_host_error.restype, lib.paged_host_error.argtypes = C.c_char_p, [C.c_void_p]
    lib.paged_host_free.argtypes = [C.c_void_p]
    for n in ("ifr_paged_plan", "ifr_paged_rope_store", "ifr_paged_attention"):
        getattr(lib, n).restype, getattr(lib, n).argtypes = I.SIGNATURES[n]
    ctx = lib.paged_host_ctx()
    yield lib, ctx
    lib.paged_host_free(ctx)


CACHE = dict(key=A, value=A, block_table=A, dtype=I.F16, n_pages=10, page_size=16, max_pages=8, n_kv_heads=2, head_size=64)
PLAN = dict(n_requests=3, n_rows=9, n_pages=10, page_size=16, max_pages=8, ctx_len=A, new_len=A, free_pages=A, free_count=A,
            free_count_out=A, block_table=A, ctx_len_out=A, row_start=A, kv_len=A, positions=A, slots=A)
ROPE = dict(n_rows=9, n_heads=4, variant=0, base_freq=1e4, q=A, k=A, v=A, positions=A, slots=A, q_out=A + 64, q_dtype=I.F16)
ATTN = dict(n_requests=3, n_rows=9, n_heads=4, q_dtype=I.F16, max_new=1, max_kv=8, row_start=A, kv_len=A, q=A, out=A)


def plan(host, **kw):
    lib, ctx = host
    return lib.ifr_paged_plan(ctx, I.PagedPlan(**{**PLAN, **kw})), lib.paged_host_error(ctx).decode()


def rope(host, cache=None, **kw):
    lib, ctx = host
    return lib.ifr_paged_rope_store(ctx, I.PagedCache(**{**CACHE, **(cache or {})}), I.PagedRope(**{**ROPE, **kw})), \
        lib.paged_host_error(ctx).decode()


def attn(host, cache=None, **kw):
    lib, ctx = host
    return lib.ifr_paged_attention(ctx, I.PagedCache(**{**CACHE, **(cache or {})}), I.PagedAttentionParams(**{**ATTN, **kw})), \
        lib.paged_host_error(ctx).decode()


def test_good_arguments_reach_the_kernels(host):
    for call, kw in ((plan, {}), (plan, dict(ctx_len_out=None)), (plan, dict(n_requests=0, ctx_len=None, kv_len=None)),
                     (plan, dict(n_rows=0, positions=None, slots=None)), (rope, {}), (rope, dict(q=None, q_out=None)),
                     (rope, dict(base_freq=0.0)), (rope, dict(cache=dict(block_table=None))), (rope, dict(q_out=A, q_dtype=I.F32)),
                     (attn, {}), (attn, dict(q_dtype=I.F32)), (attn, dict(q_dtype=I.F32, cache=dict(dtype=I.F32))),
                     (attn, dict(window=5, n_sinks=99)), (attn, dict(n_heads=130)), (attn, dict(max_new=0, max_kv=0)),
                     (attn, dict(cache=dict(head_stride=16 * 64, row_stride=64, page_stride=2 * 16 * 64)))):
        st, why = call(host, **kw)
        assert st == EUNSUPPORTED and "not in the code object" in why, (call.__name__, kw, st, why)
    lib, ctx = host
    for n in ("ifr_paged_plan", "ifr_paged_rope_store", "ifr_paged_attention"):
        assert getattr(lib, n)(None, *[None] * (len(I.SIGNATURES[n][1]) - 1)) == EINVAL
        assert getattr(lib, n)(ctx, *[None] * (len(I.SIGNATURES[n][1]) - 1)) == EINVAL


def test_nothing_to_do_is_fine(host):
    assert rope(host, n_rows=0)[0] == 0 and attn(host, n_rows=0)[0] == 0 and attn(host, n_requests=0)[0] == 0


@pytest.mark.parametrize("kw", [dict(page_size=0), dict(page_size=8), dict(page_size=48), dict(page_size=1 << 31), dict(n_pages=0),
                                dict(n_pages=0xFFFFFFFF), dict(max_pages=0), dict(max_pages=(1 << 26) + 1),
                                dict(n_rows=(1 << 30) + 1), dict(n_requests=0xFFFFFFFF)]
                         + [{k: None} for k in ("ctx_len", "new_len", "free_pages", "free_count", "free_count_out",
                                                "block_table", "row_start", "kv_len", "positions", "slots")])
def test_plan_refuses(host, kw):
    assert plan(host, **kw)[0] == EINVAL


BAD_CACHE = [dict(key=None), dict(value=None), dict(dtype=I.Q4_K), dict(page_size=24), dict(n_pages=0), dict(n_kv_heads=0),
             dict(key=A + 8), dict(value=A + 4), dict(row_stride=-128), dict(row_stride=132), dict(head_stride=68),
             dict(page_stride=4), dict(row_stride=(1 << 25) + 8), dict(page_stride=1 << 60), dict(dtype=I.F32, row_stride=130)]


@pytest.mark.parametrize("cache", BAD_CACHE)
def test_cache_refuses(host, cache):
    assert rope(host, cache)[0] == EINVAL
    assert attn(host, cache, q_dtype=I.F32)[0] == EINVAL


@pytest.mark.parametrize("hs", [0, 4, 60, 136, 256])
def test_head_sizes_refused(host, hs):
    assert rope(host, dict(head_size=hs))[0] == EUNSUPPORTED and "head_size" in rope(host, dict(head_size=hs))[1]
    assert attn(host, dict(head_size=hs))[0] == EUNSUPPORTED and "head_size" in attn(host, dict(head_size=hs))[1]


@pytest.mark.parametrize("kw", [dict(variant=2), dict(base_freq=-1.0), dict(base_freq=float("nan")), dict(base_freq=float("inf")),
                                dict(k=None), dict(v=None), dict(positions=None), dict(slots=None), dict(q=None), dict(q_out=None),
                                dict(n_heads=0), dict(n_heads=70000), dict(q_dtype=I.Q8_0), dict(ld_q=252), dict(ld_q=258),
                                dict(ld_k=124), dict(ld_v=130), dict(ld_q_out=260), dict(ld_q=-256), dict(q=A + 4), dict(k=A + 8),
                                dict(v=A + 2), dict(q_out=A + 8), dict(q_out=A), dict(q_out=A, q_dtype=I.F32, ld_q_out=512),
                                dict(n_rows=0xFFFFFFFF)])
def test_rope_store_refuses(host, kw):
    assert rope(host, **kw)[0] == EINVAL


@pytest.mark.parametrize("kw", [dict(row_start=None), dict(kv_len=None), dict(q=None), dict(out=None), dict(n_heads=0), dict(n_heads=5),
                                dict(q_dtype=I.Q8_0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(ld_q=248),
                                dict(ld_q=260), dict(ld_out=252), dict(q=A + 8), dict(out=A + 4), dict(ld_out=512),
                                dict(cache=dict(block_table=None)), dict(cache=dict(max_pages=1 << 27)), dict(n_rows=0xFFFFFFFF)])
def test_attention_refuses(host, kw):
    assert attn(host, **kw)[0] == EINVAL


def test_attention_does_not_take(host):
    assert attn(host, dict(dtype=I.F32))[0] == EUNSUPPORTED       # f16 queries over an f32 cache
    assert "f16 queries" in attn(host, dict(dtype=I.F32))[1]
    st, why = rope(host, n_rows=1 << 24)                           # a workgroup a row
    assert st == EUNSUPPORTED and "rows" in why and "code object" not in why
    st, why = attn(host, n_requests=1 << 23, n_heads=2)            # more workgroups than one launch takes
    assert st == EUNSUPPORTED and "workgroups" in why


@pytest.mark.parametrize("scale,ok", [(0.0, True), (2.0 ** -60, True), (2.0 ** 14, True), (2.0 ** -61, False), (1e-30, False),
                                      (2.0 ** 14 * 1.001, False), (1e5, False), (-0.5, False)])
def test_scales(host, scale, ok):
    assert attn(host, scale=scale)[0] == (EUNSUPPORTED if ok else EINVAL)


def test_plan_tables(host):
    """Entries of 1024 requests are counted in 32 bits."""
    assert plan(host, n_requests=31, max_pages=1 << 26)[0] == EUNSUPPORTED
    assert plan(host, n_requests=32, max_pages=1 << 26)[0] == EINVAL
    assert plan(host, n_requests=1 << 20, max_pages=(1 << 21) - 1)[0] == EUNSUPPORTED
    assert plan(host, n_requests=1 << 20, max_pages=1 << 21)[0] == EINVAL


def test_many_rows_over_long_tables(host):
    """Launches of many tiles take fewer splits, not an error."""
    assert "not in the code object" in attn(host, dict(page_size=1 << 20, max_pages=1 << 10), n_requests=1 << 20, n_rows=1 << 20,
                                            max_kv=0)[1]
