"""Argument checks of the serving operators: every one is made before the first CUDA call, so they run without a GPU."""
import ctypes as C

import pytest

from ava_b200 import build, engine, serving

ARG, CUDA, NOT = engine.ERR_ARG, engine.ERR_CUDA, engine.NOT_APPLICABLE


@pytest.fixture(scope="module")
def L():
    build.build()
    return engine.lib()


@pytest.fixture(scope="module")
def mem():
    """64-byte-aligned host bytes: the refusals below never read what a pointer points at."""
    buf = (C.c_char * 8192)()
    base = C.addressof(buf)
    mem.keep = buf
    return base + (-base) % 64


def store(at, **kw):
    f = dict(k=at, v=at, dtype=1, n_pages=4, kv_heads=2, page_size=8, head_size=64, page_stride=1024, head_stride=512, place_stride=64)
    f.update(kw)
    return serving.PagedStore(**f)


PLAN = ["cached", "fresh", "rows", "page_size", "n_pages", "table", "max_pages", "owned", "owned_out", "free_list", "free_count", "free_count_out", "trim", "q_start",
        "slot", "pos", "row", "max_tokens", "status"]


def plan(L, at, **kw):
    a = {n: at for n in PLAN}
    a.update(rows=3, page_size=8, n_pages=4, max_pages=2, trim=1, max_tokens=16)
    a.update(kw)
    return L.ava_paged_plan(99, None, *[a[n] for n in PLAN])


APPEND = ["store", "k", "v", "dtype", "token_stride", "head_stride", "slot", "tokens", "status"]


def append(L, at, **kw):
    a = dict(k=at, v=at, dtype=1, token_stride=128, head_stride=64, slot=at, tokens=5, status=at, store=store(at))
    a.update(kw)
    a["store"] = C.byref(a["store"]) if a["store"] is not None else None
    return L.ava_paged_append(99, None, *[a[n] for n in APPEND])


ATTEND = ["store", "q", "dtype", "q_token_stride", "q_head_stride", "heads", "table", "max_pages", "cached", "first", "q_start", "rows", "max_tokens", "max_fresh", "scale",
          "window", "out", "out_token_stride", "out_head_stride", "lse", "workspace", "workspace_bytes", "status"]


def attend(L, at, **kw):
    a = {n: at for n in ATTEND}
    a.update(store=store(at), dtype=1, q_token_stride=256, q_head_stride=64, heads=4, max_pages=2, rows=3, max_tokens=16, max_fresh=2, scale=0.125, window=0,
             out_token_stride=256, out_head_stride=64, workspace_bytes=1 << 40)
    a.update(kw)
    a["store"] = C.byref(a["store"]) if a["store"] is not None else None
    return L.ava_paged_attend(99, None, *[a[n] for n in ATTEND])


VERIFY = ["p", "p_stride", "q", "q_stride", "tok", "q_start", "rows", "max_tokens", "vocab", "uniform", "max_out", "out", "n_out", "status"]


def verify(L, at, **kw):
    a = {n: at for n in VERIFY}
    a.update(p_stride=100, q_stride=100, rows=2, max_tokens=6, vocab=100, max_out=3)
    a.update(kw)
    return L.ava_verify_drafts(99, None, *[a[n] for n in VERIFY])


@pytest.mark.parametrize("call", [plan, append, attend, verify])
def test_good_arguments_reach_the_device_check(L, mem, call):
    """Device 99 is on no machine: the arguments are fine, so that is what is left to refuse."""
    assert call(L, mem) == CUDA
    assert b"no such CUDA device" in L.ava_serving_last_error()


@pytest.mark.parametrize("call,kw", [
    *[(plan, {n: None}) for n in ("cached", "fresh", "table", "owned", "owned_out", "free_list", "free_count", "free_count_out", "q_start", "slot")],
    *[(plan, {n: v}) for n in ("rows", "page_size", "n_pages", "max_pages") for v in (0, -1)], (plan, dict(max_tokens=-1)),
    *[(append, {n: None}) for n in ("store", "k", "v", "slot")], (append, dict(tokens=-1)), (append, dict(dtype=2)), (append, dict(token_stride=-1)),
    *[(attend, {n: None}) for n in ("store", "q", "out", "table", "cached", "q_start")],
    *[(attend, {n: v}) for n in ("rows", "max_pages", "heads") for v in (0, -1)],
    (attend, dict(max_tokens=-1)), (attend, dict(max_fresh=-1)), (attend, dict(window=-1)), (attend, dict(heads=3)), (attend, dict(dtype=-1)),
    (attend, dict(scale=float("nan"))), (attend, dict(scale=float("inf"))), (attend, dict(out_head_stride=32)), (attend, dict(q_token_stride=-8)),
    *[(verify, {n: None}) for n in ("p", "tok", "q_start", "out", "n_out")], *[(verify, {n: 0}) for n in ("rows", "vocab", "max_out")],
    (verify, dict(p_stride=99)), (verify, dict(q_stride=99)), (verify, dict(uniform=None)),
])
def test_refused_arguments(L, mem, call, kw):
    assert call(L, mem, **kw) == ARG
    assert L.ava_serving_last_error()


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(dtype=2), dict(n_pages=0), dict(kv_heads=0), dict(page_size=0), dict(head_size=0), dict(page_stride=-1),
                                dict(place_stride=63)])
def test_refused_stores(L, mem, call, kw):
    assert call(L, mem, store=store(mem, **kw)) == ARG


def test_misaligned_pointers_are_refused(L, mem):
    for n in ("cached", "table", "free_list", "q_start", "pos", "status"):
        assert plan(L, mem, **{n: mem + 2}) == ARG
    assert plan(L, mem, slot=mem + 4) == ARG
    assert append(L, mem, k=mem + 1) == ARG and append(L, mem, slot=mem + 4) == ARG
    assert append(L, mem, dtype=0, k=mem + 2, store=store(mem, dtype=0)) == ARG
    assert append(L, mem, store=store(mem + 1)) == ARG
    assert attend(L, mem, q=mem + 1) == ARG and attend(L, mem, table=mem + 2) == ARG and attend(L, mem, lse=mem + 1) == ARG
    assert verify(L, mem, uniform=mem + 4) == ARG and verify(L, mem, p=mem + 2) == ARG


def test_types_and_sizes_that_are_not_covered(L, mem):
    assert append(L, mem, dtype=1, store=store(mem, dtype=0)) == NOT
    assert attend(L, mem, dtype=1, store=store(mem, dtype=0)) == NOT
    for hs in (1, 48, 96, 256):
        assert attend(L, mem, store=store(mem, head_size=hs, place_stride=hs), out_head_stride=hs) == NOT
    assert L.ava_paged_attend_workspace(0, 48) == -1


def test_sizes_beyond_the_kernels_indexes_are_refused(L, mem):
    for kw in (dict(rows=(1 << 24) + 1), dict(max_tokens=(1 << 30) + 1), dict(n_pages=(1 << 30) + 1)):
        assert plan(L, mem, **kw) == NOT
    assert plan(L, mem, rows=1 << 24, max_tokens=1 << 30, n_pages=1 << 30) == CUDA
    assert attend(L, mem, rows=(1 << 24) + 1) == NOT and attend(L, mem, max_tokens=(1 << 28) + 1) == NOT and attend(L, mem, max_tokens=1 << 28) == CUDA
    assert verify(L, mem, rows=(1 << 24) + 1) == NOT and verify(L, mem, vocab=(1 << 30) + 1, p_stride=1 << 40, q_stride=1 << 40) == NOT
    wide = store(mem, kv_heads=1 << 20, head_size=1 << 11, place_stride=1 << 11, head_stride=1 << 14, page_stride=1 << 40)
    assert append(L, mem, store=wide) == ARG


@pytest.mark.parametrize("kw", [dict(page_stride=0), dict(head_stride=0), dict(head_stride=256), dict(page_stride=1023), dict(place_stride=128), dict(place_stride=64, head_stride=64),
                                dict(page_stride=448, head_stride=512, place_stride=64)])
def test_a_store_that_overlaps_itself_is_refused_where_it_is_written(L, mem, kw):
    assert append(L, mem, store=store(mem, **kw)) == ARG
    assert b"overlap" in L.ava_serving_last_error()


@pytest.mark.parametrize("kw", [dict(head_stride=64, place_stride=128), dict(page_stride=64, place_stride=256, head_stride=2048), dict(n_pages=1, page_stride=0),
                                dict(kv_heads=1, head_stride=0)])
def test_a_store_in_any_order_of_its_dimensions_is_written(L, mem, kw):
    assert append(L, mem, store=store(mem, **kw)) == CUDA


def test_a_result_that_overlaps_itself_is_refused(L, mem):
    assert attend(L, mem, out_token_stride=0) == ARG and attend(L, mem, out_token_stride=128) == ARG
    assert attend(L, mem, out_token_stride=64, out_head_stride=16 * 64) == CUDA                 # [heads][tokens][channels]
    assert attend(L, mem, out_token_stride=0, max_tokens=1) == CUDA and attend(L, mem, out_token_stride=64, heads=2, out_head_stride=64) == ARG
    assert attend(L, mem, q_token_stride=0, q_head_stride=0) == CUDA                            # read: broadcasts are fine


def test_numbers_beyond_32_bits_are_refused():
    import torch
    z = torch.zeros(4, dtype=torch.int32)
    for kw in (dict(window=1 << 32), dict(max_fresh=1 << 31)):
        with pytest.raises(ValueError, match="32 bits"):
            serving.attend(z, z, z, z, z, z, z, **{**dict(max_fresh=1, workspace=z, scale=1.0), **kw})
    with pytest.raises(ValueError, match="32 bits"):
        serving.plan(z, z, z, z, z, z, (1 << 32) + 16, z, z)


def test_host_tensors_are_refused():
    import torch
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        serving.plan(z, z, z.view(4, 1), z, z, z[:1], 8, torch.zeros(5, dtype=torch.int32), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        serving.verify_drafts(torch.zeros(4, 9), z, z, z.view(4, 1), z)
