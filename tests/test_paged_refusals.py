"""What the paged cache's entry points refuse, through the C ABI: the checks come before the device, so they run without one."""
import ctypes as C

import pytest

from ferric_amd import _lib

OK, TYPE, SHAPE, ARG = _lib.OK, _lib.ERR_UNSUPPORTED_TYPE, _lib.ERR_SHAPE, _lib.ERR_ARG
P = 0x1000      # no memory of anybody: every call here returns before it would be looked at


def cache(**more):
    f = dict(type=0, page_rows=16, n_pages=8, n_kv=2, head_dim=64, d_k=P, d_v=P, d_k_scales=None, d_v_scales=None, d_table=P, n_seq=3, pages_per_seq=4, table_stride=4)
    f.update(more)
    return C.byref(_lib.Paged(*[f[n] for n, _ in _lib.Paged._fields_]))


def calls(kv, n_head=4):
    lib = _lib.load()
    yield lib.fhip_paged_append(kv, P, None, None, None, None, P, None, 1, n_head, 64, 0, 1e-6, 1e4, P, None)
    yield lib.fhip_paged_attention(kv, P, P, 64, n_head, 0, 0.0, P, P, None)
    yield lib.fhip_paged_attention_selected(kv, P, P, P, 4, n_head, 0.0, P, P, None)
    yield lib.fhip_paged_key_bounds(kv, P, None, 1, P, None)
    yield lib.fhip_paged_select(kv, P, P, 64, P, n_head, 4, 1, 1, P, P, None)
    yield lib.fhip_paged_rows(kv, 0, 0, 1, P, P, None)


@pytest.mark.parametrize("more,rc,text", [
    (dict(type=12), TYPE, "ggml type 12"), (dict(type=2), TYPE, "F32, F16, BF16 or Q8_0"),
    (dict(head_dim=96), SHAPE, "head_dim must be 64 or 128"), (dict(head_dim=0), SHAPE, "head_dim"),
    (dict(page_rows=8), SHAPE, "page_rows"), (dict(page_rows=48), SHAPE, "power of two"), (dict(page_rows=8192), SHAPE, "page_rows"), (dict(page_rows=0), SHAPE, "page_rows"),
    (dict(n_kv=0), SHAPE, "n_kv"), (dict(n_kv=4097), SHAPE, "n_kv"), (dict(n_seq=65536), SHAPE, "65535"), (dict(n_pages=2 ** 32 - 1), SHAPE, "pages"), (dict(n_pages=0), SHAPE, "pages"),
    (dict(pages_per_seq=2 ** 28, table_stride=2 ** 28), SHAPE, "2^32"), (dict(table_stride=3), SHAPE, "table_stride"),
    (dict(d_k=None), ARG, "pools"), (dict(d_v=P + 8), ARG, "16-byte"), (dict(type=8), ARG, "scales"), (dict(type=8, d_k_scales=P, d_v_scales=P + 2), ARG, "scales"),
    (dict(d_table=None), ARG, "table")])
def test_every_call_checks_the_description(more, rc, text):
    for got in calls(cache(**more)):
        assert got == rc
        assert text in _lib.last_error()
    lib = _lib.load()
    assert lib.fhip_paged_attention_ws_bytes(cache(**more), 4, 64) == 0 and lib.fhip_paged_select_ws_bytes(cache(**more), 64) == 0


def test_no_description():
    for got in calls(None):
        assert got == ARG and "NULL cache" in _lib.last_error()


@pytest.mark.parametrize("n_head", [0, 1, 3, 34])
def test_heads_that_the_cache_does_not_fit(n_head):
    got = list(calls(cache(), n_head))
    assert [got[i] for i in (0, 1, 2, 4)] == [SHAPE] * 4


def test_arguments():
    lib, kv = _lib.load(), cache()
    append = lambda qkv=P, pos=P, t=1, n_rot=64, base=1e4, q=P, bias=None: lib.fhip_paged_append(kv, qkv, bias, None, None, None, pos, None, t, 4, n_rot, 0, 1e-6, base, q, None)      # noqa: E731
    assert append(n_rot=63) == SHAPE and append(n_rot=66) == SHAPE and append(t=2 ** 31) == SHAPE
    assert append(qkv=None) == ARG and append(pos=None) == ARG and append(q=None) == ARG and append(q=P + 4) == ARG and append(bias=P + 4) == ARG
    assert append(base=0.0) == ARG and append(base=float("nan")) == ARG
    assert append(t=0, qkv=None) == OK                                       # nothing to do
    attend = lambda q=P, lens=P, out=P, cap=0.0, kv=kv, ws=P: lib.fhip_paged_attention(kv, q, lens, 64, 4, 0, cap, ws, out, None)      # noqa: E731
    assert attend(q=None) == ARG and attend(lens=None) == ARG and attend(out=None) == ARG and attend(q=P + 8) == ARG and attend(ws=P + 4) == ARG
    assert attend(cap=-1.0) == ARG and attend(cap=float("nan")) == ARG
    assert attend(kv=cache(n_seq=0), q=None) == OK
    assert lib.fhip_paged_attention(cache(n_seq=65535, n_kv=64), P, P, 64, 256, 0, 0.0, P, P, None) == SHAPE and "2^23" in _lib.last_error()
    picked = lambda sel=P, n=4: lib.fhip_paged_attention_selected(kv, P, P, sel, n, 4, 0.0, P, P, None)      # noqa: E731
    assert picked(sel=None) == ARG and picked(n=0) == SHAPE and picked(n=2 ** 20 + 1) == SHAPE
    choose = lambda n=4, first=1, last=1, ws=P, b=P, out=P: lib.fhip_paged_select(kv, P, P, 64, b, 4, n, first, last, ws, out, None)      # noqa: E731
    assert choose(n=0, first=0, last=0) == SHAPE and choose(n=2, first=2, last=1) == SHAPE and choose(first=2 ** 63, last=2 ** 63) == SHAPE
    assert choose(ws=None) == ARG and choose(b=None) == ARG and choose(out=None) == ARG and choose(b=P + 4) == ARG
    bounds = lambda lens=P, b=P, n=1: lib.fhip_paged_key_bounds(kv, lens, None, n, b, None)      # noqa: E731
    assert bounds(lens=None) == ARG and bounds(b=None) == ARG and bounds(n=0, b=None) == OK
    rows = lambda seq=0, r0=0, n=1, k=P: lib.fhip_paged_rows(kv, seq, r0, n, k, P, None)      # noqa: E731
    assert rows(seq=3) == SHAPE and rows(r0=64) == SHAPE and rows(r0=65, n=0) == SHAPE and rows(n=2 ** 64 - 1, r0=1) == SHAPE and rows(k=None) == ARG and rows(k=P + 4) == ARG
    assert rows(r0=64, n=0, k=None) == OK


def test_without_a_device_a_good_call_says_so():
    if _lib._inited:
        pytest.skip("device already initialised in this process")
    for got in calls(cache()):
        assert got == ARG and "fhip_init" in _lib.last_error()


def test_launches_of_more_than_2_32_threads():
    lib = _lib.load()
    assert lib.fhip_paged_append(cache(), P, None, None, None, None, P, None, 2 ** 25 + 1, 4, 64, 0, 1e-6, 1e4, P, None) == SHAPE and "2^25" in _lib.last_error()
    many = cache(n_seq=65535, n_kv=4096)
    assert lib.fhip_paged_select(many, P, P, 64, P, 4096, 4, 1, 1, P, P, None) == SHAPE and "2^22" in _lib.last_error()
    assert lib.fhip_paged_key_bounds(many, P, None, 1, P, None) == SHAPE and "2^22" in _lib.last_error()


def test_a_workspace_that_is_too_small(monkeypatch):
    from types import SimpleNamespace as N

    from ferric_amd import paged
    from ferric_amd.qmatrix import Tensor
    monkeypatch.setattr(_lib, "init", lambda *a: None)
    at = N(ptr=P)
    kv = paged.PagedKvCache.wrap(0, 16, 64, 2, 64, at, at, None, None, at, 1, 64)
    few, none = N(ptr=P, nbytes=16), N(ptr=P, nbytes=0)
    row, lens, bounds = Tensor(at, (1, 256)), Tensor(at, (1,)), Tensor(at, (64, 2, 2, 64))
    with pytest.raises(AssertionError, match="workspace of 16 bytes"):
        kv.attention(row, lens, 1024, 4, out=row, ws=few)
    with pytest.raises(AssertionError, match="workspace of 16 bytes"):
        kv.select(row, lens, 1024, bounds, 4, 4, out=Tensor(at, (1, 2, 4)), ws=few)
    with pytest.raises(AssertionError, match="workspace of 16 bytes"):
        kv.attention_selected(row, lens, Tensor(at, (1, 2, 40)), 4, out=row, ws=few)
    assert kv._workspace(4, 100, none, None) is none            # short: needs none
