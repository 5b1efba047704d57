"""Workspaces of the paged cache's attention: what the bound on the lengths has to do with their size. Sizes are the host's to work out, so no device is needed."""
import ctypes as C

import pytest

from ferric_amd import _lib

P = 0x1000      # no memory of anybody


def cache(**more):
    f = dict(type=30, page_rows=64, n_pages=4096, n_kv=8, head_dim=128, d_k=P, d_v=P, d_k_scales=P, d_v_scales=P, d_table=P, n_seq=2, pages_per_seq=2048, table_stride=2048)
    f.update(more)
    return C.byref(_lib.Paged(*[f[n] for n, _ in _lib.Paged._fields_]))


@pytest.mark.parametrize("ty", [0, 1, 30, 8])
@pytest.mark.parametrize("n_seq,n_kv", [(1, 1), (2, 8), (64, 8), (600, 1)])
@pytest.mark.parametrize("pages", [1, 5, 16, 100, 2048])
def test_a_bound_past_the_table_is_the_table_s_reach(ty, n_seq, n_kv, pages):
    lib, kv = _lib.load(), cache(type=ty, n_seq=n_seq, n_kv=n_kv, pages_per_seq=pages)
    at_reach = lib.fhip_paged_attention_ws_bytes(kv, n_kv, 64 * pages)
    for bound in (64 * pages + 1, 2 ** 31, 2 ** 32 - 1, 2 ** 40, 2 ** 64 - 1):
        assert lib.fhip_paged_attention_ws_bytes(kv, n_kv, bound) == at_reach


@pytest.mark.parametrize("ty", [0, 1, 30, 8])
@pytest.mark.parametrize("more", [dict(), dict(n_seq=1, n_kv=1), dict(n_seq=600), dict(n_seq=60000, n_kv=64), dict(page_rows=4096, pages_per_seq=2 ** 20 - 1, table_stride=2 ** 20)])
def test_a_workspace_for_a_bound_serves_every_smaller_one(ty, more):
    lib, kv, n_kv = _lib.load(), cache(type=ty, **more), more.get("n_kv", 8)
    sizes = [lib.fhip_paged_attention_ws_bytes(kv, n_kv, n) for n in [0, 1, 16, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 2047, 2048, 2049] + [2 ** e for e in range(12, 41)]]
    assert sizes == sorted(sizes)
