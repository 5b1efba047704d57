"""The paged cache's attention on rows whose values are far apart in size, against its definition in 64 bits: within paged_oracle.attend's allowance of f32 arithmetic, whatever
the rows are stored in."""
import numpy as np
import pytest

from oracle import paged_oracle as P
from test_gpu_paged import Filled, check_attention, paged, tensor, typed, upload, words  # noqa: F401

pytestmark = pytest.mark.gpu


def put(case, name, i, positions, rows):
    """f32 rows [n, n_kv * hd] into positions of sequence i."""
    pool, scales = P.encode(rows, case.ty)
    at = P.place(case.table[i], positions, case.R, case.n_pages)
    case.raw[name][0][at] = pool
    if scales is not None:
        case.raw[name][1][at] = scales
    upload(getattr(case.cache, name), case.raw[name][0])
    if scales is not None:
        upload(getattr(case.cache, name + "_scales"), case.raw[name][1])


# ---- Q8_0 blocks of very different scales -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,n_kv,g", [(64, 2, 3), (128, 2, 5), (128, 1, 1)])
def test_large_scales_beside_small_ones(F, paged, hd, n_kv, g):  # noqa: F811
    """Values of 1e5 and more (scales past 512, whose products with a code leave f16) in the last block of a row in ten, values of 1e-5 .. 1 in its other blocks; and rows of large values
    throughout, 40 nats behind the others."""
    lens, rng = [1, 40, 33, 700, 3001], np.random.default_rng(hd + g)
    case = Filled(F, paged, P.Q8_0, lens, n_kv, hd, 32, hd)
    q = (1.5 * rng.standard_normal((len(lens), n_kv, g, hd))).astype(np.float32)
    ahead = rng.standard_normal((n_kv, hd))
    ahead /= np.linalg.norm(ahead, axis=-1, keepdims=True)
    q += 6 * ahead[:, None].astype(np.float32)
    for i, n in enumerate(lens):
        v = rng.standard_normal((n, n_kv, hd // 32, 32))
        v[:, :, :-1] *= np.array([1e-5, 1e-3, 1.0])[:hd // 32 - 1, None]
        v[rng.random((n, n_kv)) < 0.1, -1] *= 1e5
        k = rng.standard_normal((n, n_kv, hd))
        if n > 20:
            far = rng.permutation(n)[:2]
            v[far] = 1e5 * rng.standard_normal(v[far].shape)
            k[far] = -40 * np.sqrt(hd) / 6 * ahead
        put(case, "v", i, range(n), v.reshape(n, -1).astype(np.float32))
        put(case, "k", i, range(n), k.reshape(n, -1).astype(np.float32))
    big = case.raw["v"][1][np.isfinite(case.raw["v"][1])]
    assert (big >= 512).any() and (big < 1e-6).any()
    q = q.reshape(len(lens), -1)
    out = case.cache.attention(tensor(F, q), words(lens), max(lens), n_kv * g).to_vec()
    check_attention(case, out, q, n_kv * g, lambda i: range(lens[i]))
