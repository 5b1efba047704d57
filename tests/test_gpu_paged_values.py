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


# ---- weights far apart --------------------------------------------------------------------------------------------------------------

def with_a_key_ahead(F, paged, ty, lens, n_kv, g, hd, gap, seed):
    """A cache in which one key of every sequence and KV head is `gap` nats (and a few) ahead of all others and has a value row of zeros, so that a result is what the others leave; and queries."""
    rng = np.random.default_rng(seed)
    case = Filled(F, paged, ty, lens, n_kv, hd, 32, seed)
    ahead = rng.standard_normal((n_kv, hd))
    ahead /= np.linalg.norm(ahead, axis=-1, keepdims=True)
    q = (rng.standard_normal((len(lens), n_kv, g, hd)) + 6 * ahead[:, None]).astype(np.float32)
    for i, n in enumerate(lens):
        first = int(rng.integers(n))
        put(case, "k", i, [first], ((gap + 4) * np.sqrt(hd) / 6 * ahead).reshape(1, -1).astype(np.float32))
        put(case, "v", i, [first], np.zeros((1, n_kv * hd), np.float32))
    return case, q.reshape(len(lens), -1)


@typed
@pytest.mark.parametrize("hd,n_kv,g", [(64, 2, 3), (128, 2, 5), (128, 1, 16)])
@pytest.mark.parametrize("gap", [6, 10, 14, 18, 25, 40, 75])
def test_weights_far_below_the_largest(F, paged, ty, hd, n_kv, g, gap):  # noqa: F811
    lens = [40, 33, 700, 3001]
    case, q = with_a_key_ahead(F, paged, ty, lens, n_kv, g, hd, gap, gap + hd)
    out = case.cache.attention(tensor(F, q), words(lens), max(lens), n_kv * g).to_vec()
    check_attention(case, out, q, n_kv * g, lambda i: range(lens[i]))


@typed
def test_weights_far_below_the_largest_over_chosen_pages(F, paged, ty):  # noqa: F811
    lens, n_kv, g, hd = [3001, 90], 2, 4, 128
    case, q = with_a_key_ahead(F, paged, ty, lens, n_kv, g, hd, 25, 3)
    pages = max(-(-n // case.R) for n in lens)
    listed = np.full((2, n_kv, pages), P.NO_PAGE, np.uint32)
    for i, n in enumerate(lens):
        listed[i, :, :-(-n // case.R)] = np.random.default_rng(i).permutation(-(-n // case.R))
    sel = F.Tensor(words(listed.reshape(-1)).buf, listed.shape, np.uint32)
    out = case.cache.attention_selected(tensor(F, q), words(lens), sel, n_kv * g).to_vec()
    check_attention(case, out, q, n_kv * g, lambda i: range(lens[i]))


@typed
@pytest.mark.parametrize("std", [3.0, 9.0])
def test_scores_of_a_wide_spread(F, paged, ty, std):  # noqa: F811
    """Weights of every size from the largest down to nothing, in every step."""
    lens = [1, 100, 513, 2000]
    case = Filled(F, paged, ty, lens, 2, 64, 16, 7)
    q = (std * np.random.default_rng(8).standard_normal((len(lens), 6 * 64))).astype(np.float32)
    out = case.cache.attention(tensor(F, q), words(lens), max(lens), 6).to_vec()
    check_attention(case, out, q, 6, lambda i: range(lens[i]))


# ---- a bound that says nothing ------------------------------------------------------------------------------------------------------

@typed
def test_no_bound_is_the_table_s_reach(F, paged, ty):  # noqa: F811
    """The same way of working, so the same bits: two sequences of eight KV heads, long enough that their steps are dealt out; over all rows and over chosen pages."""
    lens, n_kv, hd = [9000, 8000], 8, 64
    case = Filled(F, paged, ty, lens, n_kv, hd, 16, 1)
    reach = case.entries * 16
    q = np.random.default_rng(0).standard_normal((2, 2 * n_kv * hd)).astype(np.float32)
    qt, lt = tensor(F, q), words(lens)
    want = case.cache.attention(qt, lt, reach, 2 * n_kv).to_vec()
    check_attention(case, want, q, 2 * n_kv, lambda i: range(lens[i]))
    for bound in (2 ** 32 - 1, 2 ** 40):
        assert np.array_equal(case.cache.attention(qt, lt, bound, 2 * n_kv).to_vec().view(np.uint32), want.view(np.uint32))
    got = []
    for n in (case.entries, 300000):                           # (the list's rows are as many words apart)
        listed = np.full((2, n_kv, n), P.NO_PAGE, np.uint32)
        listed[:, :, :case.entries] = np.arange(case.entries)
        sel = F.Tensor(words(listed.reshape(-1)).buf, listed.shape, np.uint32)
        got.append(case.cache.attention_selected(qt, lt, sel, 2 * n_kv).to_vec())
    assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
    check_attention(case, got[0], q, 2 * n_kv, lambda i: range(lens[i]))


# ---- capped, extreme and infinite values --------------------------------------------------------------------------------------------

@typed
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cap", [0.5, 5.0, 30.0])
def test_scores_far_past_the_cap(F, paged, ty, hd, cap):  # noqa: F811
    """Where tanh has nearly reached one, and everything in front of that."""
    lens = [1, 33, 700]
    case = Filled(F, paged, ty, lens, 2, hd, 32, 9)
    q = (10 * np.random.default_rng(4).standard_normal((len(lens), 6 * hd))).astype(np.float32)
    out = case.cache.attention(tensor(F, q), words(lens), max(lens), 6, softcap=cap).to_vec()
    check_attention(case, out, q, 6, lambda i: range(lens[i]), cap)


@typed
def test_queries_of_every_size(F, paged, ty):  # noqa: F811
    """A query head is worked with at a power of two of its own on f16 and Q8_0 rows: heads from nothing to the largest, with keys of ordinary size and of such as bring the scores back."""
    lens, hd, sizes = [200, 1, 65], 128, [0.0, 1e-44, 1e-38, 1e-20, 1e-3, 1.0, 1e3, 3e38]
    for std in (1.0, 1e-3, 50.0):
        case = Filled(F, paged, ty, lens, 1, hd, 16, 11, std=std)
        q = np.random.default_rng(2).uniform(-1, 1, (len(lens), len(sizes), hd))
        q = (q * np.array(sizes)[:, None]).astype(np.float32)
        # scores past f32's largest are infinite in f32 arithmetic: the largest queries have one dim, against keys that are tiny there
        q[:, -1, 1:] = 0
        for i, n in enumerate(lens):
            k = case.values("k", i, range(n)).reshape(n, hd).astype(np.float32)
            k[:, 0] = 1e-6 * np.sign(k[:, 0])
            put(case, "k", i, range(n), k)
        q[:, -1, 0] *= 1e-31
        q = q.reshape(len(lens), -1)
        out = case.cache.attention(tensor(F, q), words(lens), max(lens), len(sizes)).to_vec()
        check_attention(case, out, q, len(sizes), lambda i: range(lens[i]), label=std)


@typed
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("far", [False, True])
def test_infinite_values_stay_in_their_dims(F, paged, ty, value, far):  # noqa: F811
    """An infinite value (Q8_0: a block's scale) makes its dim (block) of its KV head non-finite and nothing else, also where weights are far apart."""
    lens, n_kv, g, hd = [200, 33], 2, 3, 64
    case, q = with_a_key_ahead(F, paged, ty, lens, n_kv, g, hd, 25 if far else 1, 5)
    want = case.cache.attention(tensor(F, q), words(lens), max(lens), n_kv * g).to_vec().reshape(2, n_kv, g, hd)
    pool, scales = case.raw["v"]
    row = P.place(case.table[0], [77], case.R, case.n_pages)[0]
    if ty == P.Q8_0:
        scales[row, 1] = value                                 # KV head 0, dims 32 .. 63
        upload(case.cache.v_scales, scales)
    else:
        pool[row, 40] = P.bf16_bits(np.float32(value))[0] if ty == P.BF16 else value
        upload(case.cache.v, pool)
    out = case.cache.attention(tensor(F, q), words(lens), max(lens), n_kv * g).to_vec().reshape(2, n_kv, g, hd)
    hit = np.zeros(out.shape, bool)
    hit[0, 0, :, 32 if ty == P.Q8_0 else 40:64 if ty == P.Q8_0 else 41] = True
    assert not np.isfinite(out[hit]).any()
    # the same step may go another way (a scale that is no number): to f32 arithmetic's allowance, not to the bit
    q = q.reshape(2, n_kv * g, hd)
    for i, n in enumerate(lens):
        k, v = case.values("k", i, range(n)), case.values("v", i, range(n))
        v[~np.isfinite(v)] = 0
        _, tol = P.attend(q[i].astype(np.float64), k, v)
        keep = ~hit[i].reshape(n_kv * g, hd)
        assert (np.abs(out[i].reshape(n_kv * g, hd) - want[i].reshape(n_kv * g, hd))[keep] <= 2 * tol[keep]).all()


@typed
def test_a_key_that_is_no_number_makes_its_kv_head_s_results_none(F, paged, ty):  # noqa: F811
    lens, n_kv, g, hd = [200, 33], 2, 3, 128
    case = Filled(F, paged, ty, lens, n_kv, hd, 32, 6)
    q = np.random.default_rng(7).standard_normal((2, n_kv * g * hd)).astype(np.float32)
    want = case.cache.attention(tensor(F, q), words(lens), max(lens), n_kv * g).to_vec().reshape(2, n_kv, g, hd)
    pool, scales = case.raw["k"]
    row = P.place(case.table[0], [100], case.R, case.n_pages)[0]
    if ty == P.Q8_0:
        scales[row, hd // 32] = np.nan
        upload(case.cache.k_scales, scales)
    else:
        pool[row, hd + 5] = 0x7FC0 if ty == P.BF16 else np.nan
        upload(case.cache.k, pool)
    out = case.cache.attention(tensor(F, q), words(lens), max(lens), n_kv * g).to_vec().reshape(2, n_kv, g, hd)
    assert np.isnan(out[0, 1]).all()
    out[0, 1] = want[0, 1] = 0
    assert np.array_equal(out, want)


# ---- one cache on two streams -------------------------------------------------------------------------------------------------------

def test_one_cache_on_two_streams(F, paged):  # noqa: F811
    """A workspace for each: calls of one cache, dealt out and joined, with other queries and lengths on either stream."""
    lens = [[30000, 9000], [12000, 25000]]
    case = Filled(F, paged, P.BF16, [30000, 25000], 2, 128, 64, 1)
    streams, nh = [F.Stream(), F.Stream()], 8
    qs = [np.random.default_rng(i).standard_normal((2, nh * 128)).astype(np.float32) for i in range(2)]
    qt, lt = [tensor(F, q) for q in qs], [words(n) for n in lens]
    alone = [case.cache.attention(qt[i], lt[i], 30000, nh).to_vec() for i in range(2)]
    for i in range(2):
        case.lens = lens[i]
        check_attention(case, alone[i], qs[i], nh, lambda s, i=i: range(lens[i][s]))
        case.cache.reserve(nh, 30000, stream=streams[i])
    kept = [case.cache._workspace(nh, 30000, None, s) for s in streams]
    assert kept[0].ptr.value != kept[1].ptr.value and case.cache._workspace(nh, 30000, None, None).ptr.value not in (kept[0].ptr.value, kept[1].ptr.value)
    F._lib.check(F._lib.load().fhip_stream_sync(None))
    outs = [(i, case.cache.attention(qt[i], lt[i], 30000, nh, stream=streams[i])) for _ in range(20) for i in range(2)]
    for i, o in outs:
        assert np.array_equal(o.to_vec(streams[i]).view(np.uint32), alone[i].view(np.uint32))
