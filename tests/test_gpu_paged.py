"""The paged key/value cache on the GPU against its definitions in 64 bits (oracle/paged_oracle.py), through the package's own class and the C ABI.

Tolerances are counted roundings: see paged_oracle.attend for the attention's and `post_error` for the stored rows'."""
import ctypes as C

import numpy as np
import pytest

from conftest import bits
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
TYPES = [P.F32, P.F16, P.BF16, P.Q8_0]
NAMES = {P.F32: "f32", P.F16: "f16", P.BF16: "bf16", P.Q8_0: "q8_0"}
typed = pytest.mark.parametrize("ty", TYPES, ids=[NAMES[t] for t in TYPES])


@pytest.fixture(scope="module")
def paged(F):
    from ferric_amd import paged
    return paged


def words(values):
    from ferric_amd.decode import _u32_tensor
    return _u32_tensor(np.asarray(values, np.uint32))


def tensor(F, a):
    a = np.ascontiguousarray(a, np.float32)
    return F.Tensor.from_vec(a, a.shape)


def upload(buf, a):
    from ferric_amd.qmatrix import _arrived, _upload
    a = np.ascontiguousarray(a)
    _upload(buf, a)
    _arrived(a)


def download(F, buf, dtype, n):
    out = np.empty(n, dtype)
    F._lib.check(F._lib.load().fhip_memcpy_d2h(out.ctypes.data, buf.ptr, out.nbytes, None))
    return out


POOL = {P.F32: np.float32, P.F16: np.float16, P.BF16: np.uint16, P.Q8_0: np.int8}


class Filled:
    """A cache whose pools hold `lens` rows of random values; what no sequence has is NaN (Q8_0: NaN scales), and entries of the table without a row name no page."""

    def __init__(self, F, paged, ty, lens, n_kv, hd, R, seed, extra_entries=1, std=1.0):
        rng = np.random.default_rng(seed)
        self.F, self.ty, self.lens, self.n_kv, self.hd, self.R = F, ty, list(lens), n_kv, hd, R
        need = [-(-n // R) for n in lens]
        self.entries = max(need + [1]) + extra_entries
        self.n_pages = sum(need) + 2
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.entries), P.NO_PAGE, np.uint32)
        self.table[:, -1] = self.n_pages                       # the first number past the pool
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.cache = paged.PagedKvCache(ty, R, self.n_pages, n_kv, hd, len(lens), self.entries)
        self.cache.set_table(self.table)
        rows, width = self.n_pages * R, n_kv * hd
        live = np.zeros(rows, bool)
        for i, n in enumerate(lens):
            live[P.place(self.table[i], range(n), R, self.n_pages)] = True
        self.raw = {}
        for name in "kv":
            pool, scales = P.encode((std * rng.standard_normal((rows, width))).astype(np.float32), ty)
            if ty == P.Q8_0:
                scales[~live] = np.nan
            else:
                pool[~live] = 0x7FC0 if ty == P.BF16 else np.nan
            self.raw[name] = (pool, scales)
            upload(getattr(self.cache, name), pool)
            if scales is not None:
                upload(getattr(self.cache, name + "_scales"), scales)

    def values(self, name, i, positions):
        pool, scales = self.raw[name]
        at = P.place(self.table[i], positions, self.R, self.n_pages)
        at = at[at >= 0]
        return P.decode(pool[at], None if scales is None else scales[at], self.ty).reshape(len(at), self.n_kv, self.hd)

    def stored(self, name):
        """(pool words, scales) as they are on the device now."""
        pool, scales = self.raw[name]
        got = download(self.F, getattr(self.cache, name), POOL[self.ty], pool.size).reshape(pool.shape)
        return got, None if scales is None else download(self.F, getattr(self.cache, name + "_scales"), np.float16, scales.size).reshape(scales.shape)


def check_attention(case, out, q, n_head, positions_of, softcap=0.0, label=""):
    hd = case.hd
    out, q = out.reshape(-1, n_head, hd), q.reshape(-1, n_head, hd)
    for i in range(len(case.lens)):
        at = positions_of(i)
        k, v = case.values("k", i, at), case.values("v", i, at)
        want, tol = P.attend(q[i].astype(np.float64), k, v, softcap) if len(k) else (np.zeros((n_head, hd)), np.zeros((n_head, hd)))
        assert np.isfinite(out[i]).all(), (label, i, len(at))
        err = np.abs(out[i] - want)
        assert (err <= tol).all(), (label, i, len(at), err.max(), tol[np.unravel_index((err - tol).argmax(), err.shape)])


# ---- attention ------------------------------------------------------------------------------------------------------------------

RAGGED = [1, 0, 15, 16, 17, 33, 64, 65, 200, 511, 513, 1000]


@typed
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_kv,g", [(1, 16), (2, 5), (3, 1), (2, 8), (1, 3)])
def test_attention_over_ragged_sequences(F, paged, ty, hd, n_kv, g):
    case = Filled(F, paged, ty, RAGGED, n_kv, hd, 32, 11 * hd + g)
    q = (1.5 * np.random.default_rng(g).standard_normal((len(RAGGED), n_kv * g * hd))).astype(np.float32)
    out = case.cache.attention(tensor(F, q), words(RAGGED), max(RAGGED), n_kv * g).to_vec()
    check_attention(case, out, q, n_kv * g, lambda i: range(RAGGED[i]))


@typed
@pytest.mark.parametrize("R", [16, 64, 256, 4096])
def test_attention_by_page_size(F, paged, ty, R):
    lens = [R - 1, R, R + 1, 3, 700]
    case = Filled(F, paged, ty, lens, 2, 64, R, R)
    q = np.random.default_rng(R).standard_normal((5, 4 * 64)).astype(np.float32)
    out = case.cache.attention(tensor(F, q), words(lens), max(lens), 4).to_vec()
    check_attention(case, out, q, 4, lambda i: range(lens[i]))


@typed
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (16, 0.0), (100, 30.0), (10 ** 6, 0.0), (0, 20.0), (513, 50.0)])
def test_window_and_softcap(F, paged, ty, window, softcap):
    case = Filled(F, paged, ty, RAGGED, 2, 128, 16, window % 97)
    q = (3 * np.random.default_rng(5).standard_normal((len(RAGGED), 6 * 128))).astype(np.float32)
    out = case.cache.attention(tensor(F, q), words(RAGGED), max(RAGGED), 6, window=window, softcap=softcap).to_vec()
    check_attention(case, out, q, 6, lambda i: range(max(0, RAGGED[i] - (window or RAGGED[i])), RAGGED[i]), softcap)


@typed
@pytest.mark.parametrize("n_seq,n_kv", [(1, 1), (1, 8), (3, 2)])
def test_long_sequences(F, paged, ty, n_seq, n_kv):
    lens = [20011, 7000, 12345][:n_seq]
    case = Filled(F, paged, ty, lens, n_kv, 128, 64, 3)
    q = (2 * np.random.default_rng(6).standard_normal((n_seq, n_kv * 4 * 128))).astype(np.float32)
    out = case.cache.attention(tensor(F, q), words(lens), max(lens), 4 * n_kv).to_vec()
    check_attention(case, out, q, 4 * n_kv, lambda i: range(lens[i]))


@typed
@pytest.mark.parametrize("n_seq,most,window", [(150, 3000, 0), (70, 2500, 700), (300, 2000, 0), (600, 100, 0), (130, 40, 0)])
def test_many_sequences(F, paged, ty, n_seq, most, window):
    """More sequences than a wave has lanes, long ones among many short and empty ones; more units than the chip has workgroups and waves for."""
    rng = np.random.default_rng(n_seq)
    lens = [int(x) for x in rng.integers(0, 40, n_seq)]
    for i in rng.integers(0, n_seq, 5):
        lens[i] = int(rng.integers(most // 2, most + 1))
    lens[-1] = most
    case = Filled(F, paged, ty, lens, 2, 64, 16, n_seq, extra_entries=0)
    q = (1.5 * rng.standard_normal((n_seq, 4 * 64))).astype(np.float32)
    out = case.cache.attention(tensor(F, q), words(lens), most, 4, window=window).to_vec()
    check_attention(case, out, q, 4, lambda i: range(max(0, lens[i] - (window or lens[i])), lens[i]))


def test_lengths_are_cut_to_the_bound_and_to_the_table(F, paged):
    case = Filled(F, paged, P.F32, [100, 100, 40], 2, 64, 16, 9, extra_entries=0)
    q = np.random.default_rng(1).standard_normal((3, 4 * 64)).astype(np.float32)
    for said, bound, lens in (([100, 77, 40], 50, [50, 50, 40]), ([2 ** 32 - 1, 10 ** 6, 0], 2 ** 40, [112, 112, 0])):
        if bound > 100:      # rows 100 .. 111 of the last page are NaN: give them values, as they now count
            for name in "kv":
                pool = case.raw[name][0]
                pool[np.isnan(pool)] = 0.25
                upload(getattr(case.cache, name), pool)
        out = case.cache.attention(tensor(F, q), words(said), bound, 4).to_vec()
        check_attention(case, out, q, 4, lambda i: range(lens[i]))


def test_rows_without_a_page_are_left_out(F, paged):
    lens = [200, 90, 33]
    case = Filled(F, paged, P.BF16, lens, 2, 128, 16, 21)
    case.table[0, 2] = P.NO_PAGE
    case.table[0, 12] = case.n_pages
    case.table[2, :] = 0x80000000
    case.cache.set_table(case.table)
    q = np.random.default_rng(2).standard_normal((3, 10 * 128)).astype(np.float32)
    out = case.cache.attention(tensor(F, q), words(lens), 200, 10).to_vec()
    check_attention(case, out, q, 10, lambda i: range(lens[i]))
    assert not out.reshape(3, -1)[2].any()                     # no row left: zeros


def test_a_batch_row_has_the_same_bits_on_every_run_and_large_scores_hold(F, paged):
    lens = [3000, 17, 1025]
    case = Filled(F, paged, P.F32, lens, 2, 64, 32, 4, std=30.0)   # scores of hundreds: the maximum matters
    q = (8 * np.random.default_rng(3).standard_normal((3, 4 * 64))).astype(np.float32)
    a = case.cache.attention(tensor(F, q), words(lens), 3000, 4).to_vec()
    for _ in range(3):
        assert np.array_equal(bits(a), bits(case.cache.attention(tensor(F, q), words(lens), 3000, 4).to_vec()))
    check_attention(case, a, q, 4, lambda i: range(lens[i]))


def test_sequences_may_share_pages_and_the_table_may_be_wider(F, paged):
    lens = [64, 80, 80]
    case = Filled(F, paged, P.F16, [64, 80, 80], 2, 64, 16, 31)
    case.table[1, :4] = case.table[0, :4]                      # a common prefix of 64 rows
    wide = np.full((3, 9), 12345, np.uint32)
    wide[:, :case.entries] = case.table
    buf = F.DeviceBuffer(wide.nbytes)
    upload(buf, wide)
    d = F._lib.Paged.from_buffer_copy(case.cache._desc)
    d.d_table, d.table_stride = buf.ptr.value, 9
    q = np.random.default_rng(8).standard_normal((3, 8 * 64)).astype(np.float32)
    qt, lt, out, lib = tensor(F, q), words(lens), F.Tensor.empty((3, 8 * 64)), F._lib.load()
    ws = F.DeviceBuffer(max(16, lib.fhip_paged_attention_ws_bytes(C.byref(d), 8, 80)))
    F._lib.check(lib.fhip_paged_attention(C.byref(d), qt.buf.ptr, lt.buf.ptr, 80, 8, 0, 0.0, ws.ptr, out.buf.ptr, None))
    check_attention(case, out.to_vec(), q, 8, lambda i: range(lens[i]))


@pytest.mark.parametrize("ty", [P.BF16, P.Q8_0], ids=["bf16", "q8_0"])
def test_pools_past_four_gigavalues(F, paged, ty):
    """Pages at the far end of a pool of more than 2^32 values: stored, read back and attended to."""
    n_kv, hd, R = 8, 128, 256
    n_pages = (2 ** 32 + 2 ** 24) // (n_kv * hd * R)
    cache = paged.PagedKvCache(ty, R, n_pages, n_kv, hd, 1, 2)
    cache.set_table([[n_pages - 1, n_pages - 3]])
    t, rng = 300, np.random.default_rng(0)
    qkv = rng.standard_normal((t, (8 + 16) * hd)).astype(np.float32)
    q = cache.append(tensor(F, qkv), words([0] * t), words(range(t)), 8, 1e4, n_rot=0)
    k, v = (x.to_vec().reshape(t, n_kv, hd) for x in cache.rows(0, 0, t))
    stored = [P.decode(*P.encode(qkv[:, (8 + 8 * i) * hd:(16 + 8 * i) * hd], ty), ty).reshape(t, n_kv, hd) for i in range(2)]
    assert np.array_equal(k, stored[0]) and np.array_equal(v, stored[1])
    newest = F.Tensor.from_vec(q.to_vec().reshape(t, -1)[-1:], (1, 8 * hd))
    out = cache.attention(newest, words([t]), t, 8).to_vec().reshape(8, hd)
    want, tol = P.attend(qkv[-1, :8 * hd].reshape(8, hd).astype(np.float64), *stored)
    assert (np.abs(out - want) <= tol).all()


# ---- storing rows ---------------------------------------------------------------------------------------------------------------

def post_error(x, hd):
    """What f32 arithmetic may put between a post-processed value and its definition: the sum of squares of a head in a tree (8 roundings), its root and reciprocal (4), the bias,
    two products, the rotation's product and sum (5), and a turn rounded to 2^-25 of itself with its sine (2 pi / 2 + 4 units of 2^-24): under 32 roundings of the pair's length."""
    return 32 * 2.0 ** -24 * np.abs(x).max(-1, keepdims=True) * np.sqrt(2)


def check_stored(case, name, i, pos, want, q8_exact=None):
    """The rows of token positions `pos` of sequence i in the pool are `want` [n, kv, hd], rounded once."""
    pool, scales = case.stored(name)
    at = P.place(case.table[i], pos, case.R, case.n_pages)
    got = P.decode(pool[at], None if scales is None else scales[at], case.ty).reshape(want.shape)
    err = post_error(want, case.hd)
    if case.ty == P.Q8_0:
        d = np.abs(want).reshape(*want.shape[:-1], -1, 32).max(-1) / 127
        # half a code, a code times the scale's rounding to f16, and the value's own error
        tol = np.repeat(d * (0.5 + 127 * 2.0 ** -11 + 1e-3), 32, -1) + 2 * err
    else:
        tol = (np.abs(want) + err) * P.HALF_STEP[case.ty] + err + 2.0 ** -24 * (case.ty == P.F16)
    assert (np.abs(got - want) <= tol).all(), (name, i)


def untouched(case, name, written):
    pool, scales = case.stored(name)
    keep = np.ones(len(pool), bool)
    keep[written] = False
    assert np.array_equal(pool[keep].view(np.uint8), case.raw[name][0][keep].view(np.uint8))
    if scales is not None:
        assert np.array_equal(scales[keep].view(np.uint16), case.raw[name][1][keep].view(np.uint16))


@typed
@pytest.mark.parametrize("hd,n_kv,g,n_rot,inter,norm,bias", [(128, 2, 5, 128, False, True, True), (64, 3, 1, 64, False, True, False), (64, 1, 4, 32, True, False, True),
                                                             (128, 1, 2, 64, False, False, False), (64, 2, 3, 22, False, True, True), (128, 2, 1, 0, False, True, False),
                                                             (128, 1, 16, 128, True, True, True), (64, 1, 1, 2, False, False, False)])
@pytest.mark.parametrize("t", [1, 7, 1100])
def test_append(F, paged, ty, hd, n_kv, g, n_rot, inter, norm, bias, t):
    nh, R, rng = n_kv * g, 32, np.random.default_rng(t + hd + n_rot)
    # positions in any order; more rows than a sequence has pages for have no place
    case = Filled(F, paged, ty, [500, 64, 700], n_kv, hd, R, 5)
    seqs = rng.integers(0, 3, t).astype(np.uint32)
    pos = np.zeros(t, np.uint32)
    for i in range(3):
        pos[seqs == i] = rng.permutation(case.lens[i] if (seqs == i).sum() <= case.lens[i] else 10 ** 4)[:(seqs == i).sum()]
    qkv = (2 * rng.standard_normal((t, (nh + 2 * n_kv) * hd))).astype(np.float32)
    opt = {}
    if bias:
        opt["bias"] = rng.standard_normal(qkv.shape[1]).astype(np.float32)
    if norm:
        opt["q_norm"], opt["k_norm"] = (rng.uniform(0.5, 1.5, hd).astype(np.float32) for _ in range(2))
    if n_rot:
        opt["freq_scale"] = rng.uniform(0.5, 1.0, n_rot // 2).astype(np.float32)
    q = case.cache.append(tensor(F, qkv), words(seqs), words(pos), nh, 1e6, n_rot=n_rot, interleaved=inter, eps=1e-5, **{k: tensor(F, v) for k, v in opt.items()})
    wq, wk, wv = P.post(qkv, pos, nh, n_kv, hd, n_rot, inter, 1e6, 1e-5, **opt)
    got = q.to_vec().reshape(wq.shape)
    assert (np.abs(got - wq) <= post_error(wq, hd)).all()
    written = []
    for i in range(3):
        mine = np.flatnonzero(seqs == i)
        at = P.place(case.table[i], pos[mine], R, case.n_pages)
        mine, at = mine[at >= 0], at[at >= 0]
        written += list(at)
        if len(mine):
            check_stored(case, "k", i, pos[mine], wk[mine])
            check_stored(case, "v", i, pos[mine], wv[mine])
    untouched(case, "k", written), untouched(case, "v", written)


@pytest.mark.parametrize("inter", [False, True])
def test_dims_behind_the_rotated_ones_pass_through(F, paged, inter):
    """Each by itself: an infinite neighbour stays its own."""
    hd, t = 64, 3
    cache = paged.PagedKvCache(P.F32, 16, 1, 1, hd, 1, 1)
    cache.set_table([[0]])
    qkv = np.random.default_rng(2).standard_normal((t, 3 * hd)).astype(np.float32)
    qkv[1, 41], qkv[2, 63] = np.inf, np.nan
    q = cache.append(tensor(F, qkv), words([0] * t), words(range(t)), 1, 1e4, n_rot=32, interleaved=inter).to_vec().reshape(t, hd)
    assert np.array_equal(bits(q[:, 32:]), bits(qkv[:, 32:64]))
    assert np.isfinite(q[:, :32]).all()


def test_far_positions_turn_exactly(F, paged):
    """Angles in f64: at position 4 000 000 000 an f32 product is off by whole turns."""
    hd, R = 128, 4096
    pos = np.array([100000, 4000000, 2 ** 31 + 5, 4000000000], np.uint32)
    cache = paged.PagedKvCache(P.F32, R, 1, 1, hd, 4, 1)
    qkv = np.random.default_rng(1).standard_normal((4, 3 * hd)).astype(np.float32)
    q = cache.append(tensor(F, qkv), words(range(4)), words(pos), 1, 1e4).to_vec().reshape(4, 1, hd)
    want, _, _ = P.post(qkv, pos, 1, 1, hd, hd, False, 1e4, 1e-6)
    # the frequency's exponential, its factor and the product, there and in the definition: six roundings of 2^-53 of 4e9 rad, 2.7e-6
    assert (np.abs(q - want) <= post_error(want, hd) + 4e-6 * np.abs(want).max(-1, keepdims=True)).all()


def test_rows_that_have_no_place_leave_their_query_only(F, paged):
    case = Filled(F, paged, P.BF16, [40, 40], 1, 64, 16, 2)
    case.table[1, 1] = case.n_pages + 7
    case.cache.set_table(case.table)
    seqs = np.array([0, 2, 1, 2 ** 32 - 1, 0, 1], np.uint32)
    pos = np.array([5, 5, 20, 3, 2 ** 32 - 1, 3], np.uint32)    # none of sequence 2 or 2^32 - 1; 20 lies in an entry that is no page; the last position of all
    qkv = np.random.default_rng(4).standard_normal((6, 4 * 64)).astype(np.float32)
    q = case.cache.append(tensor(F, qkv), words(seqs), words(pos), 2, 1e4, n_rot=0).to_vec().reshape(6, 128)
    assert np.array_equal(q, qkv[:, :128])
    written = [P.place(case.table[0], [5], 16, case.n_pages)[0], P.place(case.table[1], [3], 16, case.n_pages)[0]]
    pool, _ = case.stored("k")
    assert np.array_equal(pool[written], P.bf16_bits(qkv[[0, 5], 128:192]))
    untouched(case, "k", written), untouched(case, "v", written)


def test_a_token_has_the_same_bits_in_every_batch_and_q8_blocks_are_kvq_append_s(F, paged):
    from ferric_amd import kvquant
    n_kv, hd, nh, t, R = 2, 128, 6, 1300, 64
    rng = np.random.default_rng(7)
    qkv = rng.standard_normal((t, (nh + 2 * n_kv) * hd)).astype(np.float32)
    norms = {k: tensor(F, rng.uniform(0.5, 1.5, hd)) for k in ("q_norm", "k_norm")}
    entries = -(-t // R)
    made = {}
    for ty in (P.F32, P.Q8_0):
        many, one = (paged.PagedKvCache(ty, R, entries, n_kv, hd, 1, entries) for _ in range(2))
        for c in (many, one):
            c.set_table(np.arange(entries, dtype=np.uint32)[None])
        q = many.append(tensor(F, qkv), words([0] * t), words(range(t)), nh, 5e5, **norms).to_vec().reshape(t, -1)
        for i in (0, 1, 700, t - 1):
            qi = one.append(tensor(F, qkv[i:i + 1]), None, words([i]), nh, 5e5, **norms).to_vec()
            assert np.array_equal(bits(qi), bits(q[i]))
            for name in (0, 1):
                assert np.array_equal(bits(one.rows(0, i, 1)[name].to_vec()), bits(many.rows(0, i, 1)[name].to_vec()))
        made[ty] = many
    for name, rows in zip("kv", made[P.F32].rows(0, 0, t)):
        want = kvquant.QKvCache.from_tensor(rows, kvquant.Q8_0)
        codes, scales = want.to_host()
        assert np.array_equal(download(F, getattr(made[P.Q8_0], name), np.uint32, codes.size), codes)
        assert np.array_equal(download(F, getattr(made[P.Q8_0], name + "_scales"), np.uint16, 2 * scales.size), scales.view(np.uint16))


# ---- rows read back -------------------------------------------------------------------------------------------------------------

@typed
@pytest.mark.parametrize("hd,n_kv", [(64, 1), (128, 3)])
@pytest.mark.parametrize("row0,rows", [(0, 1), (0, 300), (37, 200), (299, 1), (16, 16), (5, 0)])
def test_rows(F, paged, ty, hd, n_kv, row0, rows):
    case = Filled(F, paged, ty, [300, 20], n_kv, hd, 16, row0)
    for name, got in zip("kv", case.cache.rows(0, row0, rows)):
        if rows:
            want = case.values(name, 0, range(row0, row0 + rows)).reshape(rows, -1)
            assert np.array_equal(got.to_vec().reshape(rows, -1), want.astype(np.float32))     # every type's values are f32 values (Q8_0: 8 by 11 bits)


def test_rows_without_a_page_stay_as_they_were(F, paged):
    case = Filled(F, paged, P.F32, [64], 1, 64, 16, 1)
    case.table[0, 1] = P.NO_PAGE
    case.cache.set_table(case.table)
    out = tuple(tensor(F, np.full((64, 64), 7.0)) for _ in range(2))
    k, _ = case.cache.rows(0, 0, 64, out=out)
    k = k.to_vec().reshape(64, 64)
    assert (k[16:32] == 7).all()
    assert np.array_equal(np.delete(k, range(16, 32), 0), case.values("k", 0, range(64)).reshape(48, 64))


# ---- key bounds and the choice of pages ---------------------------------------------------------------------------------------

def bounds_of(case, i, n, R):
    """[pages, kv, 2, hd] of the first n rows of sequence i."""
    k = case.values("k", i, range(n))
    pages = -(-n // R)
    return np.stack([np.stack([k[p * R:min(n, (p + 1) * R)].min(0), k[p * R:min(n, (p + 1) * R)].max(0)], 1) for p in range(pages)]) if pages else np.zeros((0, case.n_kv, 2, case.hd))


@typed
@pytest.mark.parametrize("hd", [64, 128])
def test_key_bounds_grow_with_the_rows(F, paged, ty, hd):
    R, lens = 16, [100, 1, 16, 17, 0]
    case = Filled(F, paged, ty, lens, 2, hd, R, hd)
    bounds = tensor(F, np.full((case.n_pages, 2, 2, hd), 77.0))
    for now, new, most in (([40, 1, 10, 0, 0], [40, 1, 10, 0, 9], 40), ([41, 1, 11, 1, 0], None, 1), ([100, 1, 16, 17, 0], [59, 0, 5, 16, 0], 64)):
        case.cache.key_bounds(words(now), most, bounds, fresh=None if new is None else words(new))
        got = bounds.to_vec().reshape(case.n_pages, 2, 2, hd)
        if new is None:
            continue      # a sequence that did not grow had its newest row taken again, which changes nothing
        for i, n in enumerate(now):
            assert np.array_equal(got[case.table[i, :-(-n // R)]], bounds_of(case, i, n, R).astype(np.float32)), (now, i)
    used = np.concatenate([case.table[i, :-(-n // R)] for i, n in enumerate(lens)])
    rest = np.setdiff1d(np.arange(case.n_pages), used)
    assert (got[rest] == 77).all()                             # pages of nobody stay as they were


def test_key_bounds_of_a_long_prompt(F, paged):
    """Many pages at once, from the middle of one on."""
    n, R = 5000, 64
    case = Filled(F, paged, P.F16, [n], 1, 64, R, 8)
    bounds = tensor(F, np.zeros((case.n_pages, 1, 2, 64)))
    case.cache.key_bounds(words([37]), 37, bounds)
    case.cache.key_bounds(words([n]), n - 37, bounds)
    got = bounds.to_vec().reshape(case.n_pages, 1, 2, 64)
    assert np.array_equal(got[case.table[0, :-(-n // R)]], bounds_of(case, 0, n, R).astype(np.float32))


def test_nan_keys_make_nan_bounds_and_come_first(F, paged):
    case = Filled(F, paged, P.F32, [160], 1, 64, 16, 3)
    pool = case.raw["k"][0]
    pool[P.place(case.table[0], [70], 16, case.n_pages)[0], 9] = np.nan
    upload(case.cache.k, pool)
    bounds = case.cache.empty_bounds()
    case.cache.key_bounds(words([160]), 160, bounds)
    b = bounds.to_vec().reshape(case.n_pages, 2, 64)[case.table[0, 4]]
    assert np.isnan(b[:, 9]).all() and np.isfinite(np.delete(b, 9, 1)).all()
    q = tensor(F, np.random.default_rng(0).standard_normal((1, 64)))
    got = case.cache.select(q, words([160]), 160, bounds, 1, 3, first=1, last=1).to_vec()
    assert list(got) == [0, 4, 9]


@pytest.mark.parametrize("hd,n_kv,g", [(64, 1, 1), (128, 2, 5), (64, 3, 16), (128, 1, 3)])
@pytest.mark.parametrize("n_select,first,last", [(1, 0, 0), (4, 1, 1), (7, 0, 2), (64, 2, 1), (300, 1, 1)])
def test_select(F, paged, hd, n_kv, g, n_select, first, last):
    R, lens = 16, [3000, 0, 1, 160, 700, 113, 64]
    case = Filled(F, paged, P.F32, lens, n_kv, hd, R, g)
    # bounds that are nobody's keys: the choice goes by them alone; some equal to others, so that places decide
    rng = np.random.default_rng(n_select)
    b = np.sort(rng.standard_normal((case.n_pages, n_kv, 2, hd)).astype(np.float32), axis=2)
    for i in (0, 4):
        pages = case.table[i, :-(-lens[i] // R)]
        b[pages[5::3]] = b[pages[5]]
    q = rng.standard_normal((len(lens), n_kv * g * hd)).astype(np.float32)
    got = case.cache.select(tensor(F, q), words(lens), max(lens), tensor(F, b), n_kv * g, n_select, first=first, last=last).to_vec().reshape(len(lens), n_kv, n_select)
    for i, n in enumerate(lens):
        want = P.select(q[i].reshape(-1, hd), b[case.table[i, :-(-n // R)]], n_kv, n_select, first, last)
        assert np.array_equal(got[i], want), (i, n)


def test_select_among_very_many_pages(F, paged):
    R, n = 16, 16 * 20000 + 3
    rng = np.random.default_rng(0)
    cache = paged.PagedKvCache(P.BF16, R, 20001, 1, 64, 1, 20001)
    cache.set_table(rng.permutation(20001).astype(np.uint32)[None])
    table = download(F, cache.table, np.uint32, 20001)
    b = np.sort(rng.standard_normal((20001, 1, 2, 64)).astype(np.float32), axis=2)
    b[5000:9000] *= 1e-3                                       # scores of very different size
    q = rng.standard_normal((1, 2 * 64)).astype(np.float32)
    got = cache.select(tensor(F, q), words([n]), n, tensor(F, b), 2, 777, first=3, last=2).to_vec()
    assert np.array_equal(got, P.select(q.reshape(2, 64), b[table], 1, 777, 3, 2)[0])


@typed
@pytest.mark.parametrize("R,n_select", [(16, 5), (64, 3), (16, 40)])
def test_attention_over_selected_pages(F, paged, ty, R, n_select):
    lens, n_kv, g, hd = [700, 0, 1, 90, 333], 2, 5, 128
    case = Filled(F, paged, ty, lens, n_kv, hd, R, n_select)
    rng = np.random.default_rng(R)
    q = (1.5 * rng.standard_normal((5, n_kv * g * hd))).astype(np.float32)
    sel = np.full((5, n_kv, n_select), P.NO_PAGE, np.uint32)
    for i, n in enumerate(lens):
        pages = -(-n // R)
        for h in range(n_kv):
            chosen = rng.permutation(pages)[:n_select]          # in any order
            sel[i, h, :len(chosen)] = chosen
    sel[4, 1, 1] = -(-lens[4] // R)                             # the page behind the sequence's last: left out
    out = case.cache.attention_selected(tensor(F, q), words(lens), F.Tensor(words(sel.reshape(-1)).buf, sel.shape, np.uint32), n_kv * g, softcap=25.0).to_vec().reshape(5, n_kv, g, hd)
    for i, n in enumerate(lens):
        for h in range(n_kv):
            at = [p for e in sel[i, h] if e < -(-n // R) for p in range(int(e) * R, min(n, int(e + 1) * R))]
            k, v = case.values("k", i, at)[:, h:h + 1], case.values("v", i, at)[:, h:h + 1]
            want, tol = P.attend(q[i].reshape(n_kv, g, hd)[h].astype(np.float64), k, v, 25.0) if at else (np.zeros((g, hd)), np.zeros((g, hd)))
            assert (np.abs(out[i, h] - want) <= tol).all(), (i, h)


# ---- together -------------------------------------------------------------------------------------------------------------------

def test_a_prompt_in_two_blocks_then_tokens(F, paged):
    """Two sequences of a server: prompts appended (one in two blocks, the second behind its cached prefix), then tokens of both together, over all rows and over chosen pages."""
    from ferric_amd import decode
    n_kv, hd, nh, R, rng = 2, 128, 8, 16, np.random.default_rng(12)
    cache = paged.PagedKvCache(P.F32, R, 24, n_kv, hd, 2, 12)
    cache.set_table(rng.permutation(24).astype(np.uint32).reshape(2, 12))
    lens, steps = [150, 37], 5
    qkv = [rng.standard_normal((n + steps, (nh + 2 * n_kv) * hd)).astype(np.float32) for n in lens]
    post = [P.post(x, np.arange(len(x)), nh, n_kv, hd, hd, False, 1e4, 1e-6) for x in qkv]
    bounds, done = cache.empty_bounds(), [0, 0]
    for seq, a, b in ((0, 0, 100), (1, 0, 37), (0, 100, 150)):
        q = cache.append(tensor(F, qkv[seq][a:b]), words([seq] * (b - a)), words(range(a, b)), nh, 1e4)
        done[seq] = b
        cache.key_bounds(words(done), 100, bounds, fresh=words([b - a if i == seq else 0 for i in range(2)]))
        k, v = cache.rows(seq, 0, b)
        out = decode.causal_attention(q, k, v, nh, n_kv).to_vec().reshape(b - a, nh, hd)
        for i in (0, (b - a) // 2, b - a - 1):
            want, tol = P.attend(post[seq][0][a + i], post[seq][1][:a + i + 1], post[seq][2][:a + i + 1])
            # rows and queries are themselves rounded: 64 more roundings of the largest score, by exp into the weights
            slack = 64 * 2.0 ** -24 * np.abs(post[seq][0][a + i]).max() * np.abs(post[seq][1][:a + i + 1]).max() * np.sqrt(hd)
            assert (np.abs(out[i] - want) <= tol + 4 * slack * np.abs(want).max() + 1e-6).all(), (seq, i)
    for step in range(steps):
        now = [n + step + 1 for n in lens]
        rows = np.stack([qkv[i][now[i] - 1] for i in range(2)])
        q = cache.append(tensor(F, rows), None, words([n - 1 for n in now]), nh, 1e4)
        cache.key_bounds(words(now), 1, bounds)
        full = cache.attention(q, words(now), max(now), nh).to_vec().reshape(2, nh, hd)
        sel = cache.select(q, words(now), max(now), bounds, nh, 12)
        some = cache.attention_selected(q, words(now), sel, nh).to_vec().reshape(2, nh, hd)
        for i in range(2):
            want, tol = P.attend(post[i][0][now[i] - 1], post[i][1][:now[i]], post[i][2][:now[i]])
            slack = 64 * 2.0 ** -24 * np.abs(post[i][0][now[i] - 1]).max() * np.abs(post[i][1][:now[i]]).max() * np.sqrt(hd)
            assert (np.abs(full[i] - want) <= tol + 4 * slack * np.abs(want).max() + 1e-6).all(), (step, i)
            assert (np.abs(some[i] - want) <= tol + 4 * slack * np.abs(want).max() + 1e-6).all(), (step, i)     # all of its pages were chosen


@typed
def test_a_captured_step_serves_growing_sequences(F, paged, ty):
    n_kv, hd, nh, R, n_seq, steps = 2, 64, 6, 16, 3, 6
    rng = np.random.default_rng(1)
    start = [30, 0, 500]
    entries = 40
    table = rng.permutation(n_seq * entries).astype(np.uint32).reshape(n_seq, entries)
    caches = [paged.PagedKvCache(ty, R, n_seq * entries, n_kv, hd, n_seq, entries) for _ in range(2)]
    for c in caches:
        c.set_table(table)
        for i, n in enumerate(start):
            if n:
                c.append(tensor(F, np.random.default_rng(i).standard_normal((n, (nh + 2 * n_kv) * hd))), words([i] * n), words(range(n)), nh, 1e4)
    s = F.Stream()
    qkv, q = F.Tensor.empty((n_seq, (nh + 2 * n_kv) * hd)), F.Tensor.empty((n_seq, nh * hd))
    pos, lens = words(start), words([n + 1 for n in start])
    bounds = [c.empty_bounds() for c in caches]
    for c, b in zip(caches, bounds):
        c.key_bounds(words(start), 500, b)
    out, some, sel = F.Tensor.empty((n_seq, nh * hd)), F.Tensor.empty((n_seq, nh * hd)), F.Tensor.empty((n_seq, n_kv, 4), np.uint32)
    lib, chk = F._lib.load(), F._lib.check

    def step(c, b, outs, stream):
        c.append(qkv, None, pos, nh, 1e4, out=q, stream=stream)
        c.key_bounds(lens, 1, b, stream=stream)
        c.attention(q, lens, entries * R, nh, out=outs[0], stream=stream)
        c.select(q, lens, entries * R, b, nh, 4, out=outs[1], stream=stream)
        c.attention_selected(q, lens, outs[1], nh, out=outs[2], stream=stream)

    caches[0].reserve(nh, entries * R, 4, s)                     # before the capture begins
    chk(lib.fhip_stream_sync(None))
    g = F.Graph.begin(s)
    step(caches[0], bounds[0], (out, sel, some), s)
    g.end()
    for k in range(steps):
        upload(qkv.buf, np.random.default_rng(100 + k).standard_normal((n_seq, (nh + 2 * n_kv) * hd)).astype(np.float32))
        g.launch()
        s.synchronize()
        got = [t.to_vec(s) for t in (out, sel, some)]
        eager = (F.Tensor.empty((n_seq, nh * hd)), F.Tensor.empty((n_seq, n_kv, 4), np.uint32), F.Tensor.empty((n_seq, nh * hd)))
        step(caches[1], bounds[1], eager, None)
        for a, b in zip(got, eager):
            assert np.array_equal(a.view(np.uint32), b.to_vec().view(np.uint32)), k
        chk(lib.fhip_u32_add(pos.buf.ptr, n_seq, 1, None))
        chk(lib.fhip_u32_add(lens.buf.ptr, n_seq, 1, None))
        chk(lib.fhip_stream_sync(None))


def test_two_streams_at_once(F, paged):
    lens = [3000, 900]
    a, b = Filled(F, paged, P.BF16, lens, 2, 128, 32, 1), Filled(F, paged, P.F16, lens, 4, 64, 16, 2)
    qs = [np.random.default_rng(i).standard_normal((2, w)).astype(np.float32) for i, w in enumerate((8 * 128, 8 * 64))]
    streams, lt = [F.Stream(), F.Stream()], words(lens)
    outs = []
    for _ in range(4):
        for c, q, s in zip((a, b), qs, streams):
            outs.append((c, q, s, c.cache.attention(tensor(F, q), lt, 3000, 8, stream=s)))
    for c, q, s, o in outs:
        check_attention(c, o.to_vec(s), q, 8, lambda i: range(lens[i]))


def test_the_same_rows_as_a_contiguous_cache(F, paged):
    """One sequence on an f32 cache: fhip_decode_attention over the same rows says the same to both calls' roundings."""
    from ferric_amd import decode
    n, n_kv, hd, nh = 777, 2, 128, 10
    case = Filled(F, paged, P.F32, [n], n_kv, hd, 64, 6)
    k, v = case.cache.rows(0, 0, n)
    flat = decode.KvCache(n, n_kv * hd).append2(k, v)
    q = np.random.default_rng(0).standard_normal((1, nh * hd)).astype(np.float32)
    a = case.cache.attention(tensor(F, q), words([n]), n, nh).to_vec().reshape(nh, hd)
    b = decode.decode_attention(tensor(F, q), flat, nh, n_kv).to_vec().reshape(nh, hd)
    _, tol = P.attend(q.reshape(nh, hd).astype(np.float64), case.values("k", 0, range(n)), case.values("v", 0, range(n)))
    assert (np.abs(a - b) <= 2 * tol).all()
