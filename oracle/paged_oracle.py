"""The paged key/value cache's definitions in 64 bits (numpy), test infrastructure only: written from the formulas, one sequence at a time."""
import numpy as np

NO_PAGE = 0xFFFFFFFF
F32, F16, BF16, Q8_0 = 0, 1, 30, 8
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # a rounding to the type, relative to the value


def bf16_bits(x):
    """f32 values to bf16 patterns, to nearest, ties to even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def encode(x, ty):
    """f32 rows [n, width] as a pool holds them: (array of the pool's words, scales or None)."""
    x = np.ascontiguousarray(x, np.float32)
    if ty == F32:
        return x, None
    if ty == F16:
        return x.astype(np.float16), None
    if ty == BF16:
        return bf16_bits(x), None
    b = x.reshape(x.shape[0], -1, 32)
    d = np.abs(b).max(-1) / np.float32(127)
    with np.errstate(divide="ignore"):
        y = b * np.where(d > 0, np.float32(1) / d, np.float32(0)).astype(np.float32)[..., None]
    codes = np.clip(np.copysign(np.floor(np.abs(y) + np.float32(0.5)), y), -127, 127).astype(np.int8)
    return codes.reshape(x.shape), d.astype(np.float16)


def decode(pool, scales, ty):
    """What the pool's rows stand for, in 64 bits."""
    if ty == BF16:
        return (pool.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if ty == Q8_0:
        return pool.astype(np.float64) * np.repeat(scales.astype(np.float64), 32, -1)
    return pool.astype(np.float64)


def place(table_row, positions, page_rows, n_pages):
    """Pool rows of a sequence's positions; -1 where the table names no page."""
    out = []
    for p in positions:
        e = p // page_rows
        page = int(table_row[e]) if e < len(table_row) else NO_PAGE
        out.append(page * page_rows + p % page_rows if page < n_pages else -1)
    return np.array(out, np.int64)


def post(qkv, pos, n_head, n_kv, hd, n_rot, interleaved, base, eps, bias=None, q_norm=None, k_norm=None, freq_scale=None):
    """(q, k, v) [t, heads, hd] of fused rows: bias, head norm, rotation."""
    x = qkv.astype(np.float64) + (0 if bias is None else bias.astype(np.float64))
    x = x.reshape(len(x), -1, hd)
    q, k, v = x[:, :n_head].copy(), x[:, n_head:n_head + n_kv].copy(), x[:, n_head + n_kv:]
    half = n_rot // 2
    freq = np.float64(np.float32(base)) ** (-2.0 * np.arange(half) / n_rot) if half else np.zeros(0)
    if freq_scale is not None:
        freq = freq * freq_scale[:half].astype(np.float64)
    ang = np.asarray(pos, np.float64)[:, None] * freq
    cs, sn = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a = np.arange(half) * 2 if interleaved else np.arange(half)
    b = a + 1 if interleaved else a + half
    for y, w in ((q, q_norm), (k, k_norm)):
        if w is not None:
            y *= w.astype(np.float64) / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        y1, y2 = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = y1 * cs - y2 * sn, y2 * cs + y1 * sn
    return q, k, v


def attend(q, k, v, softcap=0.0):
    """q [heads, hd], k and v [keys, kv_heads, hd] -> (out [heads, hd], the error that f32 arithmetic is allowed there).

    The allowance: a score is a sum of hd products (each rounded once with its addition: (hd + 4) roundings of at most sum |q_d k_d| with the factor 1 / sqrt(hd));
    exp turns its absolute error into a relative one, twice (weight and sum); softcap adds a tanh and two products to it, 8 roundings of its value; the rescaling by earlier maxima and the exponentials
    are 16 roundings more, and a sum over n keys in pieces of four adds n / 4 + 32."""
    n, hd = len(k), q.shape[1]
    g = q.shape[0] // (k.shape[1] if n else q.shape[0])
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    if n == 0:
        return out, tol
    eps = 2.0 ** -24
    for h in range(q.shape[0]):
        kk, vv = k[:, h // g], v[:, h // g]
        x = kk @ q[h] / np.sqrt(hd)
        dx = (hd + 4) * eps * (np.abs(kk) @ np.abs(q[h])) / np.sqrt(hd)
        if softcap:
            x = softcap * np.tanh(x / softcap)
            dx = dx + 8 * eps * softcap
        dx = dx + 4 * eps * np.abs(x - x.max())          # the difference from the maximum, and its product with log2 e
        p = np.exp(x - x.max())
        p /= p.sum()
        out[h] = p @ vv
        tol[h] = (2 * dx.max() + (16 + n / 4 + 32) * eps) * (p @ np.abs(vv)) + 1e-37
    return out, tol


def select(q, bounds, n_kv, n_select, first, last):
    """q [heads, hd], bounds [pages, kv, 2, hd] -> [kv, n_select] page indices."""
    pages, hd = len(bounds), q.shape[1]
    g = q.shape[0] // n_kv
    out = np.full((n_kv, n_select), NO_PAGE, np.uint32)
    for h in range(n_kv):
        b = bounds[:, h].astype(np.float64)
        best = np.full(pages, -np.inf)
        for e in range(g):
            u = q[h * g + e].astype(np.float64)
            best = np.maximum(best, np.maximum(u * b[:, 0], u * b[:, 1]).sum(-1))
        kept = [p for p in range(pages) if p < first or p >= pages - last]
        rest = [p for p in np.argsort(-best, kind="stable") if first <= p < pages - last]
        chosen = sorted((kept + rest)[:n_select])
        out[h, :len(chosen)] = chosen
    return out
