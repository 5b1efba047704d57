"""The paged key/value cache's operators: the calls they are timed on, and the same in elementary torch operations.

A server keeps the keys and values of many sequences in one pool of pages: a page holds `page` rows of one sequence, a table names each
sequence's pages in order. Rows are appended from the fused projection row (bias, head norm, rotation), one new token of every sequence
attends over its own rows, over all of them or over the pages whose key bounds promise most, and a prompt behind a cached prefix
reads that prefix back as f32 rows. `listed` holds two or more cases of each, from the smallest call of a decode step to the largest;
`draw` gives further lengths, types and head layouts of the same kinds.
"""
import math

import numpy as np
import torch

own = False      # False: the plain forms below; True: the library's kernels

HALF = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROW_BYTES = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8_0": 34 / 32}
EPS = 1e-6


# ---- the cases ------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One new token of one sequence stored: the smallest call of a decode step, where only the launch counts.
        {"name": "append_token", "op": "append", "type": "f32", "seqs": 1, "rows": 1, "past": 200, "heads": 40, "kv_heads": 8, "head_dim": 128, "n_rot": 128,
         "interleaved": False, "norm": True, "bias": False, "base": 1e6, "page": 16},
        # Chunks of five long prompts of ragged lengths, at far positions, stored together.
        {"name": "append_prompts", "op": "append", "type": "bf16", "seqs": 5, "rows": 4099, "past": 120000, "heads": 40, "kv_heads": 8, "head_dim": 128,
         "n_rot": 128, "interleaved": False, "norm": True, "bias": True, "base": 1e6, "page": 64},
        # One sequence early in its answer: a call whose latency counts.
        {"name": "attend_short", "op": "attend", "type": "f32", "seqs": 1, "most": 199, "even": True, "heads": 40, "kv_heads": 8, "head_dim": 128, "page": 16,
         "window": 0, "softcap": 0.0},
        # An ordinary batch of a server: 24 sequences of every length up to 4096, small pages.
        {"name": "attend_ragged", "op": "attend", "type": "bf16", "seqs": 24, "most": 4096, "even": False, "heads": 40, "kv_heads": 8, "head_dim": 128, "page": 16,
         "window": 0, "softcap": 0.0},
        # One sequence behind a very long document: the keys are split between workgroups and joined.
        {"name": "attend_long", "op": "attend", "type": "bf16", "seqs": 1, "most": 131072, "even": True, "heads": 40, "kv_heads": 8, "head_dim": 128, "page": 64,
         "window": 0, "softcap": 0.0},
        # A full batch of long sequences with eight query heads to a key head: the largest call.
        {"name": "attend_full", "op": "attend", "type": "f16", "seqs": 64, "most": 8192, "even": True, "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 32,
         "window": 0, "softcap": 0.0},
        # A local layer with capped scores on an 8-bit cache, a key head to every query head, heads of 64.
        {"name": "attend_window", "op": "attend", "type": "q8_0", "seqs": 33, "most": 6001, "even": False, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 128,
         "window": 1024, "softcap": 50.0},
        # A layer of a decode step for eight sequences on an 8-bit cache: store the tokens' rows, then attend.
        {"name": "step_batch", "op": "step", "type": "q8_0", "seqs": 8, "most": 2500, "even": False, "heads": 40, "kv_heads": 8, "head_dim": 128, "n_rot": 128,
         "interleaved": False, "norm": True, "bias": False, "base": 1e6, "page": 32, "window": 0, "softcap": 0.0},
        # One sequence behind a very long document again, over 64 of its 2048 pages: bounds, choice, attention.
        {"name": "sparse_long", "op": "sparse", "type": "bf16", "seqs": 1, "most": 131072, "even": True, "heads": 40, "kv_heads": 8, "head_dim": 128, "page": 64,
         "select": 64, "first": 1, "last": 2},
        # A ragged batch, some sequences shorter than what may be chosen, on an f32 cache with small pages.
        {"name": "sparse_batch", "op": "sparse", "type": "f32", "seqs": 24, "most": 20000, "even": False, "heads": 32, "kv_heads": 4, "head_dim": 128, "page": 16,
         "select": 128, "first": 1, "last": 4},
        # A short cached prefix of an 8-bit cache read back for a prompt's next block.
        {"name": "rows_prefix", "op": "rows", "type": "q8_0", "row0": 0, "rows": 809, "kv_heads": 8, "head_dim": 128, "page": 32},
        # A long document's rows, from the middle of a page on.
        {"name": "rows_document", "op": "rows", "type": "bf16", "row0": 517, "rows": 100003, "kv_heads": 8, "head_dim": 128, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "step", "sparse", "sparse", "rows"])
    heads = {"kv_heads": rng.choice([1, 2, 4, 8, 16]), "head_dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128, 256])}
    if op == "rows":
        return {"op": op, "type": rng.choice(["f32", "f16", "bf16", "q8_0"]), "row0": rng.choice([0, _log(rng, 1, 5000)]), "rows": _log(rng, 1, 100003), **heads}
    heads["heads"] = heads["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 8, 16])
    post = {"interleaved": rng.random() < 0.3, "norm": rng.random() < 0.6, "bias": rng.random() < 0.4, "base": rng.choice([1e4, 5e5, 1e6]),
            "n_rot": rng.choice([heads["head_dim"]] * 3 + [heads["head_dim"] // 2, heads["head_dim"] // 4])}
    if op == "append":
        # What 8-bit blocks hold would come back through further launches that a server does not make: `step` has them.
        seqs = _log(rng, 1, 64)
        return {"op": op, "type": rng.choice(["f32", "f16", "bf16"]), "seqs": seqs, "rows": max(seqs, _log(rng, 1, 4099)), "past": rng.choice([0, _log(rng, 1, 120000)]),
                **heads, **post}
    case = {"op": op, "type": rng.choice(["f32", "f16", "bf16", "bf16", "q8_0"]), "seqs": _log(rng, 1, 128), "most": _log(rng, 1, 131072), "even": rng.random() < 0.3, **heads}
    if op == "sparse":
        return {**case, "select": _log(rng, 4, 256), "first": rng.choice([0, 1, 1, 2]), "last": rng.choice([1, 1, 2])}
    case.update(window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]))
    return {**case, **post} if op == "step" else case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50) + 4e-1 * _pool_bytes(case)      # a window's unread rows are prepared too


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    most["step"] = most["attend"]
    while True:
        c = _draw(rng)
        if _cost(c) <= most[c["op"]]:
            return c


def _lens(case):
    """Keys of every sequence, the new token among them."""
    if case["even"]:
        return [case["most"]] * case["seqs"]
    return [max(1, round(case["most"] * ((0.999 - 0.6180339887 * i) % 1.0) ** 1.5)) for i in range(case["seqs"])]


def _new_rows(case):
    """(sequence, first position, rows) of every sequence of an append."""
    n, weights = case["seqs"], [1 + (0.6180339887 * i) % 1.0 for i in range(case["seqs"])]
    ends = [round(case["rows"] * sum(weights[:i + 1]) / sum(weights)) for i in range(n)]
    return [(i, round(case["past"] * (1 - 0.37 * i / n)), e - b) for i, (b, e) in enumerate(zip([0] + ends, ends))]


def _pool_rows(case):
    if case["op"] == "append":
        return case["rows"] + 2 * case["page"] * case["seqs"]
    if case["op"] == "rows":
        return case["row0"] + case["rows"]
    return sum(-(-n // case["page"]) * case["page"] for n in _lens(case))


def _pool_bytes(case):
    return 2 * _pool_rows(case) * case["kv_heads"] * case["head_dim"] * ROW_BYTES[case["type"]]


def work(case):
    b, kvw = ROW_BYTES[case["type"]], case["kv_heads"] * case["head_dim"]
    if case["op"] == "rows":
        return {"bytes": 2 * case["rows"] * kvw * (b + 4), "flops": 0}
    q = case["heads"] * case["head_dim"]
    store = lambda t: t * (4 * (q + 2 * kvw) + 2 * kvw * b)      # projection rows in, key and value rows out
    if case["op"] == "append":
        return {"bytes": store(case["rows"]) + 4 * q * case["rows"], "flops": 10 * case["rows"] * (q + 2 * kvw)}
    lens = _lens(case)
    if case["op"] == "sparse":
        pages = [-(-n // case["page"]) for n in lens]
        rows = sum(min(n, case["select"] * case["page"]) for n in lens)
        return {"bytes": 8 * kvw * sum(pages) + 2 * rows * kvw * b + len(lens) * (8 * q + kvw * (b + 16) + 4 * case["kv_heads"] * case["select"]),
                "flops": 4 * q * sum(pages) + 4 * q * rows}
    rows = sum(min(n, case["window"] or n) for n in lens)
    return {"bytes": 2 * rows * kvw * b + 8 * q * len(lens) + (store(len(lens)) if case["op"] == "step" else 0), "flops": 4 * q * rows}


# ---- seeded inputs --------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")      # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")         # noqa: E731
    op, R, nkv, hd = case["op"], case["page"], case["kv_heads"], case["head_dim"]
    s = {"case": dict(case)}
    if op == "append":
        new = _new_rows(case)
        firsts, tops = [p // R for _, p, _ in new], [-(-(p + n) // R) for _, p, n in new]
        s["seq"] = ints([i for i, _, n in new for _ in range(n)])
        s["pos"] = ints([p + j for _, p, n in new for j in range(n)])
    else:
        lens = [case["row0"] + case["rows"]] if op == "rows" else _lens(case)
        firsts, tops = [0] * len(lens), [-(-n // R) for n in lens]
        s["lens"], s["max_len"] = ints(lens), max(lens)
        if op == "step":
            s["seq"], s["pos"] = ints(range(len(lens))), ints([n - 1 for n in lens])
    # every sequence's pages, in no order, some of the pool's unused; entries that no row needs name none
    used = sum(t - f for f, t in zip(firsts, tops))
    pages = used + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu().numpy()
    table = np.full((len(tops), max(tops)), -1, np.int32)
    at = 0
    for i, (f, t) in enumerate(zip(firsts, tops)):
        table[i, f:t] = order[at:at + t - f]
        at += t - f
    s["table"], s["pages"] = torch.from_numpy(table).cuda(), pages
    for name in ("k", "v"):
        if case["type"] == "q8_0":
            s[name] = torch.empty((pages * R, nkv * hd), dtype=torch.int8, device="cuda")
            for a in range(0, pages * R, 1 << 16):      # values as trained caches have them, a bell with a few far ones
                b = min(a + (1 << 16), pages * R)
                s[name][a:b] = (40 * randn(b - a, nkv * hd)).round_().clamp_(-127, 127).to(torch.int8)
            s[name + "_scales"] = ((0.75 + 0.5 * torch.rand((pages * R, nkv * hd // 32), generator=g, device="cuda")) / 40).to(torch.float16)
        else:
            s[name] = torch.randn((pages * R, nkv * hd), generator=g, device="cuda", dtype=HALF[case["type"]])
    if op in ("append", "step"):
        t, heads = len(s["pos"]), case["heads"] + 2 * nkv
        s["qkv"] = 2 * randn(t, heads * hd)
        s["bias"] = randn(heads * hd) if case["bias"] else None
        s["q_norm"], s["k_norm"] = (1 + 0.2 * randn(hd), 1 + 0.2 * randn(hd)) if case["norm"] else (None, None)
    if op in ("attend", "sparse"):
        s["q"] = 1.5 * randn(case["seqs"], case["heads"] * hd)
    if op == "sparse":
        # what the pages' bounds were before the newest token
        held = torch.zeros(pages, dtype=torch.int64, device="cuda")
        for i, n in enumerate(lens):
            own_pages = s["table"][i, :tops[i]].long()
            held[own_pages] = (n - 1 - R * torch.arange(tops[i], device="cuda")).clamp(0, R)
        s["bounds"] = torch.zeros((pages, nkv, 2, hd), device="cuda")
        for a in range(0, pages, 4096):
            b = min(a + 4096, pages)
            keys = _values(s, "k", torch.arange(a * R, b * R, device="cuda")).view(b - a, R, nkv, hd)
            out = (torch.arange(R, device="cuda") >= held[a:b, None])[:, :, None, None]
            s["bounds"][a:b, :, 0] = keys.masked_fill(out, math.inf).amin(1)
            s["bounds"][a:b, :, 1] = keys.masked_fill(out, -math.inf).amax(1)
    return s


def _values(s, name, rows):
    """f32 values of pool rows `rows` (any shape): [..., kv_heads * head_dim]."""
    x = s[name].index_select(0, rows.reshape(-1)).float()
    if s["case"]["type"] == "q8_0":
        d = s[name + "_scales"].index_select(0, rows.reshape(-1)).float()
        x = (x.view(-1, d.shape[1], 32) * d[:, :, None]).view(x.shape)
    return x.view(*rows.shape, -1)


def _rows_of(s, positions):
    """Pool rows of [sequences, n] positions; a position that its sequence does not have gives some row of the pool."""
    R = s["case"]["page"]
    page = s["table"].gather(1, (positions // R).clamp(max=s["table"].shape[1] - 1)).long().clamp(min=0)
    return page * R + positions % R


# ---- the plain forms ------------------------------------------------------------------------------------------------------------

def _plain_append(s):
    c = s["case"]
    t, hd, nh, nkv, R = len(s["pos"]), c["head_dim"], c["heads"], c["kv_heads"], c["page"]
    x = s["qkv"] if s["bias"] is None else s["qkv"] + s["bias"]
    x = x.view(t, nh + 2 * nkv, hd)
    qk, v = x[:, :nh + nkv], x[:, nh + nkv:]
    if c["norm"]:
        w = torch.cat([s["q_norm"].expand(nh, hd), s["k_norm"].expand(nkv, hd)])
        qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    half = c["n_rot"] // 2
    freq = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 / c["n_rot"] * math.log(c["base"])))
    angle = s["pos"].double()[:, None, None] * freq
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = (qk[..., 0:c["n_rot"]:2], qk[..., 1:c["n_rot"]:2]) if c["interleaved"] else (qk[..., :half], qk[..., half:c["n_rot"]])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([ra, rb], -1).flatten(-2) if c["interleaved"] else torch.cat([ra, rb], -1)
    qk = torch.cat([turned, qk[..., c["n_rot"]:]], -1)
    page = s["table"][s["seq"].long(), (s["pos"] // R).long()].long()
    row = page * R + s["pos"].long() % R
    for name, new in (("k", qk[:, nh:]), ("v", v)):
        new = new.reshape(t, nkv * hd)
        if c["type"] == "q8_0":
            blocks = new.reshape(t, -1, 32)
            d = blocks.abs().amax(-1, keepdim=True) / 127
            y = blocks * torch.where(d > 0, 1 / d, torch.zeros_like(d))
            codes = torch.copysign(torch.floor(y.abs() + 0.5), y).clamp(-127, 127)
            s[name].index_copy_(0, row, codes.reshape(t, -1).to(torch.int8))
            s[name + "_scales"].index_copy_(0, row, d.squeeze(-1).to(torch.float16))
        else:
            s[name].index_copy_(0, row, new.to(s[name].dtype))
    return qk[:, :nh].reshape(t, nh * hd).contiguous()


def _softmax_sum(c, q, k, v, dead):
    """q [n, g, hd] against k, v [n, keys, hd], keys that are `dead` [n, keys] left out: [n, g, hd]."""
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(c["head_dim"]))
    if c.get("softcap"):
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    x = x.masked_fill(dead[:, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return torch.matmul(p, v) / p.double().sum(-1, keepdim=True).float()


def _plain_attend(s, q):
    c = s["case"]
    n, nkv, hd, g = c["seqs"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    longest = s["max_len"]
    at = torch.arange(longest, device="cuda").expand(n, longest)
    if c["window"]:
        longest = min(longest, c["window"])
        at = at[:, :longest] + (s["lens"][:, None] - longest).clamp(min=0)
    dead = at >= s["lens"][:, None]
    rows = _rows_of(s, at)
    per_head = lambda x: x.view(n, longest, nkv, hd).transpose(1, 2).reshape(n * nkv, longest, hd)      # noqa: E731
    out = _softmax_sum(c, q.view(n * nkv, g, hd), per_head(_values(s, "k", rows)), per_head(_values(s, "v", rows)), dead.repeat_interleave(nkv, 0))
    return out.view(n, nkv * g * hd)


def _plain_sparse(s):
    c = s["case"]
    n, nkv, hd, g, R, want = c["seqs"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], c["page"], c["select"]
    # the newest token's key joins its page's bounds
    last = (s["lens"] - 1).long()[:, None]
    row = _rows_of(s, last)
    page = row[:, 0] // R
    key = _values(s, "k", row).view(n, nkv, hd)
    old, fresh = s["bounds"][page], (last % R == 0)[:, :, None]
    s["bounds"][page] = torch.stack([torch.where(fresh, key, torch.minimum(old[:, :, 0], key)), torch.where(fresh, key, torch.maximum(old[:, :, 1], key))], 2)
    # the largest score that any key within the bounds can reach, in 64 bits: pages next to the border of the choice
    m = s["table"].shape[1]
    have = (s["lens"].long()[:, None] + R - 1) // R
    at = torch.arange(m, device="cuda").expand(n, m)
    box = s["bounds"][s["table"].long().clamp(min=0)].double()                       # [n, m, kv, 2, hd]
    qd = s["q"].double().view(n, nkv, g, hd)
    flat = lambda x: x.permute(0, 2, 3, 1).reshape(n * nkv, hd, m)      # noqa: E731
    lo, hi = flat(box[:, :, :, 0]), flat(box[:, :, :, 1])
    pos, neg = qd.clamp(min=0).view(n * nkv, g, hd), qd.clamp(max=0).view(n * nkv, g, hd)
    score = (torch.matmul(pos, hi) + torch.matmul(neg, lo)).amax(1).view(n, nkv, m)
    kept = ((at < c["first"]) | (at >= have - c["last"])) & (at < have)
    score = torch.where(kept[:, None], math.inf, score).masked_fill((at >= have)[:, None], -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :want]
    best = torch.where(best < have[:, None], best, torch.full_like(best, 1 << 40)).sort(-1).values      # [n, kv, <= want], ascending
    none = best >= 1 << 40
    chosen = best.masked_fill(none, -1).to(torch.int32)
    if m < want:
        chosen = torch.cat([chosen, chosen.new_full((n, nkv, want - m), -1)], -1)
    # attention over the rows of these pages
    pos_at = (best.masked_fill(none, 0)[..., None] * R + torch.arange(R, device="cuda")).flatten(2)      # [n, kv, pages * R]
    dead = none.repeat_interleave(R, -1) | (pos_at >= s["lens"][:, None, None])
    rows = _rows_of(s, pos_at.view(n, -1)).view(n, nkv, -1)
    span = rows * nkv + torch.arange(nkv, device="cuda")[:, None]
    heads = dict(s)
    for name in ("k", "v"):
        heads[name] = s[name].view(-1, hd)
        if c["type"] == "q8_0":
            heads[name + "_scales"] = s[name + "_scales"].view(-1, hd // 32)
    rows_of = lambda name: _values(heads, name, span).view(n * nkv, -1, hd)      # noqa: E731
    out = _softmax_sum(c, s["q"].view(n * nkv, g, hd), rows_of("k"), rows_of("v"), dead.view(n * nkv, -1))
    return chosen, out.view(n, nkv * g * hd)


# ---- the library's calls --------------------------------------------------------------------------------------------------------

class _At:
    """Device memory of torch as the library's Tensor takes it."""

    def __init__(self, t):
        self.ptr = t.data_ptr()


def _tensor(F, t):
    return None if t is None else F.Tensor(_At(t), t.shape, np.float32 if t.dtype == torch.float32 else np.uint32)


def _cache(s):
    """The handle that a program makes of its pool and table once."""
    from ferric_amd import paged
    c = s["case"]
    if "cache" not in s:
        kind = {"f32": paged.F32, "f16": paged.F16, "bf16": paged.BF16, "q8_0": paged.Q8_0}[c["type"]]
        scales = [_At(s[name]) for name in ("k_scales", "v_scales")] if c["type"] == "q8_0" else [None, None]
        s["cache"] = paged.PagedKvCache.wrap(kind, c["page"], s["pages"], c["kv_heads"], c["head_dim"], _At(s["k"]), _At(s["v"]), *scales,
                                             _At(s["table"]), s["table"].shape[0], s["table"].shape[1])
    return s["cache"]


def _own_append(s):
    import ferric_amd as F
    c = s["case"]
    q = torch.empty((len(s["pos"]), c["heads"] * c["head_dim"]), device="cuda")
    _cache(s).append(_tensor(F, s["qkv"]), _tensor(F, s["seq"]), _tensor(F, s["pos"]), c["heads"], c["base"], n_rot=c["n_rot"], interleaved=c["interleaved"], eps=EPS,
                     bias=_tensor(F, s["bias"]), q_norm=_tensor(F, s["q_norm"]), k_norm=_tensor(F, s["k_norm"]), out=_tensor(F, q))
    return q


def _own_attend(s, q):
    import ferric_amd as F
    c = s["case"]
    out = torch.empty((c["seqs"], c["heads"] * c["head_dim"]), device="cuda")
    _cache(s).attention(_tensor(F, q), _tensor(F, s["lens"]), s["max_len"], c["heads"], window=c["window"], softcap=c["softcap"], out=_tensor(F, out))
    return out


def _own_sparse(s):
    import ferric_amd as F
    c, cache = s["case"], _cache(s)
    chosen = torch.empty((c["seqs"], c["kv_heads"], c["select"]), dtype=torch.int32, device="cuda")
    out = torch.empty((c["seqs"], c["heads"] * c["head_dim"]), device="cuda")
    q, lens, bounds, picked = (_tensor(F, t) for t in (s["q"], s["lens"], s["bounds"], chosen))
    cache.key_bounds(lens, 1, bounds)
    cache.select(q, lens, s["max_len"], bounds, c["heads"], c["select"], first=c["first"], last=c["last"], out=picked)
    cache.attention_selected(q, lens, picked, c["heads"], out=_tensor(F, out))
    return chosen, out


def _own_rows(s):
    import ferric_amd as F
    c = s["case"]
    k, v = (torch.empty((c["rows"], c["kv_heads"] * c["head_dim"]), device="cuda") for _ in range(2))
    _cache(s).rows(0, c["row0"], c["rows"], out=(_tensor(F, k), _tensor(F, v)))
    return k, v


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if op == "append":
        return (_own_append(s) if own else _plain_append(s)), s["k"], s["v"]
    if op == "attend":
        return _own_attend(s, s["q"]) if own else _plain_attend(s, s["q"])
    if op == "step":
        return _own_attend(s, _own_append(s)) if own else _plain_attend(s, _plain_append(s))
    if op == "sparse":
        return (*(_own_sparse(s) if own else _plain_sparse(s)), s["bounds"])
    if own:
        return _own_rows(s)
    at = _rows_of(s, s["case"]["row0"] + torch.arange(s["case"]["rows"], device="cuda")[None])[0]
    return _values(s, "k", at), _values(s, "v", at)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------

def _pool64(s, name, at):
    """[n, kv_heads, head_dim] of the pool rows `at`, in 64 bits."""
    c = s["case"]
    x = s[name][at].double()
    if c["type"] == "q8_0":
        x = x * s[name + "_scales"][at].double().repeat_interleave(32, -1)
    return x.view(len(at), c["kv_heads"], c["head_dim"])


def _place(s, i, positions):
    R = s["case"]["page"]
    return s["table"][i].long()[positions // R] * R + positions % R


def _append64(s):
    """Queries, keys and values of the new rows, and the pool rows they go to."""
    c = s["case"]
    hd, nh, nkv, rot = c["head_dim"], c["heads"], c["kv_heads"], c["n_rot"]
    x = s["qkv"].double()
    if s["bias"] is not None:
        x = x + s["bias"].double()
    x = x.view(len(x), -1, hd)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    parts = []
    for y, w in ((q, s["q_norm"]), (k, s["k_norm"])):
        y = y.clone()
        if w is not None:
            y *= torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
        first = torch.arange(rot // 2, device="cuda") * (2 if c["interleaved"] else 1)
        second = first + (1 if c["interleaved"] else rot // 2)
        turn = s["pos"].double()[:, None] * c["base"] ** (-torch.arange(0, rot, 2, device="cuda").double() / rot)
        z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.ones_like(turn), turn)[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        parts.append(y)
    rows = torch.cat([_place(s, i, s["pos"].long()[s["seq"] == i]) for i in range(c["seqs"])])      # rows come sequence by sequence
    return parts[0], parts[1], v, rows


def _attend64(q, k, v, softcap=0.0):
    """q [heads, hd], k and v [keys, kv_heads, hd]."""
    g = q.shape[0] // k.shape[1]
    x = torch.matmul(q.view(k.shape[1], g, -1), k.permute(1, 2, 0)) / math.sqrt(q.shape[1])
    if softcap:
        x = softcap * torch.tanh(x / softcap)
    return torch.matmul(torch.softmax(x, -1), v.permute(1, 0, 2)).reshape(-1)


def exact(case, seed):
    s = prepare(case, seed)
    c, op = s["case"], case["op"]
    if op == "rows":
        at = _place(s, 0, torch.arange(c["row0"], c["row0"] + c["rows"], device="cuda"))
        return _pool64(s, "k", at).flatten(1), _pool64(s, "v", at).flatten(1)
    q = s["q"].double().view(c["seqs"], c["heads"], c["head_dim"]) if "q" in s else None
    if op in ("append", "step"):
        q, k, v, rows = _append64(s)
        if op == "append":
            pools = [s["k"].double(), s["v"].double()]
            for pool, new in zip(pools, (k, v)):
                pool[rows] = new.flatten(1)
            return q.flatten(1), pools[0], pools[1]
        for name, new in (("k", k), ("v", v)):
            new = new.flatten(1)
            if c["type"] == "q8_0":
                d = new.reshape(len(new), -1, 32).abs().amax(-1) / 127
                y = new.reshape(len(new), -1, 32) / d[..., None]
                s[name][rows] = (torch.sign(y) * torch.floor(y.abs() + 0.5)).flatten(1).to(torch.int8)
                s[name + "_scales"][rows] = d.half()
            else:
                s[name][rows] = new.to(s[name].dtype)
    outs, R = [], c["page"]
    for i, n in enumerate(_lens(case)):
        if op == "sparse":
            at = _place(s, i, torch.tensor([n - 1], device="cuda"))
            page, key = int(at) // R, _pool64(s, "k", at)[0].float()
            for e, pick in ((0, torch.minimum), (1, torch.maximum)):
                s["bounds"][page, :, e] = key if (n - 1) % R == 0 else pick(s["bounds"][page, :, e], key)
            pages = -(-n // R)
            box = s["bounds"][s["table"][i, :pages].long()].double()
            heads = []
            for h in range(c["kv_heads"]):
                g = c["heads"] // c["kv_heads"]
                qh = q[i, h * g:(h + 1) * g]
                reach = torch.stack([torch.maximum(u * box[:, h, 0], u * box[:, h, 1]).sum(-1) for u in qh]).amax(0).cpu().numpy()
                held = [p for p in range(pages) if p < c["first"] or p >= pages - c["last"]]
                rest = [p for p in np.argsort(-reach, kind="stable") if c["first"] <= p < pages - c["last"]]
                chosen = sorted(held[:c["select"]] + rest[:max(0, c["select"] - len(held))])
                keys = torch.cat([torch.arange(p * R, min(n, (p + 1) * R), device="cuda") for p in chosen])
                at = _place(s, i, keys)
                heads.append(_attend64(qh, _pool64(s, "k", at)[:, h:h + 1], _pool64(s, "v", at)[:, h:h + 1]))
            outs.append(torch.cat(heads))
        else:
            at = _place(s, i, torch.arange(max(0, n - (c["window"] or n)), n, device="cuda"))
            outs.append(_attend64(q[i], _pool64(s, "k", at), _pool64(s, "v", at), c["softcap"]))
    if op == "sparse":
        return None, torch.stack(outs), s["bounds"].double()
    return torch.stack(outs)
