"""Timed cases of the paged key-value cache and the attention that reads it.

A server that holds many song requests at once keeps their keys and values in
pages: prompts are appended to pages and attended to, every decode step appends
one token per sequence and attends over its page table, takes of one prompt
share its pages, and pages are moved together when the pool is compacted. A
case is one layer's call of one of these operators (the page copies: every
layer's), at the head layouts of the 3072-wide and the 2048-wide decoder
(24 / 8 and 16 / 8 heads of 128), with cache lengths up to the context of 24576.

`own` False: the operators in elementary torch operations in 32 bits. `own`
True: the library's calls.
"""
import importlib
import math

import torch

own = False

D = 128
EPS = 1e-5
THETA = 500000.0
BLOCK = 32  # slots of a block of V, stored dim by dim
CONTEXT = 24576
WIDE = dict(heads=24, kv_heads=8)
NARROW = dict(heads=16, kv_heads=8)


def listed():
    return [
        # one request just after a short prompt: the smallest call, its latency is the step's
        dict(name="decode_b1_kv333", kind="decode", batch=1, lo=333, hi=333, page=64, window=0, sinks=0, **WIDE),
        # one request at the benchmark's cache length
        dict(name="decode_b1_kv4096", kind="decode", batch=1, lo=4096, hi=4096, page=64, window=0, sinks=0, **WIDE),
        # eight takes of unlike lengths, as the session's largest batch
        dict(name="decode_b8", kind="decode", batch=8, lo=700, hi=6144, page=32, window=0, sinks=0, **NARROW),
        # a full server: requests from their first seconds to the end of the context
        dict(name="decode_b45", kind="decode", batch=45, lo=150, hi=24500, page=128, window=0, sinks=0, **WIDE),
        # long songs that keep a window and the first tokens; the pages between were freed
        dict(name="decode_b13_window", kind="decode", batch=13, lo=3000, hi=20011, page=64, window=1000, sinks=37,
             **NARROW),
        # the rest of a prompt after a long shared prefix
        dict(name="prefill_97_after_4000", kind="prefill", batch=1, lo=97, hi=97, before=4000, page=64, window=0,
             sinks=0, **WIDE),
        # the benchmark's long prompt
        dict(name="prefill_3000", kind="prefill", batch=1, lo=3000, hi=3000, before=0, page=64, window=0, sinks=0,
             **WIDE),
        # prompts of several requests in one call, windowed
        dict(name="prefill_b5_window", kind="prefill", batch=5, lo=411, hi=5003, before=130, page=128, window=1024,
             sinks=4, **NARROW),
        # that long prompt's rows into the pages
        dict(name="append_3000", kind="append", batch=1, lo=3000, hi=3000, before=0, page=64, **WIDE),
        # short prompts of several requests after a shared prefix
        dict(name="append_b7", kind="append", batch=7, lo=19, hi=301, before=75, page=32, **NARROW),
        # seven more takes of one prompt: its partly filled last page, in every layer
        dict(name="copy_fork_8", kind="copy", pairs=7, shared=True, layers=28, pages=40, page=64, kv_heads=8),
        # a compaction: scattered pages move together, in every layer
        dict(name="copy_compact_90", kind="copy", pairs=90, shared=False, layers=28, pages=200, page=64, kv_heads=8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "prefill", "prefill", "append", "copy"))
    heads, kv_heads = rng.choice(((24, 8), (24, 8), (16, 8), (16, 8), (8, 8), (8, 2), (6, 1), (32, 4)))
    page = rng.choice((32, 64, 128))
    dims = dict(heads=heads, kv_heads=kv_heads, page=page)
    window = rng.choice((0, 0, _log_int(rng, 33, 4000)))
    seen = dict(window=window, sinks=rng.choice((0, rng.randint(1, 100))) if window else 0)
    if kind == "decode":
        batch = _log_int(rng, 1, 40)
        hi = _log_int(rng, 1, CONTEXT - 1 if batch < 20 else 14000)
        return dict(kind=kind, batch=batch, lo=_log_int(rng, 1, hi), hi=hi, **dims, **seen)
    if kind == "prefill":
        batch = rng.choice((1, 1, rng.randint(2, 7)))
        hi = _log_int(rng, 1, 4000 if batch == 1 else 1500)
        c = dict(kind=kind, batch=batch, lo=_log_int(rng, 1, hi), hi=hi,
                 before=rng.choice((0, rng.randint(1, 3000))), **dims, **seen)
        while work(c)["flops"] > 6e10:  # no more than the listed ones
            c["hi"] = c["hi"] * 2 // 3
            c["lo"] = min(c["lo"], c["hi"])
        return c
    if kind == "append":
        batch = rng.choice((1, rng.randint(2, 9)))
        hi = _log_int(rng, 1, 4000 if batch == 1 else 700)
        return dict(kind=kind, batch=batch, lo=_log_int(rng, 1, hi), hi=hi,
                    before=rng.choice((0, rng.randint(1, 3000))), **dims)
    shared = rng.random() < 0.4
    pairs = rng.randint(1, 9) if shared else _log_int(rng, 1, 80)
    return dict(kind=kind, pairs=pairs, shared=shared, layers=rng.randint(1, 28), pages=2 * pairs + rng.randint(3, 30),
                page=page, kv_heads=rng.choice((1, 2, 4, 8)))


# ---- sizes ----

def _lengths(c):
    """Tokens of each sequence (decode: with the new one), from lo to hi, long and short ones mixed."""
    b = c["batch"]
    if b == 1:
        return [c["hi"]]
    ratio = c["hi"] / c["lo"]
    return [max(1, int(round(c["lo"] * ratio ** ((i * 7 % b if b % 7 else i * 5 % b) / (b - 1))))) for i in range(b)]


def _visible(p, window, sinks):
    """Keys that position p sees."""
    if window == 0 or p < window:
        return p + 1
    return window + min(sinks, p - window + 1)


def _totals(c):
    """Of an attention case: (key, query) pairs, and keys that any query of their sequence sees."""
    pairs = keys = 0
    for n in _lengths(c):
        first = c["before"] if c["kind"] == "prefill" else n - 1
        last = first + n - 1 if c["kind"] == "prefill" else n - 1
        pairs += sum(_visible(p, c["window"], c["sinks"]) for p in range(first, last + 1))
        low = max(0, first - c["window"] + 1) if c["window"] else 0
        keys += last + 1 - low + min(c["sinks"] if c["window"] else 0, low)
    return pairs, keys


def work(case):
    c = case
    row = D * 2  # bytes of a head's row
    if c["kind"] == "copy":
        page = c["layers"] * 2 * c["kv_heads"] * c["page"] * row
        return {"bytes": (c["pairs"] + (1 if c["shared"] else c["pairs"])) * page, "flops": 0}
    rows = c["batch"] if c["kind"] == "decode" else sum(_lengths(c))
    qkv = rows * (c["heads"] + 2 * c["kv_heads"]) * row
    if c["kind"] == "append":
        return {"bytes": 2 * qkv + rows * row, "flops": 10 * qkv}
    pairs, keys = _totals(c)
    kv = keys * c["kv_heads"] * 2 * row
    moved = qkv + rows * (c["heads"] + 2 * c["kv_heads"]) * row if c["kind"] == "decode" else 2 * rows * c["heads"] * row
    return {"bytes": kv + moved, "flops": 4 * D * c["heads"] * pairs}


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _normal(g, *shape, mean=0.0, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(torch.bfloat16)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rope(positions):
    inv = 1.0 / THETA ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return a.cos().to(torch.bfloat16), a.sin().to(torch.bfloat16)


def _pool(g, layers, pages, kv_heads, page):
    """Pages of keys after their norm, and of values in blocks."""
    k = _normal(g, layers, pages, kv_heads, page, D, std=1.3)
    v = _normal(g, layers, pages, kv_heads, page // BLOCK, D, BLOCK)
    return k, v


def prepare(case, seed):
    c = dict(case)
    g = _gen(seed)
    if c["kind"] == "copy":
        k, v = _pool(g, c["layers"], c["pages"], c["kv_heads"], c["page"])
        ids = torch.randperm(c["pages"], generator=g, device="cuda").tolist()
        src = [ids[0]] * c["pairs"] if c["shared"] else ids[:c["pairs"]]
        dst = ids[-c["pairs"]:]
        return dict(kind="copy", k=k, v=v, src=src, dst=dst)
    hq, hkv, page = c["heads"], c["kv_heads"], c["page"]
    lens = _lengths(c)
    before = [n - 1 for n in lens] if c["kind"] == "decode" else [c["before"]] * c["batch"]
    ends = lens if c["kind"] == "decode" else [c["before"] + n for n in lens]
    need = [(e + page - 1) // page for e in ends]
    width, pages = max(need), sum(need) + 5
    k, v = _pool(g, 1, pages, hkv, page)
    ids = torch.randperm(pages, generator=g, device="cuda").tolist()
    table, at = [], 0
    for b, n in enumerate(need):
        row = ids[at:at + n] + [-1] * (width - n)
        at += n
        if c.get("window"):  # pages that no later token sees are not held any more
            for j in range(n):
                if (j + 1) * page <= before[b] - c["window"] + 1 and j * page >= c["sinks"]:
                    row[j] = -1
        table.append(row)
    s = dict(kind=c["kind"], heads=hq, kv_heads=hkv, page=page, k=k[0], v=v[0], table=_ints(table),
             window=c.get("window", 0), sinks=c.get("sinks", 0))
    if c["kind"] == "decode":
        s["pos"] = _ints(before)
    else:
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        s["starts"], s["before"] = _ints(starts), _ints(before)
    rows = c["batch"] if c["kind"] == "decode" else sum(lens)
    if c["kind"] == "prefill":
        s["q"] = _normal(g, rows, hq, D, std=1.5)
        return s
    s["qkv"] = _normal(g, rows, (hq + 2 * hkv) * D)
    s["q_gain"], s["k_gain"] = _normal(g, D, mean=1.5, std=0.1), _normal(g, D, mean=1.3, std=0.1)
    s["cos"], s["sin"] = _rope(max(ends))
    return s


# ---- the plain forms ----

def _norm_rope(x, gain, cos, sin):
    """RMSNorm and half-split rotation of rows [..., heads, 128], cos / sin [..., 1, 64]."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _split(s, position):
    """(q, k, v) of the rows of qkv: rotated queries and keys in 32 bits, values as they are."""
    hq, hkv = s["heads"], s["kv_heads"]
    x = s["qkv"].view(-1, hq + 2 * hkv, D)
    cos, sin = s["cos"][position].float()[:, None], s["sin"][position].float()[:, None]
    q = _norm_rope(x[:, :hq].float(), s["q_gain"].float(), cos, sin)
    k = _norm_rope(x[:, hq:hq + hkv].float(), s["k_gain"].float(), cos, sin)
    return q, k, x[:, hq + hkv:]


def _store(s, sequence, position, k, v):
    page = s["table"].long()[sequence, position // s["page"]]
    slot = position % s["page"]
    s["k"][page, :, slot] = k.to(torch.bfloat16)
    s["v"][page, :, slot // BLOCK, :, slot % BLOCK] = v


def _rows(s):
    """(sequence, position) of every row of a prompt call."""
    starts, before = s["starts"].long(), s["before"].long()
    n = starts[1:] - starts[:-1]
    sequence = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=_count(s))
    return sequence, before[sequence] + torch.arange(_count(s), device="cuda") - starts[sequence]


def _count(s):
    return (s["q"] if "q" in s else s["qkv"]).shape[0]


def _gathered(s):
    """The tables' keys and values as [sequences, kv heads, slots, 128] in 32 bits."""
    t = s["table"].long().clamp(min=0)
    b, w = t.shape
    k = s["k"][t].transpose(1, 2).reshape(b, s["kv_heads"], w * s["page"], D).float()
    v = s["v"][t].permute(0, 2, 1, 3, 5, 4).reshape(b, s["kv_heads"], w * s["page"], D).float()
    return k, v


def _attend(s, q, position):
    """q [sequences, rows, heads, 128] at position [sequences, rows] over the tables' pages."""
    b, n = position.shape
    g = s["heads"] // s["kv_heads"]
    k, v = _gathered(s)
    q = q.view(b, n, s["kv_heads"], g, D).permute(0, 2, 3, 1, 4).reshape(b, s["kv_heads"], g * n, D)
    scores = (q @ k.transpose(-1, -2).contiguous()).mul_(D ** -0.5).view(b, s["kv_heads"], g, n, -1)
    key = torch.arange(k.shape[2], device="cuda")
    p = position[:, None, None, :, None]
    seen = key <= p
    if s["window"]:
        seen = seen & ((p - key < s["window"]) | (key < s["sinks"]))
    scores.masked_fill_(~seen, -math.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    weights = weights.div_(weights.sum(-1, keepdim=True)).view(b, s["kv_heads"], g * n, -1)
    out = (weights @ v).view(b, s["kv_heads"], g, n, D)
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, s["heads"], D)


def _plain_decode(s):
    pos = s["pos"].long()
    q, k, v = _split(s, pos)
    _store(s, torch.arange(pos.numel(), device="cuda"), pos, k, v)
    return _attend(s, q[:, None], pos[:, None])[:, 0].to(torch.bfloat16), s["k"], s["v"]


def _plain_append(s):
    sequence, position = _rows(s)
    q, k, v = _split(s, position)
    _store(s, sequence, position, k, v)
    return q.to(torch.bfloat16), s["k"], s["v"]


def _plain_prefill(s):
    sequence, position = _rows(s)
    starts = s["starts"].long()
    b, n = starts.numel() - 1, int(s["table"].shape[1]) * s["page"]
    index = position - s["before"].long()[sequence]  # a row's place in its sequence
    q = torch.zeros(b, n, s["heads"], D, device="cuda")
    q[sequence, index] = s["q"].float()
    longest = min(n, _count(s))
    at = s["before"].long()[:, None] + torch.arange(longest, device="cuda")
    return _attend(s, q[:, :longest], at)[sequence, index].to(torch.bfloat16)


def _plain_copy(s):
    s["k"][:, s["dst"]] = s["k"][:, s["src"]]
    s["v"][:, s["dst"]] = s["v"][:, s["src"]]
    return s["k"], s["v"]


# ---- the library's calls ----

def _library():
    return importlib.import_module("yue2-mlx_amd.yuear")


def _workspace(s, y, rows=0):
    """The zeroed workspace that a program keeps for its calls."""
    if "workspace" not in s:
        s["workspace"] = y.paged_workspace(s["table"].shape[0], s["heads"], s["kv_heads"], rows)
    return s["workspace"]


def _own_decode(s):
    y = _library()
    out = y.paged_attention_decode(s["qkv"], s["k"], s["v"], s["table"], s["pos"], s["cos"], s["sin"],
                                   q_norm=s["q_gain"], k_norm=s["k_gain"], eps=EPS, window=s["window"],
                                   sinks=s["sinks"], workspace=_workspace(s, y))
    return out, s["k"], s["v"]


def _own_append(s):
    out = _library().paged_append(s["qkv"], s["k"], s["v"], s["table"], s["starts"], s["before"], s["cos"], s["sin"],
                                  q_norm=s["q_gain"], k_norm=s["k_gain"], eps=EPS)
    return out, s["k"], s["v"]


def _own_prefill(s):
    y = _library()
    return y.paged_attention_prefill(s["q"], s["k"], s["v"], s["table"], s["starts"], s["before"], window=s["window"],
                                     sinks=s["sinks"], workspace=_workspace(s, y, _count(s)))


def _own_copy(s):
    _library().pages_copy(s["k"], s["v"], s["src"], s["dst"])
    return s["k"], s["v"]


def run(state):
    kind = state["kind"]
    if own:
        return dict(decode=_own_decode, append=_own_append, prefill=_own_prefill, copy=_own_copy)[kind](state)
    return dict(decode=_plain_decode, append=_plain_append, prefill=_plain_prefill, copy=_plain_copy)[kind](state)


# ---- the definition in 64 bits, sequence by sequence and head by head ----

def _exact_turned(x, gain, c, s):
    """rope(x / sqrt(mean x^2 + eps) * gain) of rows [n, 128] at rows c, s [n, 64] of the tables."""
    x = x.double()
    x = x / ((x ** 2).sum(-1, keepdim=True) / D + EPS).sqrt() * gain.double()
    out = torch.empty_like(x)
    out[:, :64] = x[:, :64] * c.double() - x[:, 64:] * s.double()
    out[:, 64:] = x[:, 64:] * c.double() + x[:, :64] * s.double()
    return out


def _exact_head(k, v, table, page, head, n):
    """Keys and values [n, 128] of one kv head's first n slots (zeros where the table has no page)."""
    keys = torch.zeros(n, D, dtype=torch.float64, device="cuda")
    values = torch.zeros_like(keys)
    for j, p in enumerate(table[:(n + page - 1) // page]):
        if p >= 0:
            m = min(page, n - j * page)
            keys[j * page:j * page + m] = k[p, head, :m].double()
            values[j * page:j * page + m] = v[p, head].transpose(1, 2).reshape(page, D)[:m].double()
    return keys, values


def _exact_rows(q, first, keys, values, window, sinks):
    """softmax(q k^T / sqrt(128)) v of the rows q [g, n, 128] at positions first, first + 1, ..."""
    score = q @ keys.T / math.sqrt(D)
    p = torch.arange(first, first + q.shape[1], device="cuda")[:, None]
    t = torch.arange(keys.shape[0], device="cuda")[None, :]
    hidden = t > p
    if window:
        hidden |= (t <= p - window) & (t >= sinks)
    score[:, hidden] = -math.inf
    return torch.softmax(score, -1) @ values


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "copy":
        k, v = s["k"].double(), s["v"].double()
        for a, b in zip(s["src"], s["dst"]):
            k[:, b], v[:, b] = k[:, a], v[:, a]
        return k, v
    hq, hkv, page = s["heads"], s["kv_heads"], s["page"]
    g = hq // hkv
    tables = s["table"].tolist()
    if s["kind"] == "decode":
        first = s["pos"].tolist()
        starts = list(range(len(first) + 1))
    else:
        first, starts = s["before"].tolist(), s["starts"].tolist()
    rows = starts[-1]
    k, v = s["k"], s["v"]
    if s["kind"] != "prefill":
        position = torch.cat([torch.arange(p, p + b - a, device="cuda") for p, a, b in zip(first, starts, starts[1:])])
        c, n = s["cos"][position], s["sin"][position]
        qkv = s["qkv"].view(rows, hq + 2 * hkv, D)
        q = torch.stack([_exact_turned(qkv[:, h], s["q_gain"], c, n) for h in range(hq)], 1)
        k64, v64 = k.double(), v.double()
        for b, table in enumerate(tables):
            for r in range(starts[b], starts[b + 1]):
                at = first[b] + r - starts[b]
                p, t = table[at // page], at % page
                v[p, :, t // BLOCK, :, t % BLOCK] = qkv[r, hq + hkv:]
                v64[p, :, t // BLOCK, :, t % BLOCK] = qkv[r, hq + hkv:].double()
        new = torch.stack([_exact_turned(qkv[:, hq + h], s["k_gain"], c, n) for h in range(hkv)], 1)
        for b, table in enumerate(tables):
            for r in range(starts[b], starts[b + 1]):
                at = first[b] + r - starts[b]
                k64[table[at // page], :, at % page] = new[r]
                k[table[at // page], :, at % page] = new[r].to(torch.bfloat16)
        if s["kind"] == "append":
            return q, k64, v64
    else:
        q = s["q"].double()
    out = torch.zeros(rows, hq, D, dtype=torch.float64, device="cuda")
    for b, table in enumerate(tables):
        a, e = starts[b], starts[b + 1]
        for h in range(hkv):
            keys, values = _exact_head(k, v, table, page, h, first[b] + e - a)
            out[a:e, h * g:(h + 1) * g] = _exact_rows(q[a:e, h * g:(h + 1) * g].transpose(0, 1).contiguous(), first[b],
                                                      keys, values, s["window"], s["sinks"]).transpose(0, 1)
    return out if s["kind"] == "prefill" else (out, k64, v64)
