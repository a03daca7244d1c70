"""Plain 64-bit forms of the paged cache operators, and their error bounds.

Keys and values are plain arrays of a sequence here ([kv heads, n, 128]); the
page layout is in `gather` and `Pages` alone. Bounds count roundings by half
steps of bf16, 2^-8 of a value, and of fp32, 2^-24.
"""
import numpy as np
import torch

D = 128
HALF = 2.0 ** -8    # half a step of bf16, relative
FINE = 2.0 ** -20   # a few fp32 roundings, relative to the sum of magnitudes


def turn(x, gain, cos, sin, eps):
    """rope(norm(x)) of rows [..., 128] in 64 bits, and the magnitude that its
    fp32 roundings are relative to."""
    x = x.double()
    if gain is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    c, s = cos.double(), sin.double()
    a, b = x[..., :64], x[..., 64:]
    y = torch.cat((a * c - b * s, b * c + a * s), -1)
    size = torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), -1)
    return y, size


def visible(p, n, window, sinks):
    """Which of n keys position p sees."""
    t = np.arange(n)
    seen = t <= p
    if window:
        seen &= (p - t < window) | (t < sinks)
    return seen


def gather(k_pages, v_pages, table_row, n):
    """(keys, values, present) of a sequence's first n keys in 64 bits: [kv
    heads, n, 128] and [n]; zeros where the table has no page."""
    pages, hkv, slots, _ = k_pages.shape
    k = torch.zeros(hkv, n, D, dtype=torch.float64, device=k_pages.device)
    v = torch.zeros_like(k)
    present = np.zeros(n, bool)
    for j in range((n + slots - 1) // slots):
        page, a, b = int(table_row[j]), j * slots, min(n, (j + 1) * slots)
        if 0 <= page < pages:
            k[:, a:b] = k_pages[page, :, :b - a].double()
            rows = v_pages[page].transpose(-1, -2).reshape(hkv, slots, D)
            v[:, a:b] = rows[:, :b - a].double()
            present[a:b] = True
    return k, v, present


def attend(q, k, v, seen, p_half):
    """Attention of queries q [heads, 128] over keys and values [kv heads, n,
    128], `seen` [n]: the result and its error bound. p_half: rounding of a
    weight (the denominator sums the same rounded weights)."""
    hkv = k.shape[0]
    g = q.shape[0] // hkv
    at = torch.from_numpy(np.flatnonzero(seen)).to(k.device)
    if at.numel() == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    kk, vv = k[:, at], v[:, at]
    qq = q.reshape(hkv, g, D)
    score = qq @ kk.transpose(1, 2) / D ** 0.5
    size = (qq.abs() @ kk.abs().transpose(1, 2) / D ** 0.5).amax(-1, keepdim=True)
    w = torch.softmax(score, -1)
    out = w @ vv
    # sum w (1 + d) v / sum w (1 + d), |d| <= p_half + fp32 errors of scores and sums
    spread = (w[..., None] * (vv[:, None] - out[:, :, None]).abs()).sum(2)
    mass = w @ vv.abs()
    bound = HALF * out.abs() + 1.02 * p_half * spread + (2.0 ** -17) * (1 + size) * mass + 1e-30
    return out.reshape(-1, D), bound.reshape(-1, D)


def check(got, want, bound, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float((err / bound)[bad].max()))


class Pages:
    """A pool's tensors on `device`, every slot a NaN until it is written."""

    def __init__(self, pages, kv_heads, slots, device, fill=float("nan")):
        self.k = torch.full((pages, kv_heads, slots, D), fill, dtype=torch.bfloat16, device=device)
        self.v = torch.full((pages, kv_heads, slots // 32, D, 32), fill, dtype=torch.bfloat16, device=device)
        self.slots = slots

    def put(self, table_row, t0, k, v):
        """Keys and values [kv heads, n, 128] at positions t0, t0 + 1, ..."""
        n = k.shape[1]
        for j in range(t0 // self.slots, (t0 + n - 1) // self.slots + 1):
            page = int(table_row[j])
            if page < 0:
                continue
            a, b = max(t0, j * self.slots), min(t0 + n, (j + 1) * self.slots)
            sa, sb = a - j * self.slots, b - j * self.slots
            self.k[page, :, sa:sb] = k[:, a - t0:b - t0]
            rows = self.v[page].transpose(-1, -2).reshape(-1, self.slots, D).clone()
            rows[:, sa:sb] = v[:, a - t0:b - t0]
            self.v[page] = rows.reshape(-1, self.slots // 32, 32, D).transpose(-1, -2)


def tables(lengths, slots, pages, rng, width=None):
    """Random distinct pages for sequences of these lengths: int32 [n, width], -1
    past each sequence."""
    need = [(n + slots - 1) // slots for n in lengths]
    width = max(need + [1]) if width is None else width
    ids = rng.permutation(pages)[:sum(need)]
    out = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        out[b, :n] = ids[at:at + n]
        at += n
    return out
