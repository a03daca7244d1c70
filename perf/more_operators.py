"""Timed cases of block-scaled 8- and 4-bit rows: quantisation, norm, product.

The matrix cores multiply rows of 8-bit (e4m3) or 4-bit (e2m1) values that carry
one power-of-two scale (e8m0) per 32 values. A decoder that keeps its weights in
4 bits that way quantises them once when it loads, turns each projection's input
into 8 or 4 bits (the attention's and the SwiGLU's outputs as they are, the
residual stream through its norm), and multiplies. A case is one call of one of
these operators at the widths of the 3072-wide and the 2048-wide decoder, from a
single token to long prompts.

What is held in 8 bits is returned as tensors of those types (values and scales
apart), what is held in 4 bits as the bfloat16 values that it stands for.

`own` False: the operators in elementary torch operations in 32 bits. `own`
True: the library's calls.
"""
import importlib
import math

import torch

own = False

EPS = 1e-5
BLOCK = 32  # values of a scale
TOP = {8: 8, 4: 2}  # exponent of the largest value of a type: 448 = 1.75 * 2^8, 6 = 1.5 * 2^2
MOST_VALUES = 16384 * 3072  # of a drawn quantisation or norm: no more than the listed ones


def listed():
    return [
        # a token's attention output before the output projection: the smallest call, its latency is the step's
        dict(name="quantize8_1", kind="quantize", bits=8, rows=1, k=3072),
        # the SwiGLU outputs of the benchmark's long prompt, before the down projection
        dict(name="quantize8_3000", kind="quantize", bits=8, rows=3000, k=8192),
        # a ragged prompt's rows in 4 bits, and back
        dict(name="quantize4_517", kind="quantize", bits=4, rows=517, k=2048),
        # the gate/up weights when a model loads, and back
        dict(name="quantize4_weights", kind="quantize", bits=4, rows=16384, k=3072),
        # a token's residual stream before QKV
        dict(name="norm8_1", kind="norm", bits=8, rows=1, k=3072, residual=True),
        # the long prompt's
        dict(name="norm8_3000", kind="norm", bits=8, rows=3000, k=3072, residual=True),
        # QKV of one token: latency and the stream of the weights
        dict(name="gemm_1_qkv", kind="gemm", bits=8, m=1, n=5120, k=3072, epilogue="store"),
        # gate/up of a full batch's decode step
        dict(name="gemm_8_gate_up", kind="gemm", bits=8, m=8, n=16384, k=3072, epilogue="swiglu"),
        # the output layer of a few takes: the largest weights
        dict(name="gemm_5_lm_head", kind="gemm", bits=8, m=5, n=83968, k=3072, epilogue="store"),
        # the down projection of a short prompt, into the residual stream
        dict(name="gemm_197_down", kind="gemm", bits=8, m=197, n=3072, k=8192, epilogue="residual"),
        # gate/up of the long prompt
        dict(name="gemm_3000_gate_up", kind="gemm", bits=8, m=3000, n=16384, k=3072, epilogue="swiglu"),
        # several prompts at once with 4-bit activations, 2048 wide
        dict(name="gemm4_6001_gate_up", kind="gemm", bits=4, m=6001, n=12288, k=2048, epilogue="swiglu"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("quantize", "norm", "gemm", "gemm"))
    if kind != "gemm":
        k = BLOCK * _log_int(rng, 1, 256)
        rows = _log_int(rng, 1, min(24576, MOST_VALUES // k))
        if kind == "quantize":
            return dict(kind=kind, bits=rng.choice((8, 4)), rows=rows, k=k)
        return dict(kind=kind, bits=8, rows=rows, k=k, residual=rng.random() < 0.7)
    epilogue = rng.choice(("store", "residual", "swiglu"))
    m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 1, 20000), 128 * _log_int(rng, 1, 64)
    n += n % 2 if epilogue == "swiglu" else 0
    while 2 * m * n * k > 3e11:  # no more than the listed ones
        m = m * 2 // 3
    return dict(kind=kind, bits=rng.choice((8, 8, 4)), m=m, n=n, k=k, epilogue=epilogue)


def _row_bytes(k, bits):
    """Bytes of a row's codes and scales."""
    return k * bits // 8 + k // BLOCK


def work(case):
    c = case
    if c["kind"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        out = {"store": m * n, "residual": 2 * m * n, "swiglu": m * n // 2}[c["epilogue"]]
        return {"bytes": m * _row_bytes(k, c["bits"]) + n * _row_bytes(k, 4) + 2 * out, "flops": 2 * m * n * k}
    rows, k = c["rows"], c["k"]
    if c["kind"] == "norm":
        return {"bytes": rows * ((6 if c["residual"] else 2) * k + _row_bytes(k, c["bits"])) + 2 * k,
                "flops": 8 * rows * k}
    if c["bits"] == 8:
        return {"bytes": rows * (2 * k + _row_bytes(k, 8)), "flops": 4 * rows * k}
    return {"bytes": 2 * rows * (2 * k + _row_bytes(k, 4)), "flops": 5 * rows * k}  # there and back


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _normal(g, *shape, mean=0.0, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean)


def _activations(g, rows, k):
    """A residual stream's rows: some channels many times the others."""
    return _normal(g, rows, k).mul_(_normal(g, k).mul_(0.8).exp_()).to(torch.bfloat16)


def prepare(case, seed):
    c = dict(case)
    g = _gen(seed)
    if c["kind"] == "quantize":
        c["x"] = _normal(g, c["rows"], c["k"], std=0.02).to(torch.bfloat16) if c["rows"] > 10000 else _activations(
            g, c["rows"], c["k"])
        return c
    if c["kind"] == "norm":
        c["x"], c["gain"] = _activations(g, c["rows"], c["k"]), _normal(g, c["k"], mean=1.0, std=0.2).to(torch.bfloat16)
        c["stream"] = _activations(g, c["rows"], c["k"]) if c["residual"] else None
        return c
    m, n, k = c["m"], c["n"], c["k"]
    c["a"] = _packed(_activations(g, m, k), c["bits"])
    c["w"] = _packed(_normal(g, n, k, std=0.02).to(torch.bfloat16), 4)
    c["stream"] = _normal(g, m, n, std=2.0).to(torch.bfloat16) if c["epilogue"] == "residual" else None
    return c


# ---- the plain forms ----

def _power(e):
    """2^e in 32 bits, for integers from -126 to 127."""
    return ((e + 127) << 23).view(torch.float32)


def _plain_quantize(x, bits):
    """x [rows, k] in 32 bits -> (the values of the codes, the scales' exponents [rows, k / 32])."""
    x = x.view(x.shape[0], -1, BLOCK)
    top = x.abs().amax(-1)
    e = ((top.view(torch.int32) >> 23) - 127 - TOP[bits]).clamp(min=-127)
    x = x * _power(-e)[..., None]
    if bits == 8:
        q = x.clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        a = x.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        q = torch.copysign(((a / step).round() * step).clamp(max=6), x)
    return q.view(x.shape[0], -1), e


def _packed(x, bits):
    """The codes and scales of rows x as a program holds them."""
    q, e = _plain_quantize(x.float(), bits)
    scales = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    if bits == 8:
        return q, scales
    a = q.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | torch.signbit(q).byte() << 3
    return code[:, 0::2] | code[:, 1::2] << 4, scales


def _values(packed):
    """The values in 32 bits of codes [rows, k] in 8 bits, or [rows, k / 2] in 4 bits, with their scales."""
    codes, scales = packed
    if codes.dtype == torch.uint8:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
        codes = table[torch.stack((codes & 15, codes >> 4), -1).int()]
    rows = scales.shape[0]
    return (codes.float().view(rows, -1, BLOCK) * scales.float()[..., None]).view(rows, -1)


def _plain_returned(x, bits):
    q, e = _plain_quantize(x, bits)
    if bits == 8:
        return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    return (q.view(*e.shape, BLOCK) * _power(e)[..., None]).view(q.shape).to(torch.bfloat16)


def _plain_norm(s):
    x, h = s["x"].float(), None
    if s["residual"]:
        h = (x + s["stream"].float()).to(torch.bfloat16)
        x = h.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["gain"].float()
    return h, _plain_returned(y, s["bits"])


def _plain_gemm(s):
    y = _values(s["a"]) @ _values(s["w"]).T
    if s["epilogue"] == "residual":
        y = y + s["stream"].float()
    elif s["epilogue"] == "swiglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(torch.bfloat16)


# ---- the library's calls ----

def _library():
    return importlib.import_module("yue2-mlx_amd.yuear")


def _own_quantize(s):
    y = _library()
    packed = y.mx_quantize(s["x"], s["bits"])
    return packed if s["bits"] == 8 else y.mx_dequantize(packed)


def _own_norm(s):
    packed, h = _library().mx_rms_norm(s["x"], s["gain"], EPS, residual=s["stream"], bits=s["bits"])
    return h, packed


def _own_gemm(s):
    return _library().mx_gemm(s["a"], s["w"], residual=s["stream"], swiglu=s["epilogue"] == "swiglu")


def run(state):
    kind = state["kind"]
    if own:
        return dict(quantize=_own_quantize, norm=_own_norm, gemm=_own_gemm)[kind](state)
    if kind == "quantize":
        return _plain_returned(state["x"].float(), state["bits"])
    return dict(norm=_plain_norm, gemm=_plain_gemm)[kind](state)


# ---- the definition in 64 bits ----

def _exact_power(e):
    """2^e by its bits: pow() may be half a step off, and ties with it."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_grid(bits):
    """The magnitudes of a type in order of their codes."""
    mantissa, bias = (3, 7) if bits == 8 else (1, 1)
    steps = 1 << mantissa
    grid = [(c % steps + (steps if c >= steps else 0)) / steps * 2.0 ** (max(c // steps, 1) - bias)
            for c in range(127 if bits == 8 else 8)]
    return torch.tensor(grid, dtype=torch.float64, device="cuda")


def _exact_block(x, bits):
    """(values of the codes, scales) of x [rows, k] in 64 bits: the nearest of the grid, ties to the even code."""
    rows, k = x.shape
    x = x.reshape(rows, k // BLOCK, BLOCK)
    exponent = torch.frexp(x.abs().max(-1).values).exponent - 1 - TOP[bits]
    scale = _exact_power(exponent.clamp(min=-127))
    scale[x.abs().max(-1).values == 0] = 2.0 ** -127
    x = x / scale[..., None]
    grid = _exact_grid(bits)
    middle = (grid[1:] + grid[:-1]) / 2
    a = x.abs()
    at = torch.searchsorted(middle, a)
    tied = a == middle[at.clamp(max=middle.numel() - 1)]
    at = at + (tied & (at % 2 == 1)).long()
    return torch.where(x < 0, -grid[at], grid[at]).reshape(rows, k), scale


def _exact_returned(x, bits):
    q, scale = _exact_block(x, bits)
    return (q, scale) if bits == 8 else q * scale.repeat_interleave(BLOCK, 1)


def _exact_codes(packed):
    codes, scales = packed
    scale = _exact_power(scales.view(torch.uint8).long() - 127)
    if codes.dtype != torch.uint8:
        return codes.double() * scale.repeat_interleave(BLOCK, 1)
    grid, q = _exact_grid(4), torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device="cuda")
    for half, nibble in enumerate((codes % 16, codes // 16)):
        value = grid[(nibble % 8).long()]
        q[:, half::2] = torch.where(nibble >= 8, -value, value)
    return q * scale.repeat_interleave(BLOCK, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "quantize":
        return _exact_returned(s["x"].double(), s["bits"])
    if s["kind"] == "norm":
        x, h = s["x"].double(), None
        if s["residual"]:
            h = x + s["stream"].double()
            x = h.to(torch.bfloat16).double()  # the norm is that of the sum as it is kept
        y = x / ((x ** 2).sum(-1, keepdim=True) / s["k"] + EPS).sqrt() * s["gain"].double()
        return h, _exact_returned(y, s["bits"])
    y = _exact_codes(s["a"]) @ _exact_codes(s["w"]).T.contiguous()
    if s["epilogue"] == "residual":
        return y + s["stream"].double()
    if s["epilogue"] == "swiglu":
        return y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2]
    return y
