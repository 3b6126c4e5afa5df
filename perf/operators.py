"""The operators of models served in microscaling formats, as cases that can be timed one by one.

Groups of 32 values along a row share a power of two, kept as one byte s (2^(s - 127); 255: the group is no number); the values themselves
are e2m1 numbers of 4 bits (matrices) or e4m3 numbers of 8 bits (rows). A group whose largest magnitude is m 2^x, 1 <= m < 2, takes
s - 127 = x - emax + (1 if m > 1.75 else 0), emax being 2 or 8.

  product: out = act(rows . matrix^T + bias), or stream += rows . matrix^T + bias, the matrix in 4 bits, the rows bfloat16, float32 or in 8 bits
  norm:    stream <- stream + add; its root-mean-square norm (or layer norm) times a weight, in 8 bits
  glu:     act(gate) * up of a feed-forward's first product [gate | up], in 8 bits

`listed()` holds the cases, `draw()` makes others of the same ranges, `prepare()` what a program has in hand before the call, `run()` is one
call, `exact()` what it returns from the definition in 64 bits, `work()` its bytes and operations. 8-bit outputs are the e4m3 numbers of the
rows and the powers of two of their groups.
"""

import math

import torch

own = False  # true: the framework's operators; false: the same in elementary torch operations

# A case's fields. `rows`, `inner`, `features`: a product's sizes; norm and glu have `inner` values a row
FIELDS = {"op": "product", "rows": 1, "inner": 64, "features": 0, "rows_in": "bfloat16", "epilogue": "none", "centred": False, "add": "float32", "activation": "silu"}


def _case(**fields):
    return dict(FIELDS, **fields)


def listed():
    return [
        # one person's chat at GPT-2 medium's sizes: attention's output projection of a single token, added to the stream; latency is all of it
        _case(name="medium_out_1", rows=1, inner=1024, features=1024, epilogue="residual"),
        # the same at width 4,096: a feed-forward's first product, bound by the matrix's bytes
        _case(name="wide_up_1", rows=1, inner=4096, features=16384, epilogue="gelu_tanh"),
        # eight requests at GPT-2 XL's sizes; 1,600 is no multiple of the matrix instruction's 128
        _case(name="xl_up_8", rows=8, inner=1600, features=6400, epilogue="gelu_tanh"),
        # a full server's step: 64 requests, the product back to the model's width
        _case(name="wide_down_64", rows=64, inner=16384, features=4096, epilogue="residual"),
        # a ragged portion of a prompt, rows in 16 bits
        _case(name="wide_up_1999", rows=1999, inner=4096, features=16384, epilogue="gelu_tanh"),
        # the 32-bit path at GPT-2 large's sizes, a few requests
        _case(name="large_up_5_float32", rows=5, inner=1280, features=5120, rows_in="float32"),
        # rows in 8 bits: eight requests, and a step of prompts
        _case(name="wide_out_8_mxfp8", rows=8, inner=4096, features=4096, rows_in="mxfp8", epilogue="residual"),
        _case(name="wide_up_2048_mxfp8", rows=2048, inner=4096, features=16384, rows_in="mxfp8", epilogue="gelu_tanh"),
        # the norm ahead of these: eight requests at XL's width (GPT-2's layer norm), a step of prompts at width 4,096 (a root-mean-square norm)
        _case(name="norm_xl_8", op="norm", rows=8, inner=1600, centred=True),
        _case(name="norm_wide_2048", op="norm", rows=2048, inner=4096, add="bfloat16"),
        # the gate between a feed-forward's products: eight requests, a step of prompts
        _case(name="glu_large_8", op="glu", rows=8, inner=5120),
        _case(name="glu_wide_2048", op="glu", rows=2048, inner=16384, activation="gelu_tanh"),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the ranges above; sizes of every remainder are among them."""
    def size(low, high):
        v = _log_uniform(rng, low, high)
        return v if rng.random() < 0.3 else max(low, v // 64 * 64) if rng.random() < 0.7 else max(low, v // 8 * 8)

    op = rng.choice(["product"] * 4 + ["norm", "glu"])
    if op == "norm":
        return _case(op="norm", rows=_log_uniform(rng, 1, 2048), inner=size(64, 6400), centred=rng.random() < 0.5, add=rng.choice(["float32", "bfloat16", "none"]))
    if op == "glu":
        return _case(op="glu", rows=_log_uniform(rng, 1, 2048), inner=size(64, 16384), activation=rng.choice(["silu", "gelu_tanh"]))
    rows_in = rng.choice(["bfloat16", "bfloat16", "mxfp8", "mxfp8", "float32"])
    rows = _log_uniform(rng, 1, 64) if rng.random() < 0.5 else _log_uniform(rng, 1, 512 if rows_in == "float32" else 1999)
    return _case(rows=rows, inner=size(64, 8192), features=size(64, 8192), rows_in=rows_in, epilogue=rng.choice(["none", "gelu_tanh", "gelu_erf", "residual"]))


# ---------------------------------------------------------------------------------------------------------------
# the formats


def _power(s):
    """2^(s - 127) of bytes s in 1 .. 254, in 32 bits."""
    return (s.to(torch.int32) << 23).view(torch.float32)


def _group_scales(y, emax):
    """The bytes of the groups of y [rows, groups, 32]."""
    bits = y.abs().amax(dim=2).view(torch.int32)
    s = (((bits + 0x1FFFFF) >> 23) - emax).clamp(min=0)
    return torch.where(bits >= 0x7F800000, torch.full_like(s, 255), s)


def _grouped(y):
    rows, width = y.shape
    groups = -(-width // 32)
    return torch.nn.functional.pad(y, (0, groups * 32 - width)).view(rows, groups, 32)


def _mx8(y):
    """float32 rows in 8 bits: (the e4m3 numbers, the groups' bytes)."""
    g = _grouped(y)
    s = _group_scales(g, 8)
    v = g * _power(254 - s.clamp(max=253)).unsqueeze(2)
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=-6).float() - 3)
    v = torch.where((s == 255).unsqueeze(2), torch.zeros_like(v), torch.round(v / step) * step)
    return v.reshape(y.shape[0], -1)[:, : y.shape[1]].to(torch.float8_e4m3fn), s.to(torch.uint8)


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx4(w):
    """float32 rows in 4 bits: (codes, two a byte, the first in the low half; the groups' bytes)."""
    g = _grouped(w)
    s = _group_scales(g, 2)
    v = g * _power(254 - s.clamp(max=253)).unsqueeze(2)
    a, c = v.abs(), torch.zeros_like(v, dtype=torch.uint8)
    for k in range(7):  # ties go to the even code
        half = (E2M1[k] + E2M1[k + 1]) / 2
        c += (a > half) if k % 2 == 0 else (a >= half)
    c = torch.where((s == 255).unsqueeze(2), torch.zeros_like(c), c | ((v < 0).to(torch.uint8) << 3)).reshape(w.shape[0], -1)
    return c[:, 0::2] | (c[:, 1::2] << 4), s.to(torch.uint8)


# ---------------------------------------------------------------------------------------------------------------
# inputs


def _values(gen, rows, width, spread=0.0):
    """Activations: normal, a few channels far larger, rows of different sizes."""
    x = torch.randn(rows, width, generator=gen, device="cuda")
    x *= 1.0 + 9.0 * (torch.rand(width, generator=gen, device="cuda") < 0.01)
    return x * torch.exp(spread * torch.randn(rows, 1, generator=gen, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, d = case["rows"], case["inner"]
    state = {"case": case}
    if case["op"] == "norm":
        state["x"] = _values(gen, n, d, 0.5)
        state["add"] = None if case["add"] == "none" else _values(gen, n, d).to(getattr(torch, case["add"]))
        state["weight"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")
        state["bias"] = 0.1 * torch.randn(d, generator=gen, device="cuda") if case["centred"] else None
        state["stream"] = torch.empty_like(state["x"])
    elif case["op"] == "glu":
        state["gu"] = _values(gen, n, 2 * d)
    else:
        N = case["features"]
        state["codes"], state["scales"] = _mx4(0.02 * torch.randn(N, d, generator=gen, device="cuda"))
        state["bias"] = 0.1 * torch.randn(N, generator=gen, device="cuda")
        a = _values(gen, n, d)
        state["a"] = _mx8(a) if case["rows_in"] == "mxfp8" else a.to(getattr(torch, case["rows_in"]))
        if case["epilogue"] == "residual":
            state["out"] = torch.randn(n, N, generator=gen, device="cuda")
        else:
            state["out"] = torch.empty(n, N, device="cuda", dtype=torch.float32 if case["rows_in"] == "float32" else torch.bfloat16)
    if own:  # the framework's objects around the same data: the matrix as it is laid out once at load, the places of the rows
        from liyab_amd.kernels import mx

        if case["op"] == "product":
            state["matrix"] = mx.Mxfp4Matrix.pack(state.pop("codes"), state.pop("scales"), d)
            if case["rows_in"] == "mxfp8":
                state["a"] = mx.Mxfp8Rows.pack(*state["a"])
        else:
            state["out"] = mx.Mxfp8Rows.empty(n, d)
    return state


# ---------------------------------------------------------------------------------------------------------------
# one call


def _plain_matrix(codes, scales, width):
    c = torch.stack((codes & 15, codes >> 4), dim=2).view(codes.shape[0], -1)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    return (table[c.int()].view(c.shape[0], -1, 32) * _power(scales).unsqueeze(2)).view(c.shape[0], -1)[:, :width]


def _plain_rows(a):
    if isinstance(a, torch.Tensor):
        return a.float()
    codes, scales = a
    return (_grouped(codes.float()) * _power(scales).unsqueeze(2)).view(codes.shape[0], -1)[:, : codes.shape[1]]


def _plain_act(v, name):
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    if name == "gelu_erf":
        return 0.5 * v * (1.0 + torch.erf(v * 0.7071067811865476))
    return v / (1.0 + torch.exp(-v)) if name == "silu" else v


def _run_plain(state):
    case = state["case"]
    if case["op"] == "norm":
        t = state["x"] if state["add"] is None else state["x"] + state["add"].float()
        c = t - t.mean(dim=1, keepdim=True) if case["centred"] else t
        y = c / torch.sqrt((c * c).mean(dim=1, keepdim=True) + 1e-5) * state["weight"]
        codes, scales = _mx8(y + state["bias"] if case["centred"] else y)
        return [codes, scales.view(torch.float8_e8m0fnu), t]
    if case["op"] == "glu":
        gate, up = state["gu"].chunk(2, dim=1)
        codes, scales = _mx8(_plain_act(gate, case["activation"]) * up)
        return [codes, scales.view(torch.float8_e8m0fnu)]
    v = _plain_rows(state["a"]) @ _plain_matrix(state["codes"], state["scales"], case["inner"]).t() + state["bias"]
    if case["epilogue"] == "residual":
        state["out"] += v
    else:
        state["out"].copy_(_plain_act(v, case["epilogue"]))
    return [state["out"]]


def run(state):
    if not own:
        return _run_plain(state)
    from liyab_amd.kernels import mx

    case = state["case"]
    if case["op"] == "norm":
        out, d = state["out"], case["inner"]
        mx.norm_mx(out, state["x"], state["weight"], 1e-5, bias=state["bias"], centred=case["centred"], add=state["add"], stream=state["stream"])
        return [out.codes[:, :d].view(torch.float8_e4m3fn), out.scales[:, : -(-d // 32)].view(torch.float8_e8m0fnu), state["stream"]]
    if case["op"] == "glu":
        out, d = state["out"], case["inner"]
        mx.glu_mx(out, state["gu"], case["activation"])
        return [out.codes[:, :d].view(torch.float8_e4m3fn), out.scales[:, : -(-d // 32)].view(torch.float8_e8m0fnu)]
    if case["epilogue"] == "residual":
        mx.gemm_mx(state["a"], state["matrix"], state["bias"], residual=state["out"])
    else:
        mx.gemm_mx(state["a"], state["matrix"], state["bias"], out=state["out"], activation=case["epilogue"])
    return [state["out"]]


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits


def _exact_rows(y):
    """float64 rows in 8 bits, as the definition says it: the numbers and the powers of two, both in 64 bits."""
    n, d = y.shape
    codes, powers = torch.zeros_like(y), torch.zeros(n, -(-d // 32), dtype=torch.float64, device=y.device)
    padded = torch.zeros(n, powers.shape[1] * 32, dtype=torch.float64, device=y.device)
    padded[:, :d] = y
    amax = padded.view(n, -1, 32).abs().max(dim=2).values
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [1/2, 1)
    e = torch.where(amax > 0, (exponent - 1 - 8 + (mantissa > 0.875).int()).clamp(min=-127), torch.full_like(exponent, -127))
    powers = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=y.device), e.double())
    v = padded / powers.repeat_interleave(32, dim=1)
    lowest = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3  # the exponent of the last place
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=y.device), lowest)
    codes = torch.round(v / unit) * unit
    return codes[:, :d], powers


def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "norm":
        t = state["x"].double() + (0.0 if state["add"] is None else state["add"].double())
        c = t - t.sum(dim=1, keepdim=True) / t.shape[1] if case["centred"] else t
        y = c * state["weight"].double() / ((c ** 2).sum(dim=1, keepdim=True) / t.shape[1] + 1e-5).sqrt()
        return list(_exact_rows(y + state["bias"].double() if case["centred"] else y)) + [t]
    if case["op"] == "glu":
        g, u = state["gu"][:, : case["inner"]].double(), state["gu"][:, case["inner"] :].double()
        return list(_exact_rows((g * torch.sigmoid(g) if case["activation"] == "silu" else torch.nn.functional.gelu(g, approximate="tanh")) * u))
    low, high = state["codes"].long() & 15, state["codes"].long() >> 4
    c = torch.zeros(low.shape[0], 2 * low.shape[1], dtype=torch.long, device=low.device)
    c[:, 0::2], c[:, 1::2] = low, high
    m, e = c & 1, (c >> 1) & 3  # e2m1: m/2 where the exponent is 0, else (1 + m/2) 2^(e - 1)
    w = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * (1 << e) / 2.0).double() * (1 - 2 * (c >> 3)).double()
    w *= torch.pow(torch.tensor(2.0, dtype=torch.float64, device=w.device), state["scales"].double() - 127).repeat_interleave(32, dim=1)
    if case["rows_in"] == "mxfp8":
        codes, scales = state["a"]
        a = codes.double() * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=w.device), scales.double() - 127).repeat_interleave(32, dim=1)[:, : codes.shape[1]]
    else:
        a = state["a"].double()
    v = a @ w[:, : case["inner"]].t() + state["bias"].double()
    if case["epilogue"] == "residual":
        return [state["out"].double() + v]
    if case["epilogue"] == "none":
        return [v]
    return [torch.nn.functional.gelu(v, approximate="tanh" if case["epilogue"] == "gelu_tanh" else "none")]


def _inputs(case, seed):
    """The inputs alone, whichever side is run."""
    global own
    before, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = before


# ---------------------------------------------------------------------------------------------------------------
# what a call cannot do without


def work(case):
    n, d, N = case["rows"], case["inner"], case["features"]
    eighth = d + -(-d // 32)  # bytes of a row in 8 bits
    if case["op"] == "norm":
        add = {"none": 0, "float32": 4, "bfloat16": 2}[case["add"]]
        return {"bytes": n * (d * (4 + add + 4) + eighth) + 4 * d * (2 if case["centred"] else 1), "flops": 8 * n * d}
    if case["op"] == "glu":
        return {"bytes": n * (8 * d + eighth), "flops": 12 * n * d}
    row = {"bfloat16": 2 * d, "float32": 4 * d, "mxfp8": eighth}[case["rows_in"]]
    out = 8 if case["epilogue"] == "residual" else 4 if case["rows_in"] == "float32" else 2
    return {"bytes": N * (-(-d // 2) + -(-d // 32)) + 4 * N + n * row + n * N * out, "flops": 2 * n * N * d}
