"""The 8-bit linear layers as measured work: rows quantised to 8 bits with a
scale for each token (alone, and as the output of residual + RMSNorm), and the
matrix product of such rows with 8-bit weights that have a scale for each
channel, with its bias / residual / gated epilogues.

Every case runs in two ways on the same inputs: ``own`` False computes the
operator from elementary torch operations in 32 bits (64 for the quantiser,
where a rounding decides a code), ``own`` True calls
:mod:`llamamps_b200.kernels`.

A row of k fp16 elements is held as k signed codes in [-127, 127] and one fp32
scale, max|row| / 127 (code 0 and scale 0 for a zero row); rows of codes start
at multiples of 16 bytes.
"""
import math
import random

import torch

own = False

TOP = 127.0
EPS = 1e-6
# output channels and inner length of the projections: q|k|v, o, down, and one rank's shares of them in the two-way
# split; then a vocabulary slice and sizes that divide nothing
LINEAR = [(2048, 1536), (1536, 1536), (1536, 8960), (1024, 1536), (1536, 768), (1536, 4480), (8192, 1536), (4097, 1535),
          (333, 1201), (129, 272)]
# gated output channels and inner length: the whole feed-forward block, one rank's half, odd ones
GATED = [(8960, 1536), (4480, 1536), (1537, 1000), (200, 333)]
ROW = [1536, 1536, 768, 8960, 4480, 1535, 2048, 333, 9000]  # elements of a quantised row


# -- cases ---------------------------------------------------------------------
def listed():
    return [
        # the norm before a projection, one decoded token: the latency case
        dict(name="norm 1x1536", op="norm", rows=1, k=1536, residual=False),
        # a decode batch of 64: the o projection's output joins the residual stream, then the norm
        dict(name="norm+residual 64x1536", op="norm", rows=64, k=1536, residual=True),
        # the same for the benchmark's prefill, 8 prompts of 2048
        dict(name="norm+residual 16384x1536", op="norm", rows=16384, k=1536, residual=True),
        # the activations before the down projection, a decode batch
        dict(name="quantise 64x8960", op="quantise", rows=64, k=8960),
        # the same for the benchmark's prefill: the bandwidth case
        dict(name="quantise 16384x8960", op="quantise", rows=16384, k=8960),
        # q|k|v of one decoded token
        dict(name="gemm+bias 1x2048x1536", op="gemm", rows=1, n=2048, k=1536, add="bias"),
        # the down projection of a decode batch
        dict(name="gemm+residual 64x1536x8960", op="gemm", rows=64, n=1536, k=8960, add="residual"),
        # a short prompt against sizes that divide nothing
        dict(name="gemm 201x4097x1535", op="gemm", rows=201, n=4097, k=1535, add="none"),
        # the down projection of the benchmark's prefill
        dict(name="gemm+residual 16384x1536x8960", op="gemm", rows=16384, n=1536, k=8960, add="residual"),
        # gate and up projections with the gated activation: one token, a decode batch, the benchmark's prefill
        dict(name="gated 1x8960x1536", op="gated", rows=1, n=8960, k=1536),
        dict(name="gated 64x8960x1536", op="gated", rows=64, n=8960, k=1536),
        dict(name="gated 16384x8960x1536", op="gated", rows=16384, n=8960, k=1536),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for kind in w:
            most[kind] = max(most.get(kind, 0), w[kind])
    while True:
        op = rng.choice(["norm", "quantise", "gemm", "gemm", "gated"])
        c = dict(op=op, rows=_log_int(rng, 1, 16384))
        if op in ("gemm", "gated"):
            c["n"], c["k"] = rng.choice(LINEAR if op == "gemm" else GATED)
            if rng.random() < 0.4:  # other models' widths
                c["n"], c["k"] = _log_int(rng, 64, 12000), _log_int(rng, 64, 9000)
            if op == "gemm":
                c["add"] = rng.choice(["none", "bias", "residual", "both"])
        else:
            c["k"] = rng.choice(ROW) if rng.random() < 0.6 else _log_int(rng, 8, 9000)
            if op == "norm":
                c["residual"] = rng.random() < 0.5
        same = [d for d in listed() if {**d, "name": None} == {**c, "name": None}]
        if not same and all(work(c)[kind] <= most[kind] for kind in most):
            return c


def work(case):
    m, k = case["rows"], case["k"]
    if case["op"] in ("norm", "quantise"):
        # fp16 rows in; codes, scales and the values of the codes out
        b = m * (2 * k + k + 4 + 2 * k)
        if case["op"] == "norm":
            b += 2 * k + (4 * m * k if case["residual"] else 0)  # gamma; the residual in, the sum out
        return {"bytes": b, "flops": 8 * m * k}
    n = case["n"]
    w = 2 * n if case["op"] == "gated" else n
    b = m * (k + 4) + w * (k + 4) + 2 * m * n  # codes and scales in, fp16 out
    add = case.get("add", "none")
    b += (2 * n if add in ("bias", "both") else 0) + (2 * m * n if add in ("residual", "both") else 0)
    return {"bytes": b, "flops": 2 * m * w * k}


# -- inputs ------------------------------------------------------------------------
def _codes(gen, rows, k, dev):
    """Codes as quantised rows have them, bell-shaped with the row's largest element at 127, rows padded to 16 bytes."""
    x = torch.empty(rows, -(-k // 16) * 16, dtype=torch.int8, device=dev)
    for a in range(0, rows, 4096):
        part = x[a:a + 4096]
        g = torch.randn(part.shape, generator=gen, device=dev)
        part.copy_((g * 34.0).round_().clamp_(-TOP, TOP))
    return x[:, :k]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    m, k, op = case["rows"], case["k"], case["op"]
    s = dict(case=dict(case))
    half = dict(dtype=torch.float16, device=dev)
    if op in ("norm", "quantise"):
        x = torch.randn(m, k, generator=gen, device=dev)
        if op == "quantise":  # products of a gate and an up value: long tails
            x = x * torch.randn(m, k, generator=gen, device=dev)
        else:  # a few channels of the residual stream are far larger than the rest
            x = x * (1.0 + 20.0 * (torch.rand(k, generator=gen, device=dev) < 0.004).float())
        if m >= 16:  # a padding row
            x[m // 3] = 0
        s["x"] = x.half()
        ld = -(-k // 16) * 16
        s["codes"] = torch.zeros(m, ld, dtype=torch.int8, device=dev)[:, :k]
        s["scales"] = torch.zeros(m, dtype=torch.float32, device=dev)
        s["values"] = torch.zeros(m, k, **half)
        if op == "norm":
            s["gamma"] = (1.0 + 0.25 * torch.randn(k, generator=gen, device=dev)).half()
            if case["residual"]:
                s["residual"] = (4.0 * torch.randn(m, k, generator=gen, device=dev)).half()
                s["sum"] = torch.zeros(m, k, **half)
        return s
    n = case["n"]
    w = 2 * n if op == "gated" else n
    s["x"], s["w"] = _codes(gen, m, k, dev), _codes(gen, w, k, dev)
    # tokens differ in size by some e^+-1, channels less
    s["x_scales"] = 0.03 * torch.exp(0.5 * torch.randn(m, generator=gen, device=dev))
    s["w_scales"] = 0.0008 * torch.exp(0.2 * torch.randn(w, generator=gen, device=dev))
    if case.get("add") in ("bias", "both"):
        s["bias"] = torch.randn(n, generator=gen, device=dev).half()
    if case.get("add") in ("residual", "both"):
        s["residual"] = torch.randn(m, n, generator=gen, device=dev).half()
    s["out"] = torch.zeros(m, n, **half)
    s["error"] = torch.zeros(1, dtype=torch.int32, device=dev)
    return s


# -- the plain forms -----------------------------------------------------------------
def _quantise(y, s):
    """fp64 rows as codes, scales and values, into the state's buffers."""
    top = y.abs().amax(dim=1, keepdim=True)
    code = torch.where(top > 0, torch.round(y / top * TOP), torch.zeros((), dtype=y.dtype, device=y.device))
    scale = top / TOP
    s["codes"].copy_(code)
    s["scales"].copy_(scale[:, 0])
    s["values"].copy_(code * scale)
    return s["values"], s["scales"]


def _plain(s):
    c = s["case"]
    if c["op"] == "quantise":
        return _quantise(s["x"].double(), s)
    if c["op"] == "norm":
        x = s["x"]
        if c["residual"]:
            x = (s["residual"].float() + x.float()).half()
            s["sum"].copy_(x)
        x = x.double()
        y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * s["gamma"].double()
        return _quantise(y, s) + ((s["sum"],) if c["residual"] else ())
    acc = torch.matmul(s["x"].float(), s["w"].float().t())
    acc *= s["x_scales"][:, None]
    acc *= s["w_scales"]
    if c["op"] == "gated":
        g, u = acc[:, :c["n"]], acc[:, c["n"]:]
        acc = g / (1.0 + torch.exp(-g)) * u
    if "bias" in s:
        acc += s["bias"].float()
    if "residual" in s:
        acc += s["residual"].float()
    s["out"].copy_(acc)
    return s["out"]


# -- the framework's calls -------------------------------------------------------------
def _framework(s):
    from llamamps_b200 import kernels as K

    c = s["case"]
    if c["op"] == "quantise":
        K.quantise_rows_q8(s["x"], codes=s["codes"], scales=s["scales"], values=s["values"])
        return s["values"], s["scales"]
    if c["op"] == "norm":
        if c["residual"]:
            K.rms_norm_q8(s["x"], s["gamma"], EPS, residual=s["residual"], sum_out=s["sum"], codes=s["codes"],
                          scales=s["scales"], values=s["values"])
            return s["values"], s["scales"], s["sum"]
        K.rms_norm_q8(s["x"], s["gamma"], EPS, codes=s["codes"], scales=s["scales"], values=s["values"])
        return s["values"], s["scales"]
    return K.w8a8_gemm(s["x"], s["x_scales"], s["w"], s["w_scales"], bias=s.get("bias"), residual=s.get("residual"),
                       swiglu=c["op"] == "gated", out=s["out"], error=s["error"])


def run(state):
    return _framework(state) if own else _plain(state)


# -- 64 bits -----------------------------------------------------------------------------
def _exact_rows(y):
    """What 8-bit rows of fp64 y stand for, and their scales: the grid of 127 steps up to the row's largest element."""
    values, scales = torch.zeros_like(y), torch.zeros(y.shape[0], dtype=torch.float64, device=y.device)
    for a in range(0, y.shape[0], 2048):
        part = y[a:a + 2048]
        step = torch.maximum(part.max(dim=1).values, -part.min(dim=1).values) / TOP
        live = step > 0
        at = torch.where(live, step, torch.ones_like(step))[:, None]
        values[a:a + 2048] = torch.round(part / at) * at
        scales[a:a + 2048] = step
    return values, scales


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantise":
        return _exact_rows(s["x"].to(torch.float64))
    if op == "norm":
        x, total = s["x"].to(torch.float64), ()
        if case["residual"]:
            x = s["x"].to(torch.float64) + s["residual"].to(torch.float64)
            total = (x,)
            x = x.to(torch.float16).to(torch.float64)  # the norm is of the rounded residual stream
        size = torch.sqrt(torch.einsum("mk,mk->m", x, x) / case["k"] + EPS)
        return _exact_rows(x / size[:, None] * s["gamma"].to(torch.float64)) + total
    n = case["n"]
    out = torch.empty(case["rows"], n, dtype=torch.float64, device=s["x"].device)
    w = s["w"].to(torch.float64) * s["w_scales"].to(torch.float64)[:, None]
    for a in range(0, case["rows"], 2048):
        x = s["x"][a:a + 2048].to(torch.float64) * s["x_scales"][a:a + 2048].to(torch.float64)[:, None]
        if op == "gated":
            gate = x @ w[:n].T
            out[a:a + 2048] = gate * torch.sigmoid(gate) * (x @ w[n:].T)
            continue
        y = x @ w.T
        if "bias" in s:
            y = y + s["bias"].to(torch.float64)
        if "residual" in s:
            y = y + s["residual"][a:a + 2048].to(torch.float64)
        out[a:a + 2048] = y
    return out
