"""Products grouped by expert, their gradients, and products with 4-bit weights and group scales, as cases that can be timed
and compared.

Five kinds, each through the entry point that a program calls:
  linear    G4Linear.run (4-bit weights with group scales, 16-bit rows)
  experts4  grouped_mm over a G4Tensor (rows sorted by expert, 4-bit weights)
  grouped   grouped_mm (rows sorted by expert, 16-bit weights)
  dx        grouped_mm_dx (gradient of the rows)
  dw        grouped_mm_dw (gradient of the weights)

Rows ends[e - 1] .. ends[e] - 1 (from 0 for e = 0) belong to expert e; rows behind the last end belong to none, and a result
that the call allocates is 0 there. 4-bit weights are w = (q - z) s with whole numbers q and z from 0 to 15 (z = 8 where none are
given) and one 16-bit scale s, one z for each `group` neighbouring inputs; two q to a byte, the even one in the low half.
"""
import importlib
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode token through one projection: the smallest call, all latency
        dict(name="linear_token", kind="linear", rows=1, k=4096, n=4096, group=128, zeros=False, bias=False, dtype="bf16",
             out="bf16"),
        # a verify block of 6 tokens through the widest projection of a 31B-class dense model, scales and zeros per 64
        dict(name="linear_verify", kind="linear", rows=6, k=5376, n=21504, group=64, zeros=True, bias=False, dtype="fp16",
             out="fp32"),
        # a ragged prompt through that projection, with a bias
        dict(name="linear_prompt", kind="linear", rows=1021, k=5376, n=21504, group=128, zeros=False, bias=True, dtype="bf16",
             out="bf16"),
        # one decode token's ten picks of many small experts, gate and up in one
        dict(name="experts4_token", kind="experts4", rows=10, E=512, k=2048, n=1024, group=32, zeros=False, pad=0,
             dtype="fp16", out="fp16"),
        # a prefill chunk (1024 tokens, ten picks each) through the down projections of many small experts
        dict(name="experts4_prompt", kind="experts4", rows=10240, E=512, k=640, n=2560, group=128, zeros=False, pad=0,
             dtype="bf16", out="bf16"),
        # one decode token's ten picks, 16-bit experts
        dict(name="grouped_token", kind="grouped", rows=10, E=512, k=2048, n=1024, pad=0, dtype="bf16", out="bf16"),
        # a short prompt: a few rows for each of many experts, padding behind them
        dict(name="grouped_short", kind="grouped", rows=2085, E=512, k=2560, n=1280, pad=27, dtype="fp16", out="fp16"),
        # one GPU's share of wide experts in a training batch, gate and up in one: the largest call
        dict(name="grouped_batch", kind="grouped", rows=16384, E=16, k=7168, n=4096, pad=0, dtype="bf16", out="bf16"),
        # the rows' gradient of a small ragged batch
        dict(name="dx_small", kind="dx", rows=1013, E=64, k=2048, n=1024, pad=11, dtype="fp16", out="fp16"),
        # the rows' gradient of the training batch
        dict(name="dx_batch", kind="dx", rows=16384, E=16, k=7168, n=4096, pad=0, dtype="bf16", out="bf16"),
        # the weights' gradient of a small ragged batch, kept in 32 bits
        dict(name="dw_small", kind="dw", rows=1013, E=64, k=2048, n=1024, pad=11, dtype="bf16", out="fp32"),
        # the weights' gradient of the training batch
        dict(name="dw_batch", kind="dw", rows=16384, E=16, k=7168, n=4096, pad=0, dtype="bf16", out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(("linear", "experts4", "grouped", "dx", "dw"))
        t = rng.choice(("fp16", "bf16"))
        c = dict(kind=kind, dtype=t, out=rng.choice((t, t, "fp32")))
        if kind in ("linear", "experts4"):
            c["group"] = rng.choice((32, 64, 128))
            c["k"] = c["group"] * max(1, _log(rng, 512, 8192) // c["group"])
            c["zeros"] = rng.random() < 0.5
        else:
            c["k"] = 8 * _log(rng, 64, 896) if rng.random() < 0.75 else _log(rng, 512, 7168)
        if kind == "linear":
            c["rows"], c["bias"] = _log(rng, 1, 1024), rng.random() < 0.3
            c["n"] = 32 * _log(rng, 16, 672) if rng.random() < 0.75 else _log(rng, 512, 21504)
        else:
            c["E"] = rng.choice((8, 16, 32, 64, 128, 256, 512))
            c["rows"] = _log(rng, 1, 16384)
            c["n"] = 8 * _log(rng, 64, 896) if rng.random() < 0.75 else _log(rng, 512, 7168)
            c["pad"] = rng.choice((0, 0, rng.randrange(1, 64)))
        # no dearer than the largest listed ones: operations, and weights to make, read or write
        size = c["k"] * c["n"] * c.get("E", 1)
        if work(c)["flops"] > (2.4e11 if kind == "linear" else 9.7e11) or size > (8.4e8 if kind == "experts4" else 1.7e9 if kind == "grouped" else 4.8e8):
            continue
        return c


# ------------------------------------------------------------------------------------------------ work
def work(case):
    """Bytes: the weights of every expert that rows are expected to touch once (dw: every expert's gradient), rows in and out
    once. Operations: the products."""
    c, r, k, n = case, case["rows"], case["k"], case["n"]
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    per = 0.5 + (3 if c["zeros"] else 2) / c["group"] if "group" in c else 2.0
    touched = c["E"] * (1 - (1 - 1 / c["E"]) ** r) if "E" in c else 1
    if c["kind"] == "dw":
        return {"bytes": 2.0 * r * (k + n) + size[c["out"]] * c["E"] * k * n, "flops": 2.0 * r * k * n}
    rows_in, rows_out = (n, k) if c["kind"] == "dx" else (k, n)
    return {"bytes": touched * per * k * n + 2.0 * r * rows_in + size[c["out"]] * r * rows_out, "flops": 2.0 * r * k * n}


# ------------------------------------------------------------------------------------------------ the plain forms
def _weights(s, e=None):
    """fp32 weights [..., n, k] of all experts, or of those that e picks."""
    if "codes" not in s:
        return (s["w"] if e is None else s["w"][e]).float()
    codes, scales, zeros = (t if t is None or e is None else t[e] for t in (s["codes"], s["scales"], s["zeros"]))
    q = torch.stack((codes & 15, codes >> 4), -1).reshape(*scales.shape, -1).float()
    z = 8.0 if zeros is None else zeros.float()[..., None]
    return ((q - z) * scales.float()[..., None]).reshape(*codes.shape[:-1], -1)


def _plain_rows(c, s, rows, width, forward):
    """rows of every expert times its weights (forward) or their transpose, in fp32: zeros where a row has no expert."""
    ends, E = s["ends"], c["E"]
    out = torch.zeros(rows.shape[0], width, dtype=torch.float32, device=rows.device)
    if c["rows"] <= 64:               # the rows' experts' weights, row by row
        of = (ends[None, :] <= torch.arange(c["rows"], device=rows.device)[:, None]).sum(1)
        w = _weights(s, of)
        v = rows[:c["rows"]].float()
        out[:c["rows"]] = (torch.matmul(w, v[:, :, None])[..., 0] if forward
                           else torch.matmul(w.transpose(1, 2).contiguous(), v[:, :, None])[..., 0])
        return out
    at = 0
    for e, end in enumerate(ends.tolist()):
        if end > at:
            w = _weights(s, e)
            out[at:end] = rows[at:end].float() @ (w.t() if forward else w)
        at = end
    return out


def _plain(c, s):
    t = DTYPES[c["out"]]
    if c["kind"] == "linear":
        y = s["x"].float() @ _weights(s).t()
        return (y + s["bias"].float() if c["bias"] else y).to(t)
    if c["kind"] in ("grouped", "experts4"):
        return _plain_rows(c, s, s["x"], c["n"], True).to(t)
    if c["kind"] == "dx":
        return _plain_rows(c, s, s["dy"], c["k"], False).to(t)
    dw = torch.zeros(c["E"], c["n"], c["k"], dtype=t, device=s["x"].device)
    at = 0
    for e, end in enumerate(s["ends"].tolist()):
        if end > at:
            dw[e] = (s["dy"][at:end].float().t() @ s["x"][at:end].float()).to(t)
        at = end
    return dw


def run(state):
    c = state["case"]
    if not own:
        return _plain(c, state)
    exl3 = state["exl3"]
    if c["kind"] == "linear":
        y = torch.empty(c["rows"], c["n"], dtype=DTYPES[c["out"]], device="cuda")
        state["linear"].run(state["x"], y)
        return y
    if c["kind"] in ("grouped", "experts4"):
        return exl3.grouped_mm(state["x"], state["weight"], state["ends"], out_dtype=DTYPES[c["out"]])
    if c["kind"] == "dx":
        return exl3.grouped_mm_dx(state["dy"], state["weight"], state["ends"], out_dtype=DTYPES[c["out"]])
    return exl3.grouped_mm_dw(state["dy"], state["x"], state["ends"], out_dtype=DTYPES[c["out"]])


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6007 + 41)


def _rows(rows, k, dtype, g):
    """Rows as after a norm: N(0, 1), a few channels many times larger."""
    x = torch.randn(rows, k, device="cuda", generator=g)
    return (x * torch.exp2(torch.randn(k, device="cuda", generator=g))).to(dtype)


def _quantised(lead, n, k, c, dtype, g):
    """Codes, scales and zeros of normal weights of deviation 1 / sqrt(k), apart from a spread per row (made in pieces)."""
    count, per = lead[0] if lead else 1, c["group"]
    codes = torch.empty(count * n, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(count * n, k // per, dtype=dtype, device="cuda")
    zeros = torch.empty(count * n, k // per, dtype=torch.uint8, device="cuda") if c["zeros"] else None
    step = max(1, (1 << 26) // k)
    for i in range(0, count * n, step):
        m = min(step, count * n - i)
        v = torch.randn(m, k // per, per, device="cuda", generator=g)
        v *= torch.exp2(0.5 * torch.randn(m, 1, 1, device="cuda", generator=g)) / math.sqrt(k)
        if c["zeros"]:
            lo, hi = v.amin(-1), v.amax(-1)
            sc = ((hi - lo) / 15.0).to(dtype)
            z = torch.round(-lo / sc.float()).clamp(0, 15)
            zeros[i:i + m] = z.to(torch.uint8)
        else:
            sc = (v.abs().amax(-1) / 7.5).to(dtype)
            z = torch.full_like(v[..., 0], 8.0)
        scales[i:i + m] = sc
        q = (torch.round(v / sc.float()[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8).reshape(m, -1, 2)
        codes[i:i + m] = q[..., 0] | q[..., 1] << 4
    return [None if t is None else t.reshape(*lead, n, -1) for t in (codes, scales, zeros)]


def prepare(case, seed):
    c, g = case, _gen(seed)
    dtype, s = DTYPES[c["dtype"]], {"case": case}
    if own:
        s["exl3"] = importlib.import_module("b70-inference_amd")
    if c["kind"] == "linear":
        s["x"] = _rows(c["rows"], c["k"], dtype, g)
        s["codes"], s["scales"], s["zeros"] = _quantised((), c["n"], c["k"], c, dtype, g)
        s["bias"] = torch.randn(c["n"], device="cuda", generator=g).to(dtype) if c["bias"] else None
        if own:
            s["linear"] = s["exl3"].G4Linear(s["exl3"].G4Tensor(s["codes"], s["scales"], s["zeros"]), s["bias"])
        return s
    # rows of each expert, as a router that leans towards some experts sends them
    lean = torch.exp(0.7 * torch.randn(c["E"], device="cuda", generator=g))
    of = torch.multinomial(lean, c["rows"], replacement=True, generator=g)
    s["ends"] = torch.cumsum(torch.bincount(of, minlength=c["E"]), 0).to(torch.int32)
    all_rows = c["rows"] + c["pad"]
    if c["kind"] != "dx":
        s["x"] = _rows(all_rows, c["k"], dtype, g)
    if c["kind"] in ("dx", "dw"):     # gradients: small, a few rows much larger
        dy = torch.randn(all_rows, c["n"], device="cuda", generator=g)
        s["dy"] = (dy * torch.exp2(torch.randn(all_rows, 1, device="cuda", generator=g) - 6.0)).to(dtype)
    if c["kind"] == "experts4":
        s["codes"], s["scales"], s["zeros"] = _quantised((c["E"],), c["n"], c["k"], c, dtype, g)
        if own:
            s["weight"] = s["exl3"].G4Tensor(s["codes"], s["scales"], s["zeros"])
    elif c["kind"] != "dw":
        s["w"] = torch.empty(c["E"], c["n"], c["k"], dtype=dtype, device="cuda")
        for e in range(0, c["E"], 16):
            s["w"][e:e + 16] = torch.randn(min(16, c["E"] - e), c["n"], c["k"], device="cuda", generator=g) / math.sqrt(c["k"])
        s["weight"] = s["w"]
    return s


# ------------------------------------------------------------------------------------------------ in 64 bits
def _w64(s, e):
    """The weights of expert e (None: the only matrix), in 64 bits."""
    if "codes" not in s:
        return s["w"][e].double()
    b, sc = (s[name] if e is None else s[name][e] for name in ("codes", "scales"))
    n, groups = sc.shape
    q = torch.empty(n, 2 * b.shape[1], dtype=torch.int64, device=b.device)
    q[:, 0::2] = torch.remainder(b, 16)
    q[:, 1::2] = torch.div(b, 16, rounding_mode="floor")
    z = torch.full((n, groups), 8, device=b.device) if s["zeros"] is None else (s["zeros"] if e is None else s["zeros"][e]).long()
    per = q.shape[1] // groups
    return (q - z.repeat_interleave(per, 1)).double() * sc.double().repeat_interleave(per, 1)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = case
    if c["kind"] == "linear":
        y = torch.empty(c["rows"], c["n"], dtype=torch.float64, device="cuda")
        for j in range(0, c["n"], 4096):
            part = {"codes": s["codes"][j:j + 4096], "scales": s["scales"][j:j + 4096],
                    "zeros": None if s["zeros"] is None else s["zeros"][j:j + 4096]}
            y[:, j:j + 4096] = torch.mm(s["x"].double(), _w64(part, None).t())
        return y + s["bias"].double() if c["bias"] else y
    ends = s["ends"].cpu()
    sizes = torch.diff(ends, prepend=torch.zeros(1, dtype=ends.dtype))
    kind = c["kind"]
    if kind == "dw":
        out = torch.zeros(c["E"], c["n"], c["k"], dtype=torch.float64, device="cuda")
    else:
        out = torch.zeros(c["rows"] + c["pad"], c["k"] if kind == "dx" else c["n"], dtype=torch.float64, device="cuda")
    for e in torch.nonzero(sizes)[:, 0].tolist():
        rows = slice(int(ends[e] - sizes[e]), int(ends[e]))
        if kind in ("grouped", "experts4"):
            out[rows] = torch.mm(s["x"][rows].double(), _w64(s, e).t())
            continue
        # the gradients, as derivatives of the product itself
        dy = s["dy"][rows].double()
        if kind == "dx":
            x = torch.zeros(dy.shape[0], c["k"], dtype=torch.float64, device="cuda", requires_grad=True)
            out[rows] = torch.autograd.grad(torch.mm(x, _w64(s, e).t()), x, dy)[0]
        else:
            w = torch.zeros(c["n"], c["k"], dtype=torch.float64, device="cuda", requires_grad=True)
            out[e] = torch.autograd.grad(torch.mm(s["x"][rows].double(), w.t()), w, dy)[0]
    return out
