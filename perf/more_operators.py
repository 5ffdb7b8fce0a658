"""Performance cases of the ops around products in 8-bit integers: rows in 8
bits with a scale each, the norm with the residual's addition in front of a
product, the gated activation in front of the down projection, and the product.

``run`` calls the library where ``own`` is true. Where it is false it computes
the same from elementary torch operations, for every kind of case:

* ``quant``  -- rows (weights in bf16, attention's output in f32) in 8 bits;
* ``norm``   -- residual + rows, their norm in 8 bits (and in f32 where a
  product in bf16 follows);
* ``gate``   -- silu(gate) * up in 8 bits, gate and up being the two halves of
  one product's rows;
* ``linear`` -- W and X in 8 bits, a scale for each of their rows, f32 out.

A code is the integer next to value / scale: which one it is follows the 64-bit
value, so the plain forms go to 64 bits there; the product is in 32. Codes are
returned as the values that they stand for. Widths and heads are those of the
decoders named in ``vvli_amd.config``, or any.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = float(np.float32(1e-6))
WIDTHS = [896, 2048, 3584, 4864, 8192, 18944]
# (N, K) of projections: q|k|v, o, gate|up, down
SHAPES = [(1152, 896), (896, 896), (9728, 896), (896, 4864), (2048, 2048), (16384, 2048), (2048, 8192), (4608, 3584),
          (3584, 3584), (37888, 3584), (3584, 18944), (6144, 2048)]


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed() -> list:
    return [
        # Attention's output of one token, before the o projection (hidden 2048): latency.
        dict(name="quant-1x2048-f32", kind="quant", rows=1, width=2048, bf16=False, pad=0),
        # A projection's weights, once a model (7B gate projection: 18944 channels).
        dict(name="quant-18944x3584-bf16", kind="quant", rows=18944, width=3584, bf16=True, pad=0),
        # One token's norm in front of q|k|v: latency.
        dict(name="norm-1x2048", kind="norm", rows=1, width=2048, delta=True, y=False, bf16=True, pad=0),
        # Drafts of a batch behind the last layer: 8 bits and f32, odd rows.
        dict(name="norm-75x3584-y", kind="norm", rows=75, width=3584, delta=True, y=True, bf16=True, pad=0),
        # The rows of long prompts.
        dict(name="norm-6001x3584", kind="norm", rows=6001, width=3584, delta=True, y=False, bf16=True, pad=0),
        # A small batch's gate and up rows.
        dict(name="gate-5x4864", kind="gate", rows=5, width=4864, pad=0),
        # A prompt's.
        dict(name="gate-2500x18944", kind="gate", rows=2500, width=18944, pad=0),
        # One token through gate|up (7B): the weights' bytes.
        dict(name="linear-1x37888x3584", kind="linear", M=1, N=37888, K=3584, bias=False, pad=0),
        # A token and its drafts through the down projection (1B).
        dict(name="linear-5x2048x8192", kind="linear", M=5, N=2048, K=8192, bias=False, pad=0),
        # A batch's step through q|k|v with bias.
        dict(name="linear-48x4608x3584", kind="linear", M=48, N=4608, K=3584, bias=True, pad=0),
        # A short prompt, odd rows, padded rows of X.
        dict(name="linear-333x896x4864", kind="linear", M=333, N=896, K=4864, bias=False, pad=32),
        # A long prompt through gate|up.
        dict(name="linear-4096x37888x3584", kind="linear", M=4096, N=37888, K=3584, bias=False, pad=0),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["quant", "norm", "gate", "linear", "linear", "linear"])
    pad = rng.choice([0, 0, rng.randint(1, 9)])
    if kind != "linear":
        width = rng.choice([rng.choice(WIDTHS), _log_int(rng, 1, 20000)])
        rows = _log_int(rng, 1, max(1, min(6000, 40_000_000 // width)))
        if kind == "quant":
            return dict(kind=kind, rows=rows, width=width, bf16=rng.random() < 0.4, pad=pad)
        if kind == "gate":
            return dict(kind=kind, rows=rows, width=width, pad=pad)
        return dict(kind=kind, rows=rows, width=width, delta=rng.random() < 0.8, y=rng.random() < 0.3, bf16=rng.random() < 0.7,
                    pad=pad)
    if rng.random() < 0.6:
        N, K = rng.choice(SHAPES)
    else:
        K = 16 * _log_int(rng, 1, 1184)
        N = _log_int(rng, 1, max(1, min(40000, 130_000_000 // K)))
    M = _log_int(rng, 1, max(1, min(4096, 500_000_000_000 // (N * K))))
    return dict(kind=kind, M=M, N=N, K=K, bias=rng.random() < 0.4, pad=16 * pad)


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed))


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def _rows(g, rows: int, width: int, ld: int, dtype=torch.float32, outliers: bool = True) -> torch.Tensor:
    """Activations as layers have them: rows of other sizes, a few wide channels. [rows, ld], the first `width` of a row used."""
    x = torch.randn(rows, ld, device=DEV, generator=g)
    x *= torch.empty(rows, 1, device=DEV).uniform_(0.3, 3.0, generator=g)
    if outliers:
        x[:, torch.randint(0, max(1, width), (1 + width // 500,), device=DEV, generator=g)] *= 8
    return x.to(dtype)


def _codes(x: torch.Tensor) -> tuple:
    """Rows of x in 8 bits, for the product's inputs."""
    scale = x.abs().amax(-1, keepdim=True) / 127
    return torch.round(x / scale).clamp_(-127, 127).to(torch.int8), scale[:, 0].contiguous()


def _prepare_rows(case, g) -> dict:
    T, W, kind = case["rows"], case["width"], case["kind"]
    unit = 8 if case.get("bf16") and kind == "quant" else 4
    ld = _up(W, unit) + unit * case["pad"]
    ldc = _up(W, 16) + 16 * (case["pad"] // 3)
    st = dict(ld=ld, ldc=ldc, codes=torch.zeros(T, ldc, dtype=torch.int8, device=DEV), scale=torch.zeros(T, device=DEV),
              values=torch.zeros(T, W, device=DEV))
    if kind == "quant":
        st["x"] = _rows(g, T, W, ld, torch.bfloat16 if case["bf16"] else torch.float32, outliers=not case["bf16"])
        if T >= 5:
            st["x"][3] = 0  # a row of padding
    elif kind == "norm":
        st["x"] = _rows(g, T, W, ld)
        st["delta"] = _rows(g, T, W, ld, outliers=False) if case["delta"] else None
        st["weight"] = (1 + 0.2 * torch.randn(W, device=DEV, generator=g)).to(torch.bfloat16 if case["bf16"] else torch.float32)
        st["sum"] = torch.zeros(T, ld, device=DEV) if case["delta"] else None
        st["y"] = torch.zeros(T, W, device=DEV) if case["y"] and W % 4 == 0 else torch.zeros(T, ld, device=DEV) if case["y"] else None
    else:
        st["ld"] = ld = _up(2 * W, 4) + 4 * case["pad"] if W % 4 == 0 else 2 * _up(W, 4) + 4 * case["pad"]
        st["gu"] = _rows(g, T, ld, ld, outliers=False) * 1.5
    return st


def _prepare_linear(case, g) -> dict:
    M, N, K = case["M"], case["N"], case["K"]
    ldx = K + case["pad"]
    w, ws = _codes(torch.randn(N, K, device=DEV, generator=g).mul_(0.02))
    x, xs = _codes(_rows(g, M, K, K))
    xp = torch.randint(-127, 128, (M, ldx), dtype=torch.int8, device=DEV, generator=g)
    xp[:, :K] = x
    bias = torch.randn(N, device=DEV, generator=g).bfloat16() if case["bias"] else None
    return dict(w=w, ws=ws, x=xp, xs=xs, bias=bias, out=torch.zeros(M, N, device=DEV), ldx=ldx)


def prepare(case, seed: int) -> dict:
    st = (_prepare_linear if case["kind"] == "linear" else _prepare_rows)(case, _gen(seed))
    st["case"] = case
    st["stream"] = torch.cuda.current_stream().cuda_stream
    st["kept"] = {}  # the workspace that the program keeps from call to call
    return st


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------
def _p(t) -> int | None:
    return None if t is None else t.data_ptr()


def _values(st) -> dict:
    """The values that the codes stand for."""
    torch.mul(st["codes"][:, : st["case"]["width"]], st["scale"][:, None], out=st["values"])
    return {"values": st["values"], "scale": st["scale"]}


def _own(st):
    from vvli_amd import runtime as R

    c = st["case"]
    if c["kind"] == "linear":
        if "workspace" not in st["kept"]:
            size = R.linear_i8_workspace(c["M"], c["N"], c["K"])
            st["kept"]["workspace"] = torch.zeros(max(1, size), dtype=torch.uint8, device=DEV)
        ws = st["kept"]["workspace"]
        R.linear_i8(_p(st["w"]), c["K"], _p(st["ws"]), _p(st["x"]), st["ldx"], _p(st["xs"]), _p(st["bias"]), _p(st["out"]), c["N"],
                    c["M"], c["N"], c["K"], ws.data_ptr(), ws.numel(), st["stream"])
        return {"y": st["out"]}
    T, W, ld = c["rows"], c["width"], st["ld"]
    codes = (_p(st["codes"]), st["ldc"], _p(st["scale"]), st["stream"])
    if c["kind"] == "quant":
        R.quantize_rows(_p(st["x"]), "bf16" if c["bf16"] else "f32", ld, T, W, *codes)
        return _values(st)
    if c["kind"] == "gate":
        base, up = _p(st["gu"]), _up(W, 4)
        R.silu_mul(base, ld, base + 4 * up, ld, T, W, *codes)
        return _values(st)
    R.add_norm(_p(st["x"]), ld, _p(st["delta"]), ld, T, W, _p(st["weight"]), "bf16" if c["bf16"] else "f32", EPS, _p(st["sum"]), ld,
               _p(st["y"]), 0 if st["y"] is None else st["y"].shape[1], *codes)
    return {**_values(st), **_others(st)}


def _others(st) -> dict:
    W = st["case"]["width"]
    return {k: st[k][:, :W] for k in ("sum", "y") if st[k] is not None}


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _plain_codes(st, n: torch.Tensor) -> dict:
    """Rows of 64-bit values to codes, scales and the values that they stand for."""
    W = st["case"]["width"]
    scale = (n.abs().amax(-1) / 127).float()
    scale = torch.where(torch.isfinite(scale), scale, math.nan)
    code = n.div_(scale.double()[:, None]).round_().clamp_(-127, 127)
    code = torch.where((scale > 0)[:, None], code, 0.0)
    st["codes"][:, :W] = code.to(torch.int8)
    st["codes"][:, W:_up(W, 16)] = 0
    st["scale"].copy_(scale)
    return _values(st)


def run(st):
    if own:
        return _own(st)
    c = st["case"]
    if c["kind"] == "linear":
        y = torch.matmul(st["x"][:, : c["K"]].float(), st["w"].float().t()) * st["xs"][:, None] * st["ws"]
        if st["bias"] is not None:
            y += st["bias"].float()
        st["out"].copy_(y)
        return {"y": st["out"]}
    W = c["width"]
    if c["kind"] == "quant":
        return _plain_codes(st, st["x"][:, :W].double())
    if c["kind"] == "gate":
        g, u = st["gu"][:, :W].double(), st["gu"][:, _up(W, 4):_up(W, 4) + W].double()
        return _plain_codes(st, g / (1 + torch.exp(-g)) * u)
    h = st["x"][:, :W]
    if st["delta"] is not None:
        h = h + st["delta"][:, :W]
        st["sum"][:, :W] = h
    h = h.double()
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * st["weight"].double()
    if st["y"] is not None:
        st["y"][:, :W] = n.float()
    return {**_plain_codes(st, n), **_others(st)}


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case) -> dict:
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * K + M * K + 4 * M * N + 4 * (M + N) + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    n, T, W = case["rows"] * case["width"], case["rows"], case["width"]
    if case["kind"] == "quant":
        return {"bytes": n * ((2 if case["bf16"] else 4) + 1) + 4 * T, "flops": 4 * n}
    if case["kind"] == "gate":
        return {"bytes": 9 * n + 4 * T, "flops": 10 * n}
    return {"bytes": n * (4 + (8 if case["delta"] else 0) + (4 if case["y"] else 0) + 1) + 4 * T + W * (2 if case["bf16"] else 4),
            "flops": 10 * n}


# ---------------------------------------------------------------------------
# The results in 64 bits
# ---------------------------------------------------------------------------
def _exact_codes(n: torch.Tensor) -> dict:
    """By the distance to the integers on both sides; a scale is f32 by definition, what a code stands for is not."""
    scale = torch.max(n.max(-1).values, -n.min(-1).values).div(127).float().double()
    at = n / torch.where(scale > 0, scale, 1.0)[:, None]
    below = at.floor()
    part = at - below
    code = below + ((part > 0.5) | ((part == 0.5) & (below % 2 == 1))).double()
    code = code.clamp(-127, 127) * (scale > 0)[:, None]
    return {"values": code * scale[:, None], "scale": scale}


def exact(case, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "linear":
        y = torch.empty(case["M"], case["N"], dtype=torch.float64, device=DEV)
        w, x = st["w"].double(), st["x"][:, : case["K"]].double()
        for m in range(0, case["M"], 512):  # row by row of W's scale: every product of codes is a whole number
            y[m:m + 512] = torch.matmul(w, x[m:m + 512].t().contiguous()).t()
        y *= st["xs"].double()[:, None] * st["ws"].double()[None]
        return {"y": y if st["bias"] is None else y + st["bias"].double()}
    W = case["width"]
    if case["kind"] == "quant":
        return _exact_codes(st["x"][:, :W].double())
    if case["kind"] == "gate":
        up = _up(W, 4)
        return _exact_codes(st["gu"][:, :W].double() * torch.sigmoid(st["gu"][:, :W].double()) * st["gu"][:, up:up + W].double())
    h = st["x"][:, :W]
    out = {}
    if st["delta"] is not None:
        out["sum"] = (h.double() + st["delta"][:, :W].double()).float().double()  # the residual's rows are f32 by definition
        h = out["sum"]
    h = h.double()
    n = h / (torch.linalg.vector_norm(h, dim=-1, keepdim=True).square() / W + EPS).sqrt() * st["weight"].double()
    out.update(_exact_codes(n))
    if st["y"] is not None:
        out["y"] = n
    return out
