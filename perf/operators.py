"""What the row and weight operators of ``ce4b200.kernels`` around quantised products cost.

Operators (all BF16 activations, row-major):

* ``norm``:    ``add_rmsnorm_forward`` -- s = bf16(x + residual), n = bf16(rmsnorm(s) * w).
* ``norm8``:   ``add_rmsnorm_mxfp8`` -- the same, with n as E4M3 codes and E8M0 scales.
* ``pack``:    ``quantize_mxfp4`` and ``dequantize_mxfp4`` -- a weight to 4-bit E2M1 codes
               with one E8M0 scale per row and 32 columns, and back.
* ``linear``:  ``mxfp4_linear`` -- a few activation rows times a 4-bit weight (+ residual).
* ``swiglu``:  ``mxfp4_swiglu`` -- the same for a gate|up weight, with silu(gate) * up.

``own`` False computes them from elementary torch operations, True through the package.
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # E2M1 magnitudes by code


@functools.cache
def _kernels():
    package = str(Path(__file__).resolve().parents[1] / "chess-engine-4_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from ce4b200 import kernels

    return kernels


# ------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # One position between two blocks of a d512 tower: pure latency.
        {"name": "norm 1x512", "op": "norm", "rows": 1, "width": 512},
        # Rows and a width that fill no vector and no tile.
        {"name": "norm 1021x769", "op": "norm", "rows": 1021, "width": 769},
        # The largest batch of the benchmark at d1024.
        {"name": "norm 65536x1024", "op": "norm", "rows": 65536, "width": 1024},
        # A search batch entering an MXFP8 block; rows end inside a scale tile.
        {"name": "norm8 64x512", "op": "norm8", "rows": 64, "width": 512},
        # A throughput batch entering an MXFP8 block of the d2048 tower.
        {"name": "norm8 16384x2048", "op": "norm8", "rows": 16384, "width": 2048},
        # A d512 tower's down weight at load time.
        {"name": "pack 512x1536", "op": "pack", "n": 512, "k": 1536},
        # A large weight at load time.
        {"name": "pack 8192x8192", "op": "pack", "n": 8192, "k": 8192},
        # The down product of one position at d512, added to the residual stream.
        {"name": "linear 1x512<1536", "op": "linear", "rows": 1, "n": 512, "k": 1536, "residual": True},
        # The down product of a full search batch at d1024, ratio 4.
        {"name": "linear 64x1024<4096", "op": "linear", "rows": 64, "n": 1024, "k": 4096, "residual": True},
        # A few rows against a weight as large as the L2 cache, no residual.
        {"name": "linear 7x28672<8192", "op": "linear", "rows": 7, "n": 28672, "k": 8192, "residual": False},
        # The gate and up products of a full search batch at d1024, ratio 4.
        {"name": "swiglu 64x4096<1024", "op": "swiglu", "rows": 64, "n": 4096, "k": 1024},
        # A ragged search batch at d2048, ratio 4.
        {"name": "swiglu 33x8192<2048", "op": "swiglu", "rows": 33, "n": 8192, "k": 2048},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng) -> dict:
    op = rng.choice(("norm", "norm8", "pack", "linear", "swiglu"))
    while True:
        if op in ("norm", "norm8"):
            rows = _log_int(rng, 1, 65536)
            width = _log_int(rng, 1, 8192) if op == "norm" else 128 * _log_int(rng, 1, 64)
            if rows * width <= 65536 * 1024:
                return {"op": op, "rows": rows, "width": width}
        elif op == "pack":
            return {"op": op, "n": _log_int(rng, 1, 8192), "k": 128 * _log_int(rng, 1, 64)}
        else:
            case = {"op": op, "rows": _log_int(rng, 1, 64), "n": _log_int(rng, 1, 28672),
                    "k": 128 * _log_int(rng, 1, 64)}
            # No more multiplications than the largest listed product.
            if case["rows"] * case["n"] * case["k"] * (2 if op == "swiglu" else 1) <= 7 * 28672 * 8192:
                if op == "linear":
                    case["residual"] = rng.random() < 0.5
                return case


def work(case: dict) -> dict:
    op = case["op"]
    if op in ("norm", "norm8"):
        n, w = case["rows"] * case["width"], case["width"]
        # x and the residual in, the sum out, w once; n out as BF16, or codes and scales.
        return {"bytes": n * 6 + w * 2 + (n * 2 if op == "norm" else n + n / 32), "flops": 6 * n}
    if op == "pack":
        # The weight in and its values out; the 4-bit form in between is written and read.
        n = case["n"] * case["k"]
        return {"bytes": n * 4 + 2 * (n / 2 + n / 32), "flops": 3 * n}
    rows, n, k = case["rows"], case["n"], case["k"]
    wide = n * (2 if op == "swiglu" else 1)
    moved = wide * k / 2 + wide * k / 32 + 2 * rows * k + 2 * rows * n
    if case.get("residual"):
        moved += 2 * rows * n
    return {"bytes": moved, "flops": 2 * rows * wide * k}


# ------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _scale_rows(scales: torch.Tensor, n: int) -> torch.Tensor:
    """[n/128, k/128, 32, 16] scale tiles -> [n, k/32] codes."""

    rt, ct = scales.shape[:2]
    return scales.reshape(rt, ct, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, ct * 4)[:n]


def _scale_tiles(codes: torch.Tensor) -> torch.Tensor:
    """[rows, k/32] codes -> scale tiles; rows past the last one are zero."""

    rows, groups = codes.shape
    rt, ct = -(-rows // 128), groups // 4
    full = torch.zeros(rt * 128, groups, dtype=torch.uint8, device=codes.device)
    full[:rows] = codes
    return full.reshape(rt, 4, 32, ct, 4).permute(0, 3, 2, 1, 4).reshape(rt, ct, 32, 16).contiguous()


def _quantize4(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """FP32 [n, k] -> E2M1 codes [n, k] (ties to even) and scale codes [n, k/32]: the scale
    is the smallest power of two, 2^-39 at least, that leaves no magnitude over 6."""

    n, k = w.shape
    blocks = w.reshape(n, k // 32, 32)
    amax = blocks.abs().amax(2)
    mantissa, exponent = torch.frexp(amax)
    exponent = torch.where(mantissa <= 0.75, exponent - 3, exponent - 2)
    exponent = torch.where(amax > 0, exponent, -39).clamp(min=-39)
    mag = torch.ldexp(blocks.abs(), -exponent[:, :, None])
    code = (mag > 0.25).to(torch.uint8)
    for limit, at in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (mag >= limit) if at else (mag > limit)
    code += (blocks < 0).to(torch.uint8) * 8
    return code.reshape(n, k), (exponent + 127).to(torch.uint8)


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    op = case["op"]
    state = dict(case)
    if op in ("norm", "norm8"):
        rows, width = case["rows"], case["width"]
        # A residual stream of a few units with the odd large channel, and a block's output.
        state["residual"] = (3.0 * torch.randn(rows, width, generator=g, device="cuda")).bfloat16()
        state["residual"][:, seed % width] *= 16
        state["x"] = torch.randn(rows, width, generator=g, device="cuda").bfloat16()
        state["weight"] = (1.0 + 0.1 * torch.randn(width, generator=g, device="cuda")).bfloat16()
        return state
    n, k = case["n"], case["k"]
    if op == "pack":
        state["w"] = (0.02 * torch.randn(n, k, generator=g, device="cuda")).bfloat16()
        state["w"][seed % n, :32] = 0  # a pruned group
        return state
    wide = 2 * n if op == "swiglu" else n
    codes = torch.empty(wide, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(wide, k // 32, dtype=torch.uint8, device="cuda")
    for r in range(0, wide, 4096):
        part = 0.02 * torch.randn(min(4096, wide - r), k, generator=g, device="cuda")
        code, scale = _quantize4(part)
        codes[r:r + 4096] = code[:, 0::2] | (code[:, 1::2] << 4)
        scales[r:r + 4096] = scale
    state["codes"], state["scales"] = codes, _scale_tiles(scales)
    # Normalised rows, or SwiGLU's hidden ones: most near zero, a few large.
    x = torch.randn(case["rows"], k, generator=g, device="cuda")
    state["x"] = (x if op == "swiglu" else x * x.abs()).bfloat16()
    if case.get("residual"):
        state["residual"] = (3.0 * torch.randn(case["rows"], n, generator=g, device="cuda")).bfloat16()
    else:
        state["residual"] = None
    return state


# ------------------------------------------------------------------ one pass
def _plain_norm8(s: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    # In 64 bits: a value next to a border between two codes decides for one of them.
    rows, width = s.shape
    v = s.double()
    n = (v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * w.double()).bfloat16()
    blocks = n.float().reshape(rows, width // 32, 32)
    amax = (blocks.abs().amax(2) * torch.tensor(0.002232142857, device=s.device)).clamp(min=1e-12)
    mantissa, exponent = torch.frexp(amax)  # smallest 2^e >= amax
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    codes = torch.ldexp(blocks, -exponent[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.reshape(rows, width), _scale_tiles((exponent + 127).to(torch.uint8))


def _plain_weight(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    wide, k = codes.shape[0], 2 * codes.shape[1]
    nibbles = torch.stack((codes & 15, codes >> 4), 2).reshape(wide, k).int()
    table = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    scale = torch.exp2(_scale_rows(scales, wide).float() - 127.0)
    return (table[nibbles].reshape(wide, k // 32, 32) * scale[:, :, None]).reshape(wide, k)


def run(state: dict):
    op = state["op"]
    if op == "norm":
        x, residual, w = state["x"], state["residual"], state["weight"]
        if own:
            total, n = _kernels().add_rmsnorm_forward(x, residual, w, EPS)
        else:
            total = (x.float() + residual.float()).bfloat16()
            s = total.float()
            n = (s * torch.rsqrt((s * s).mean(1, keepdim=True) + EPS) * w.float()).bfloat16()
        return {"sum": total, "normalized": n}
    if op == "norm8":
        x, residual, w = state["x"], state["residual"], state["weight"]
        if own:
            total, q = _kernels().add_rmsnorm_mxfp8(x, residual, w, EPS)
            codes, scales = q.values, q.scales
        else:
            total = (x.float() + residual.float()).bfloat16()
            codes, scales = _plain_norm8(total, w)
        return {"sum": total, "values": codes, "scales": scales.view(torch.float8_e8m0fnu)}
    if op == "pack":
        if own:
            kernels = _kernels()
            return kernels.dequantize_mxfp4(kernels.quantize_mxfp4(state["w"]))
        code, scale = _quantize4(state["w"].float())
        return _plain_weight(code[:, 0::2] | (code[:, 1::2] << 4), _scale_tiles(scale)).bfloat16()
    if own:
        kernels = _kernels()
        weight = kernels.Mxfp4Tensor(values=state["codes"], scales=state["scales"])
        if op == "swiglu":
            return kernels.mxfp4_swiglu(state["x"], weight)
        return kernels.mxfp4_linear(state["x"], weight, residual=state["residual"])
    y = state["x"].float() @ _plain_weight(state["codes"], state["scales"]).T
    if op == "swiglu":
        gate, up = y[:, :state["n"]], y[:, state["n"]:]
        return (gate / (1.0 + torch.exp(-gate)) * up).bfloat16()
    return (y if state["residual"] is None else y + state["residual"].float()).bfloat16()


# ------------------------------------------------------------------ in 64 bits
def exact(case: dict, seed: int):
    state = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "norm8"):
        total = state["x"].double() + state["residual"].double()
        s = total.bfloat16().double()  # the stream that is kept, and that the norm is of
        norm = s.square().sum(1, keepdim=True).div(case["width"]).add(EPS).sqrt()
        n = s / norm * state["weight"].double()
        if op == "norm":
            return {"sum": total, "normalized": n}
        n = n.bfloat16().double().reshape(case["rows"], -1, 32)
        top = (n.abs().amax(2) * 0.002232142857).clamp(min=1e-12)
        power = torch.ceil(torch.log2(top))
        power = torch.where(torch.exp2(power - 1) >= top, power - 1, power)
        codes = (n * torch.exp2(-power)[:, :, None]).clamp(-448, 448)
        mag = codes.abs().clamp(min=2.0**-6)
        step = torch.exp2(torch.floor(torch.log2(mag)) - 3)
        codes = torch.round(codes / step) * step
        return {"sum": total, "values": codes.reshape(case["rows"], -1),
                "scales": torch.exp2(_scale_tiles((power + 127).to(torch.uint8)).double() - 127)}
    if op == "pack":
        v = state["w"].double().reshape(case["n"], -1, 32)
        top = v.abs().amax(2, keepdim=True).clamp(min=6 * 2.0**-39)
        power = torch.ceil(torch.log2(top / 6))
        power = torch.where(6 * torch.exp2(power - 1) >= top, power - 1, power)
        power = torch.where(6 * torch.exp2(power) < top, power + 1, power)
        v = v * torch.exp2(-power)
        step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
        return (torch.round(v / step) * step * torch.exp2(power)).reshape(case["n"], -1)
    # The product group by group of rows, so that a large weight fits in 64 bits.
    x = state["x"].double()
    codes, scales = state["codes"], _scale_rows(state["scales"], state["codes"].shape[0])
    parts = []
    for r in range(0, codes.shape[0], 2048):
        c = codes[r:r + 2048]
        nibble = torch.empty(c.shape[0], 2 * c.shape[1], dtype=torch.int64, device="cuda")
        nibble[:, 0::2], nibble[:, 1::2] = c & 15, c >> 4
        # E2M1 by its fields: 2^(e - 1) * (1 + m / 2), or m / 2 where e is 0.
        e, m = (nibble >> 1) & 3, (nibble & 1).double()
        value = torch.where(e > 0, torch.exp2(e.double() - 1) * (1 + m / 2), m / 2)
        value = torch.where(nibble > 7, -value, value)
        value *= torch.exp2(scales[r:r + 2048].double() - 127).repeat_interleave(32, 1)
        parts.append(x @ value.T)
    y = torch.cat(parts, 1)
    if op == "swiglu":
        gate, up = y[:, :case["n"]], y[:, case["n"]:]
        return gate * torch.sigmoid(gate) * up
    return y if state["residual"] is None else y + state["residual"].double()
