"""Cases that measure the engine's operators around a microscaled linear layer.

Four kinds of pass, each the call a user's program makes:

  norm      v = alpha * x + beta * gate * norm(y) * w_post, x_out = v, and
            h = norm(v) * w_pre in the input's type or as MXFP8 codes and scales
  norm_grad the gradient of that pass
  cast      a matrix to 4 or 8 bits with one scale per block, along the rows and
            (training) along the columns too, and read back
  few       y = alpha * x . W^T of a few tokens with W in 4 or 8 bits
  step      one training step of a linear layer with operands in 4 or 8 bits:
            y = x . W^T, dx = dy . W, dw = dy^T . x, operands cast on the way

norm(v) = v / sqrt(mean(v^2) + eps) over the last dimension.
"""
import math
import os
import sys

import torch

own = False

_ENGINE = []
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# format: (scale block, largest element, exponent of the largest power of two)
FORMATS = {"nvfp4": (16, 6.0, 2), "mxf4": (32, 6.0, 2), "mxf8": (32, 448.0, 8)}
EPS = 1e-6


def _b2g():
    path = os.path.join(os.getcwd(), "microbench-blackwell_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b2g

    return b2g


def _engine():
    if not _ENGINE:
        _ENGINE.append(_b2g().Engine(0))
    return _ENGINE[0]


def _code(fmt):
    b2g = _b2g()
    return {"nvfp4": b2g.FMT_NVFP4, "mxf4": b2g.FMT_MXF4, "mxf8": b2g.FMT_MXF8}[fmt]


def _up(n, m):
    return (n + m - 1) // m * m


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token between two blocks of a decode step, its h cast for the next product
        {"name": "norm, one token", "kind": "norm", "T": 1, "D": 8192, "type": "bf16",
         "out": "mxf8", "rows_per_gate": 1, "pad": 0},
        # packed ragged batch: a gate for each sequence, rows cut out of a wider buffer
        {"name": "norm, a gate per sequence", "kind": "norm", "T": 4095, "D": 5000, "type": "f16",
         "out": "f16", "rows_per_gate": 1365, "pad": 24},
        # prefill or training forward at the widest rows, one gate vector
        {"name": "norm, prefill", "kind": "norm", "T": 16384, "D": 8192, "type": "bf16",
         "out": "mxf8", "rows_per_gate": 16384, "pad": 0},
        # a small model's backward in 32 bits, a gate for each token
        {"name": "norm gradient, small", "kind": "norm_grad", "T": 301, "D": 1000, "type": "f32",
         "rows_per_gate": 1, "pad": 0},
        # the backward of the widest training forward
        {"name": "norm gradient, training", "kind": "norm_grad", "T": 16384, "D": 8192,
         "type": "bf16", "rows_per_gate": 16384, "pad": 0},
        # an activation whose sizes fit no block, both ways
        {"name": "cast both ways, ragged", "kind": "cast", "T": 4099, "K": 5000, "type": "f16",
         "fmt": "mxf4", "both": True, "stochastic": False},
        # a gradient, both ways, rounded by given random numbers
        {"name": "cast both ways, gradient", "kind": "cast", "T": 8192, "K": 8192, "type": "bf16",
         "fmt": "nvfp4", "both": True, "stochastic": True},
        # decode: one token against a square projection
        {"name": "few, one token", "kind": "few", "T": 1, "N": 8192, "K": 8192, "type": "bf16",
         "fmt": "nvfp4"},
        # drafted tokens against an odd, small output layer
        {"name": "few, odd sizes", "kind": "few", "T": 5, "N": 1001, "K": 2050, "type": "f16",
         "fmt": "mxf8"},
        # batched decode against a wide projection
        {"name": "few, a batch", "kind": "few", "T": 16, "N": 16384, "K": 8192, "type": "bf16",
         "fmt": "mxf4"},
        # a small layer's training step
        {"name": "step, small", "kind": "step", "T": 500, "N": 1024, "K": 2048, "type": "bf16",
         "fmt": "mxf8"},
        # a training step of the square projection
        {"name": "step, large", "kind": "step", "T": 8192, "N": 8192, "K": 8192, "type": "bf16",
         "fmt": "nvfp4"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm_grad", "cast", "few", "step"))
    c = {"kind": kind, "type": rng.choice(("bf16", "bf16", "f16"))}
    if kind in ("norm", "norm_grad"):
        D = _log(rng, 200, 12000)
        T = _log(rng, 1, min(16384, (16384 * 8192) // D))
        if kind == "norm_grad" and rng.random() < 0.2:
            c["type"], T = "f32", max(1, T // 4)
        if kind == "norm":
            c["out"] = rng.choice((c["type"], "mxf8"))
        c.update(T=T, D=D, rows_per_gate=rng.choice((1, max(1, -(-T // 3)), T)),
                 pad=rng.choice((0, 8, 24, 1)))
        # a gate per token in 32 bits costs more than any listed case at the largest sizes
        if kind == "norm_grad" and c["rows_per_gate"] == 1:
            c["T"] = max(1, c["T"] // 2)
    elif kind == "cast":
        both = rng.random() < 0.7
        c.update(T=_log(rng, 1, 8192), K=_log(rng, 64, 8192), fmt=rng.choice(("nvfp4", "mxf4", "mxf8")),
                 both=both, stochastic=rng.random() < 0.4)
    elif kind == "few":
        c.update(T=_log(rng, 1, 64), N=_log(rng, 256, 16384), K=_log(rng, 256, 16384),
                 fmt=rng.choice(("nvfp4", "mxf4", "mxf8")))
        if c["N"] * c["K"] > 16384 * 8192:
            c["K"] = 16384 * 8192 // c["N"]
    else:
        c["type"] = "bf16"
        c.update(T=_log(rng, 100, 8192), N=_log(rng, 256, 8192), K=_log(rng, 256, 8192),
                 fmt=rng.choice(("nvfp4", "mxf4", "mxf8")))
    return c


def _size(t):
    return {"bf16": 2, "f16": 2, "f32": 4}[t]


def _bits(fmt):
    """Bits an element costs with its share of the scale."""
    return (4 if fmt != "mxf8" else 8) + 8 / FORMATS[fmt][0]


def work(case):
    c = case
    if c["kind"] == "norm":
        n, s = c["T"] * c["D"], _size(c["type"])
        gates = -(-c["T"] // c["rows_per_gate"]) * c["D"]
        h = n * _bits("mxf8") / 8 if c["out"] == "mxf8" else n * s
        return {"bytes": 3 * n * s + h + (gates + 2 * c["D"]) * s + 8 * c["T"], "flops": 12 * n}
    if c["kind"] == "norm_grad":
        n, s = c["T"] * c["D"], _size(c["type"])
        gates = -(-c["T"] // c["rows_per_gate"]) * c["D"]
        return {"bytes": 6 * n * s + gates * (s + 4) + c["D"] * (2 * s + 8) + 8 * c["T"],
                "flops": 30 * n}
    if c["kind"] == "cast":
        n, s, ways = c["T"] * c["K"], _size(c["type"]), 2 if c["both"] else 1
        # codes written and read back, the values they stand for written in bf16
        return {"bytes": n * (s + (1 if c["stochastic"] else 0) + ways * (2 * _bits(c["fmt"]) / 8 + 2)),
                "flops": 4 * ways * n}
    if c["kind"] == "few":
        s = _size(c["type"])
        return {"bytes": c["N"] * c["K"] * _bits(c["fmt"]) / 8 + c["T"] * (c["N"] + c["K"]) * s,
                "flops": 2 * c["T"] * c["N"] * c["K"]}
    T, N, K = c["T"], c["N"], c["K"]
    # x, w, dy (and its random numbers) read; y, dx, dw written
    return {"bytes": 2 * (T * K + N * K + T * N) * 2 + T * N, "flops": 6 * T * N * K}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _normal(g, rows, cols, dtype, scale=1.0, pad=0):
    """rows x cols of a wider buffer (pad columns more), with a few large channels."""
    t = torch.randn(rows, cols + pad, generator=g, device="cuda", dtype=torch.float32)
    big = 1.0 + 7.0 * (torch.rand(cols + pad, generator=g, device="cuda") > 0.99)
    return t.mul_(big * scale).to(dtype)[:, :cols]


def _codes(v, fmt):
    """fp32 values (rows x K, K a multiple of 32) -> stored codes and scale bytes."""
    val, sf = _block_cast(v, fmt, None)
    rows = v.shape[0]
    block = FORMATS[fmt][0]
    el = val.view(rows, -1, block)
    if fmt == "nvfp4":
        sfb = sf.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        sfb = (torch.frexp(sf)[1] - 1 + 127).clamp_(0, 254).to(torch.uint8)
    if fmt == "mxf8":
        return el.reshape(rows, -1).to(torch.float8_e4m3fn).view(torch.uint8), sfb
    a = el.reshape(rows, -1).abs()
    code = torch.zeros(a.shape, dtype=torch.uint8, device=a.device)
    for lo in E2M1[1:]:
        code += a >= lo
    code += 8 * (el.reshape(rows, -1) < 0).to(torch.uint8)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), sfb


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = TYPES[c["type"]]
    s = {"case": c}
    dev = {"device": "cuda"}
    if c["kind"] in ("norm", "norm_grad"):
        T, D, per = c["T"], c["D"], c["rows_per_gate"]
        s["x"] = _normal(g, T, D, dt, 1.0, c["pad"])
        s["y"] = _normal(g, T, D, dt, 0.7, c["pad"])
        s["gate"] = (0.5 * torch.randn(-(-T // per), D, generator=g, **dev)).to(dt)
        s["w_post"] = (1 + 0.2 * torch.randn(D, generator=g, **dev)).to(dt)
        s["w_pre"] = (1 + 0.2 * torch.randn(D, generator=g, **dev)).to(dt)
        s["alpha"], s["beta"] = 1.0, 0.5
        f32 = {"device": "cuda", "dtype": torch.float32}
        if c["kind"] == "norm":
            s["x_out"] = torch.empty(T, D, device="cuda", dtype=dt)
            s["rstd_post"], s["rstd_pre"] = torch.empty(T, **f32), torch.empty(T, **f32)
            if c["out"] == "mxf8":
                Kp = _up(D, 32)
                s["codes"] = torch.empty(T, Kp, dtype=torch.uint8, **dev)
                s["sf"] = torch.empty(T, Kp // 32, dtype=torch.uint8, **dev)
            else:
                s["h"] = torch.empty(T, D, device="cuda", dtype=dt)
        else:
            # what the forward pass saved: x holds its x_out
            s["rstd_post"] = torch.rsqrt(s["y"].float().square().mean(1) + EPS)
            s["rstd_pre"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
            s["dx_out"] = _normal(g, T, D, dt, 0.01, c["pad"])
            s["dh"] = _normal(g, T, D, dt, 0.01, c["pad"])
            s["dx"], s["dy"] = (torch.empty(T, D, device="cuda", dtype=dt) for _ in range(2))
            s["dgate"] = torch.empty(s["gate"].shape, **f32)
            s["dw_post"], s["dw_pre"] = torch.empty(D, **f32), torch.empty(D, **f32)
    elif c["kind"] == "cast":
        T, K = c["T"], c["K"]
        s["x"] = _normal(g, T, K, dt, 0.02 if c["stochastic"] else 1.0)
        # a gradient is small: it is scaled into the format's range by a power of two
        s["scale"] = 256.0 if c["stochastic"] else 1.0
        s["rand"] = None
        if c["stochastic"]:
            s["rand"] = torch.randint(0, 256, (T, K), generator=g, dtype=torch.uint8, **dev)
        s.update(_cast_buffers(T, K, c["fmt"], c["both"]))
        s["back"] = torch.empty(T, K, dtype=torch.bfloat16, **dev)
        if c["both"]:
            s["back_t"] = torch.empty(K, T, dtype=torch.bfloat16, **dev)
    elif c["kind"] == "few":
        T, N, K = c["T"], c["N"], c["K"]
        Kp = _up(K, 32)
        w = torch.zeros(N, Kp, device="cuda")
        w[:, :K] = torch.randn(N, K, generator=g, **dev) * (K ** -0.5)
        if c["fmt"] == "nvfp4":
            w *= 64.0
        s["w"], s["sfw"] = _codes(w, c["fmt"])
        s["x"] = _normal(g, T, K, dt)
        s["alpha"] = 1.0 / 64.0 if c["fmt"] == "nvfp4" else 1.0
        s["out"] = torch.empty(T, N, device="cuda", dtype=dt)
    else:
        T, N, K = c["T"], c["N"], c["K"]
        s["x"] = _normal(g, T, K, dt)
        s["w"] = (torch.randn(N, K, generator=g, **dev) * (K ** -0.5)).to(dt)
        s["dy"] = _normal(g, T, N, dt, 0.01)
        s["rand"] = torch.randint(0, 256, (T, N), generator=g, dtype=torch.uint8, **dev)
        s["scale_w"], s["scale_dy"] = 64.0, 256.0
        s["qx"] = _cast_buffers(T, K, c["fmt"], True)
        s["qw"] = _cast_buffers(N, K, c["fmt"], True)
        s["qdy"] = _cast_buffers(T, N, c["fmt"], True)
        s["y"] = torch.empty(T, N, device="cuda", dtype=dt)
        s["dx"] = torch.empty(T, K, device="cuda", dtype=dt)
        s["dw"] = torch.empty(N, K, device="cuda", dtype=dt)
    return s


def _cast_buffers(rows, cols, fmt, both):
    u8 = {"dtype": torch.uint8, "device": "cuda"}
    block = FORMATS[fmt][0]

    def pair(r, k):
        kp = _up(k, 32)
        return (torch.empty(r, kp if fmt == "mxf8" else kp // 2, **u8),
                torch.empty(r, kp // block, **u8))

    b = dict(zip(("codes", "sf"), pair(rows, cols)))
    b["codes_t"], b["sf_t"] = pair(cols, rows) if both else (None, None)
    return b


# ------------------------------------------------------------------ the passes
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    c, eng = s["case"], _engine()
    if c["kind"] == "norm":
        eng.residual_norm(s["x"], y=s["y"], gate=s["gate"], rows_per_gate=c["rows_per_gate"],
                          w_post=s["w_post"], w_pre=s["w_pre"], x_out=s["x_out"], h=s.get("h"),
                          codes=s.get("codes"), sf=s.get("sf"),
                          h_format=_code("mxf8") if c["out"] == "mxf8" else 0,
                          rstd_post=s["rstd_post"], rstd_pre=s["rstd_pre"],
                          alpha=s["alpha"], beta=s["beta"], eps=EPS)
        out = {"x_out": s["x_out"], "rstd_post": s["rstd_post"], "rstd_pre": s["rstd_pre"]}
        if c["out"] == "mxf8":
            out["codes"] = s["codes"].view(torch.float8_e4m3fn)
            out["sf"] = s["sf"].view(torch.float8_e8m0fnu)
        else:
            out["h"] = s["h"]
        return out
    if c["kind"] == "norm_grad":
        eng.residual_norm_backward(
            s["dh"], s["x"], s["rstd_pre"], s["w_pre"], s["dx"], dx_out=s["dx_out"], y=s["y"],
            rstd_post=s["rstd_post"], w_post=s["w_post"], gate=s["gate"],
            rows_per_gate=c["rows_per_gate"], dy=s["dy"], dgate=s["dgate"],
            dw_post=s["dw_post"], dw_pre=s["dw_pre"], alpha=s["alpha"], beta=s["beta"])
        return {k: s[k] for k in ("dx", "dy", "dgate", "dw_post", "dw_pre")}
    if c["kind"] == "cast":
        f = _code(c["fmt"])
        eng.quantize_block(f, s["x"], s["codes"], s["sf"], codes_t=s["codes_t"], sf_t=s["sf_t"],
                           scale=s["scale"], rand=s["rand"])
        eng.dequantize_block(f, s["codes"], s["sf"], s["back"])
        if not c["both"]:
            return {"rows": s["back"]}
        eng.dequantize_block(f, s["codes_t"], s["sf_t"], s["back_t"])
        return {"rows": s["back"], "cols": s["back_t"]}
    if c["kind"] == "few":
        return eng.linear(s["x"], s["w"], s["sfw"], s["out"], _code(c["fmt"]), alpha=s["alpha"])
    f, T, N, K = _code(c["fmt"]), c["T"], c["N"], c["K"]
    qx, qw, qd = s["qx"], s["qw"], s["qdy"]
    eng.quantize_block(f, s["x"], qx["codes"], qx["sf"], codes_t=qx["codes_t"], sf_t=qx["sf_t"])
    eng.quantize_block(f, s["w"], qw["codes"], qw["sf"], codes_t=qw["codes_t"], sf_t=qw["sf_t"],
                       scale=s["scale_w"])
    eng.gemm(qx["codes"], qw["codes"], s["y"], f, sfa=qx["sf"], sfb=qw["sf"],
             alpha=1.0 / s["scale_w"])
    eng.quantize_block(f, s["dy"], qd["codes"], qd["sf"], codes_t=qd["codes_t"], sf_t=qd["sf_t"],
                       scale=s["scale_dy"], rand=s["rand"])
    eng.gemm(qd["codes"], qw["codes_t"], s["dx"], f, sfa=qd["sf"], sfb=qw["sf_t"],
             alpha=1.0 / (s["scale_w"] * s["scale_dy"]))
    eng.gemm(qd["codes_t"], qx["codes_t"], s["dw"], f, sfa=qd["sf_t"], sfb=qx["sf_t"],
             alpha=1.0 / s["scale_dy"])
    return {"y": s["y"], "dx": s["dx"], "dw": s["dw"]}


def _pow2(e):
    """2^e in 32 bits, e from -127 to 127."""
    return torch.where(e < -126, 2.0 ** -127, ((e.int().clamp(min=-126) + 127) << 23).view(torch.float32))


def _element(a, fmt, rand):
    """|values| over their scale -> the element format: to nearest even, or up where the
    fraction of a step and (rand + 1/2) / 256 reach the next step together."""
    top = FORMATS[fmt][1]
    low, mant = (1, 1) if fmt != "mxf8" else (-5, 3)
    # spacing of the element format at a: 2^(max(exponent, lowest) - mantissa bits)
    e = torch.frexp(a)[1].clamp_(min=low) - 1 - mant
    n = a * _pow2(-e)
    n = torch.round(n) if rand is None else torch.floor(n + (rand.float() + 0.5) / 256)
    return (n * _pow2(e)).clamp_(max=top)


def _block_cast(v, fmt, rand):
    """(elements, scales) of v (rows x K, K whole blocks): one scale for each block."""
    block, _, emax = FORMATS[fmt]
    v = v.view(v.shape[0], -1, block)
    amax = v.abs().amax(2)
    if fmt == "nvfp4":
        sf = (amax / 6.0).clamp_(max=448.0).to(torch.float8_e4m3fn).float()
    else:
        sf = _pow2(torch.where(amax > 0, torch.frexp(amax)[1] - 1 - emax, -127).clamp_(-127, 127))
    d = torch.where(sf > 0, sf, torch.ones_like(sf)).unsqueeze(2)
    a = torch.where(sf.unsqueeze(2) > 0, v / d, torch.zeros_like(v))
    r = rand.view(v.shape) if rand is not None else None
    el = torch.copysign(_element(a.abs(), fmt, r), a)
    return el.view(v.shape[0], -1), sf


def _pad(v, cols):
    return torch.nn.functional.pad(v, (0, cols - v.shape[1])) if cols != v.shape[1] else v


def _cast_values(v, fmt, rand):
    """The values that v's codes stand for, block scales along the rows."""
    rows, K = v.shape
    Kp = _up(K, 32)
    el, sf = _block_cast(_pad(v, Kp), fmt, None if rand is None else _pad(rand, Kp))
    block = FORMATS[fmt][0]
    return (el.view(rows, -1, block) * sf.unsqueeze(2)).view(rows, Kp)[:, :K]


def _norm_forward(s):
    c = s["case"]
    x, y, w1, w2, g = (s[k].float() for k in ("x", "y", "w_post", "w_pre", "gate"))
    if g.shape[0] > 1:
        g = g.repeat_interleave(c["rows_per_gate"], 0)[:c["T"]]
    r1 = 1.0 / torch.sqrt((y * y).mean(1) + EPS)
    v = s["alpha"] * x + s["beta"] * g * (y * r1.unsqueeze(1) * w1)
    r2 = 1.0 / torch.sqrt((v * v).mean(1) + EPS)
    return v, v * r2.unsqueeze(1) * w2, r1, r2


def _norm_backward(s):
    """The gradient of the norm pass; x holds the forward's x_out."""
    c = s["case"]
    T, D, per = c["T"], c["D"], c["rows_per_gate"]
    v, y, dh, dxo, w1, w2, g = (s[k].float() for k in ("x", "y", "dh", "dx_out", "w_post", "w_pre", "gate"))
    r1, r2 = s["rstd_post"].unsqueeze(1), s["rstd_pre"].unsqueeze(1)
    G = g.shape[0]
    gt = g.repeat_interleave(per, 0)[:T] if G > 1 else g
    vh, yh = v * r2, y * r1
    wd = w2 * dh
    dv = dxo + r2 * (wd - vh * (wd * vh).mean(1, keepdim=True))
    dw_pre = (dh * vh).sum(0)
    dz = s["beta"] * gt * dv
    dw_post = (dz * yh).sum(0)
    dg = s["beta"] * (yh * w1) * dv
    if G == 1:
        dg = dg.sum(0, keepdim=True)
    elif per > 1:
        dg = torch.nn.functional.pad(dg, (0, 0, 0, G * per - T)).view(G, per, D).sum(1)
    wz = w1 * dz
    dy = r1 * (wz - yh * (wz * yh).mean(1, keepdim=True))
    return {"dx": s["alpha"] * dv, "dy": dy, "dgate": dg, "dw_post": dw_post, "dw_pre": dw_pre}


def _decoded(codes, sf, fmt):
    """The values that stored codes stand for."""
    rows = codes.shape[0]
    if fmt == "mxf8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
        v = lut[torch.stack((codes & 15, codes >> 4), 2).view(rows, -1).int()]
    if fmt == "nvfp4":
        scale = sf.view(torch.float8_e4m3fn).float()
    else:
        scale = _pow2(sf.int() - 127)
    return (v.view(rows, -1, FORMATS[fmt][0]) * scale.unsqueeze(2)).view(rows, -1)


def _run_plain(s):
    c = s["case"]
    dt = TYPES[c["type"]]
    if c["kind"] == "norm":
        v, h, r1, r2 = _norm_forward(s)
        out = {"x_out": v.to(dt), "rstd_post": r1, "rstd_pre": r2}
        if c["out"] == "mxf8":
            el, sf = _block_cast(_pad(h, _up(c["D"], 32)), "mxf8", None)
            out["codes"] = el.to(torch.float8_e4m3fn)
            out["sf"] = sf.to(torch.float8_e8m0fnu)
        else:
            out["h"] = h.to(dt)
        return out
    if c["kind"] == "norm_grad":
        out = _norm_backward(s)
        out["dx"], out["dy"] = out["dx"].to(dt), out["dy"].to(dt)
        return out
    if c["kind"] == "cast":
        v = s["x"].float() * s["scale"]
        out = {"rows": _cast_values(v, c["fmt"], s["rand"]).to(torch.bfloat16)}
        if c["both"]:
            r = s["rand"].t().contiguous() if s["rand"] is not None else None
            out["cols"] = _cast_values(v.t().contiguous(), c["fmt"], r).to(torch.bfloat16)
        return out
    if c["kind"] == "few":
        w = _decoded(s["w"], s["sfw"], c["fmt"])[:, :c["K"]]
        return (s["alpha"] * (s["x"].float() @ w.t())).to(dt)
    return {k: v.to(dt) for k, v in _step(s).items()}


def _step(s):
    fmt, r = s["case"]["fmt"], s["rand"]
    x, w, dy = s["x"].float(), s["w"].float() * s["scale_w"], s["dy"].float() * s["scale_dy"]
    out = {"y": _cast_values(x, fmt, None) @ _cast_values(w, fmt, None).t() / s["scale_w"]}
    wt = _cast_values(w.t().contiguous(), fmt, None)
    out["dx"] = _cast_values(dy, fmt, r) @ wt.t() / (s["scale_w"] * s["scale_dy"])
    dyt = _cast_values(dy.t().contiguous(), fmt, r.t().contiguous())
    xt = _cast_values(x.t().contiguous(), fmt, None)
    out["dw"] = dyt @ xt.t() / s["scale_dy"]
    return out


# ------------------------------------------------------------------ the definitions in 64 bits
def _grid(fmt):
    """Every magnitude of the element format, ascending, in 64 bits."""
    if fmt == "mxf8":
        return torch.tensor([m * 2.0 ** -9 for m in range(8)]
                            + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1],
                            dtype=torch.float64, device="cuda")
    return torch.tensor(E2M1, dtype=torch.float64, device="cuda")


def _two_to(e):
    """2^e in 64 bits, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_cast(v, fmt, rand):
    """Values of the codes of v (64 bits, rows x K): the scale of each block from its
    largest magnitude; each element between the two neighbours of the format's grid."""
    rows, K = v.shape
    block, top, emax = FORMATS[fmt]
    Kp = _up(K, 32)
    b = torch.zeros(rows, Kp, dtype=torch.float64, device=v.device)
    b[:, :K] = v
    b = b.view(-1, block)
    amax = b.abs().max(1).values
    if fmt == "nvfp4":
        g8 = _grid("mxf8")
        sf = _nearest(torch.clamp(amax / 6, max=448.0), g8)
    else:
        e = torch.where(amax > 0, torch.frexp(amax)[1].long() - 1 - emax, -127)
        sf = _two_to(torch.clamp(e, -127, 127))
    q = torch.where(sf[:, None] > 0, b.abs() / torch.clamp(sf, min=2.0 ** -300)[:, None], 0.0)
    grid = _grid(fmt)
    q = torch.clamp(q, max=top)
    if rand is None:
        m = _nearest(q, grid)
    else:
        r = torch.zeros(rows, Kp, dtype=torch.float64, device=v.device)
        r[:, :K] = rand.double()
        lo = torch.clamp(torch.searchsorted(grid, q, right=True) - 1, max=len(grid) - 2)
        step = grid[lo + 1] - grid[lo]
        m = torch.where((q - grid[lo]) / step + (r.view(-1, block) + 0.5) / 256 >= 1, grid[lo + 1], grid[lo])
    return (torch.sign(b) * m * sf[:, None]).view(rows, Kp)[:, :K], sf.view(rows, -1), \
        (torch.sign(b) * m).view(rows, Kp)


def _nearest(q, grid):
    """The grid value next to q, of two equally near the one with the even index."""
    lo = torch.clamp(torch.searchsorted(grid, q, right=True) - 1, max=len(grid) - 2)
    d = (q - grid[lo]) - (grid[lo + 1] - q)
    return torch.where((d > 0) | ((d == 0) & (lo % 2 == 1)), grid[lo + 1], grid[lo])


def exact(case, seed):
    c, s = case, prepare(case, seed)
    f64 = torch.float64
    if c["kind"] in ("norm", "norm_grad"):
        T, D, per = c["T"], c["D"], c["rows_per_gate"]
        w1, w2 = s["w_post"].double(), s["w_pre"].double()
        gate_of = torch.arange(T, device="cuda") // per
        chunk = max(1, (1 << 26) // D)
        parts, sums = [], {}
        for t0 in range(0, T, chunk):
            rows = slice(t0, min(T, t0 + chunk))
            x, y, g = s["x"][rows].double(), s["y"][rows].double(), s["gate"][gate_of[rows]].double()
            if c["kind"] == "norm":
                r1 = (y.square().mean(1) + EPS) ** -0.5
                v = s["alpha"] * x + s["beta"] * g * y * r1[:, None] * w1
                r2 = (v.square().mean(1) + EPS) ** -0.5
                h = v * r2[:, None] * w2
                one = {"x_out": v, "rstd_post": r1, "rstd_pre": r2}
                if c["out"] == "mxf8":
                    _, one["sf"], one["codes"] = _exact_cast(h, "mxf8", None)
                else:
                    one["h"] = h
            else:
                r1, r2 = s["rstd_post"][rows].double()[:, None], s["rstd_pre"][rows].double()[:, None]
                dh = s["dh"][rows].double()
                p = dh * w2
                dv = s["dx_out"][rows].double() + r2 * p - x * r2 ** 3 * (p * x).mean(1, keepdim=True)
                z = y * r1 * w1
                dz = s["beta"] * g * dv
                u = dz * w1
                dy = r1 * u - y * r1 ** 3 * (u * y).mean(1, keepdim=True)
                one = {"dx": s["alpha"] * dv, "dy": dy}
                for k, a in (("dw_post", dz * y * r1), ("dw_pre", dh * x * r2)):
                    sums[k] = sums.get(k, 0) + a.sum(0)
                sums.setdefault("dgate", torch.zeros(s["gate"].shape, dtype=f64, device="cuda"))
                sums["dgate"].index_add_(0, gate_of[rows], s["beta"] * z * dv)
            parts.append({k: a.cpu() for k, a in one.items()})
        out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
        return {**out, **sums}
    if c["kind"] == "cast":
        v = s["x"].double() * s["scale"]
        out = {"rows": _exact_cast(v, c["fmt"], s["rand"])[0]}
        if c["both"]:
            r = s["rand"].t() if s["rand"] is not None else None
            out["cols"] = _exact_cast(v.t(), c["fmt"], r)[0]
        return out
    if c["kind"] == "few":
        w = _exact_decoded(s["w"], s["sfw"], c["fmt"])[:, :c["K"]]
        return s["alpha"] * (s["x"].double() @ w.t())
    x, w = s["x"].double(), s["w"].double() * s["scale_w"]
    dy, fmt = s["dy"].double() * s["scale_dy"], c["fmt"]
    y = _exact_cast(x, fmt, None)[0] @ _exact_cast(w, fmt, None)[0].t() / s["scale_w"]
    dx = _exact_cast(dy, fmt, s["rand"])[0] @ _exact_cast(w.t(), fmt, None)[0].t()
    dw = _exact_cast(dy.t(), fmt, s["rand"].t())[0] @ _exact_cast(x.t(), fmt, None)[0].t()
    return {"y": y, "dx": dx / (s["scale_w"] * s["scale_dy"]), "dw": dw / s["scale_dy"]}


def _exact_decoded(codes, sf, fmt):
    rows, block = codes.shape[0], FORMATS[fmt][0]
    grid8 = _grid("mxf8")
    value8 = torch.cat((grid8, torch.zeros(1, dtype=torch.float64, device="cuda")))
    if fmt == "mxf8":
        c = codes.long()
        v = value8[c & 127] * (1 - 2 * (c >> 7))
    else:
        c = torch.stack((codes.long() & 15, codes.long() >> 4), 2).view(rows, -1)
        v = _grid(fmt)[c & 7] * (1 - 2 * (c >> 3))
    scale = value8[sf.long() & 127] if fmt == "nvfp4" else _two_to(sf.long() - 127)
    return (v.view(rows, -1, block) * scale[:, :, None]).view(rows, -1)
