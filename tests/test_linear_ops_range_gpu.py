"""Operators around a linear layer at the ends of their range: blocks of zeros, tiny and huge
blocks under a scale, bytes next to the point where a code goes up, rows of any magnitude."""
import numpy as np
import pytest
import torch

import linear_ops_ref as ref
from test_linear_ops_gpu import FMT, TINY, TYPE, ULP, check_cast, code_buffers, dev, grad_bounds, host, rounded
from test_linear_ops_gpu import test_norm_gradient as check_gradient

pytestmark = pytest.mark.gpu


def cast_and_check(engine, fmt, typ, x, scale, rand=None):
    """Both ways against the definition, and the read-back finite; x * scale is exact."""
    rows, cols = x.shape
    (c, s), (ct, st) = code_buffers(fmt, rows, cols), code_buffers(fmt, cols, rows)
    r = None if rand is None else dev(rand, torch.uint8, fill=0)
    engine.quantize_block(FMT[fmt], dev(x, TYPE[typ]), c, s, codes_t=ct, sf_t=st, scale=scale, rand=r)
    check_cast(c, s, x * scale, fmt, rand)
    check_cast(ct, st, x.T * scale, fmt, None if rand is None else rand.T)
    c1, s1 = code_buffers(fmt, rows, cols)
    engine.quantize_block(FMT[fmt], dev(x, TYPE[typ]), c1, s1, scale=scale, rand=r)
    assert torch.equal(c, c1) and torch.equal(s, s1)
    out = torch.empty(rows, cols, dtype=torch.float32, device="cuda")
    engine.dequantize_block(FMT[fmt], c, s, out)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("stochastic", [False, True])
@pytest.mark.parametrize("scale", [2.0, 64.0, 4096.0])
@pytest.mark.parametrize("typ", list(TYPE))
@pytest.mark.parametrize("fmt", list(FMT))
def test_cast_of_zero_and_tiny_blocks_with_a_scale(engine, fmt, typ, scale, stochastic):
    rng = np.random.default_rng(70)
    x = rng.normal(size=(70, 130))
    x[3], x[4] = 0.0, -0.0          # masked tokens
    x[:, 7] = 0.0                   # a feature no token uses
    x[10:42, 32:64] = 0.0           # a zero block both ways
    x[43:, :32] *= 2.0 ** -124      # bf16, fp32: next to the least of the type; fp16: zeros
    x[50, 64:96] = 2.0 ** -126 * (np.arange(32) % 5 - 2)
    x[51, 64:] = 2.0 ** -24 * (np.arange(66) % 3 - 1)
    rand = rng.integers(0, 256, x.shape) if stochastic else None
    cast_and_check(engine, fmt, typ, rounded(x, typ), scale, rand)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", list(FMT))
def test_cast_with_a_scale_near_the_largest(engine, fmt, typ):
    x = np.random.default_rng(73).normal(size=(40, 96)) * 2.0 ** -115
    x[5], x[:, 9], x[7, 32:64] = 0.0, 0.0, 2.0 ** -126
    cast_and_check(engine, fmt, typ, rounded(x, typ), 2.0 ** 120)


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -30, 2.0 ** 12])
@pytest.mark.parametrize("typ", list(TYPE))
@pytest.mark.parametrize("fmt", ["mxf4", "mxf8"])
def test_stochastic_cast_of_large_blocks(engine, fmt, typ, scale):
    rng = np.random.default_rng(71)
    # a row's magnitude, up to what the type and the product with scale hold
    top = 15 if typ == "f16" else 110
    x = np.clip(rng.normal(size=(48, 96)), -3, 3) * 2.0 ** np.linspace(-10, top - 3, 48)[:, None]
    cast_and_check(engine, fmt, typ, rounded(x, typ), scale, rng.integers(0, 256, x.shape))


def around_the_step(fmt, s, q):
    """The byte from which |x| = q * s goes up, and the one before (clipped to a byte)."""
    grid = ref.GRID[fmt]
    lo = np.clip(np.searchsorted(grid, q, side="right") - 1, 0, len(grid) - 2)
    f = (q - grid[lo]) / (grid[lo + 1] - grid[lo])
    r = np.ceil(256 * (1 - f) - 0.5)
    return np.clip(np.stack([r - 1, r]), 0, 255).astype(np.int64)


def blocks_of(first, elements, fmt):
    """Rows of one block: `first`, which fixes the scale, then the elements."""
    n = ref.BLOCK[fmt] - 1
    e = np.resize(elements, -(-len(elements) // n) * n).reshape(-1, n)
    return np.concatenate([np.broadcast_to(first, (len(e), 1)), e], 1)


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -8, 256.0])
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_stochastic_nvfp4_of_every_value_at_its_step(engine, typ, scale):
    # every 16-bit magnitude whose code is neither 0 for all bytes nor saturated, over every
    # ue4m3 scale, with the two bytes between which its code changes
    bits = np.arange(1, 1 << 15, dtype=np.int32)
    v = torch.from_numpy(bits.astype(np.int16)).view(TYPE[typ]).double().numpy()
    v = v[np.isfinite(v)]
    xs, rs = [], []
    for s in ref.E4M3[1:]:
        first = 6 * s / scale
        if rounded(np.array([first]), typ)[0] != first:
            continue  # beyond fp16
        el = v[(v >= 2.0 ** -10 * s / scale) & (v <= first)]
        el = np.concatenate([el, -el[::3]])
        x = blocks_of(first, el, "nvfp4")
        for r in around_the_step("nvfp4", s, np.abs(x) * scale / s):
            xs.append(x), rs.append(r)
    x, r = np.concatenate(xs), np.concatenate(rs)
    x, r = np.pad(x, ((0, 0), (0, 16))), np.pad(r, ((0, 0), (0, 16)))  # whole 32 columns
    c, sf = code_buffers("nvfp4", *x.shape)
    engine.quantize_block(FMT["nvfp4"], dev(x, TYPE[typ]), c, sf, scale=scale, rand=dev(r, torch.uint8, fill=0))
    check_cast(c, sf, x * scale, "nvfp4", r)


@pytest.mark.parametrize("fmt", list(FMT))
def test_stochastic_cast_of_fp32_next_to_each_step(engine, fmt):
    # x = s (n + 1 - (r + 1/2) / 256) steps goes up, its fp32 neighbour below does not
    grid = ref.GRID[fmt]
    xs, rs = [], []
    for s in (ref.E4M3[[1, 9, 60, 77, 101, 126]] if fmt == "nvfp4" else 2.0 ** np.array([-100, -3, 0, 20, 90])):
        lo, r = np.meshgrid(np.arange(len(grid) - 1), np.arange(0, 256, 5 if fmt == "mxf8" else 1))
        lo, r = lo.ravel(), r.ravel()
        at = (s * (grid[lo] + (grid[lo + 1] - grid[lo]) * (1 - (r + 0.5) / 256))).astype(np.float32)
        for x in (at, np.nextafter(at, np.float32(0))):
            e = blocks_of(s * grid[-1], x.astype(np.float64), fmt)
            xs.append(e)
            rs.append(np.concatenate([np.zeros((len(e), 1)), np.resize(r, (len(e), e.shape[1] - 1))], 1))
    x, r = np.concatenate(xs), np.concatenate(rs).astype(np.int64)
    if fmt == "nvfp4":
        x, r = np.pad(x, ((0, 0), (0, 16))), np.pad(r, ((0, 0), (0, 16)))
    c, sf = code_buffers(fmt, *x.shape)
    engine.quantize_block(FMT[fmt], dev(x, torch.float32), c, sf, rand=dev(r, torch.uint8, fill=0))
    check_cast(c, sf, x, fmt, r)


# ------------------------------------------------------------------ the gradient
@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("size_v,size_y", [(1e13, 1e13), (1e15, 1e-3), (1e-3, 1e15), (1e16, 1e16), (1e-14, 1e-14),
                                           (1e-18, 1e17)])
@pytest.mark.parametrize("rows,cols", [(12, 200), (12, 1001), (3, 9000)])
def test_norm_gradient_of_rows_of_any_magnitude(engine, typ, size_v, size_y, rows, cols):
    # the rows' projections are of the same size as the rest of dx and dy; epsilon 0
    rng = np.random.default_rng(72)
    a = {"y": size_y * (1 + rng.random((rows, cols))), "w_post": 1 + 0.2 * rng.normal(size=cols),
         "w_pre": 1 + 0.2 * rng.normal(size=cols), "gate": 1 + 0.2 * rng.normal(size=(rows, cols))}
    a = {k: rounded(m, typ) for k, m in a.items()}
    v = rounded(size_v * (1 + rng.random((rows, cols))), typ)
    r1, r2 = (rounded((m * m).mean(1) ** -0.5, "f32") for m in (a["y"], v))
    dh = rounded(1 + 0.1 * rng.normal(size=(rows, cols)), typ)
    dxo = rounded((1 + 0.1 * rng.normal(size=(rows, cols))) / size_v, typ)
    want = ref.norm_backward(dh, dxo, v, r2, a["w_pre"], a["y"], r1, a["w_post"], a["gate"], 1)
    bound = grad_bounds(a, v, dh, dxo, r1, r2, 1, 1.0, 1.0, typ, cols, rows)
    dt = TYPE[typ]
    w1, w2, g = (torch.as_tensor(a[k]).to(dt).cuda() for k in ("w_post", "w_pre", "gate"))
    f1, f2 = (torch.as_tensor(r).float().cuda() for r in (r1, r2))
    out = {k: dev(np.zeros((rows, cols)), dt) for k in ("dx", "dy")}
    out.update({k: torch.full(want[k].shape, float("nan"), device="cuda") for k in ("dgate", "dw_post", "dw_pre")})
    engine.residual_norm_backward(
        dev(dh, dt), dev(v, dt), f2, w2, out["dx"], dx_out=dev(dxo, dt), y=dev(a["y"], dt), rstd_post=f1,
        w_post=w1, gate=g, dy=out["dy"], dgate=out["dgate"], dw_post=out["dw_post"], dw_pre=out["dw_pre"])
    for k, b in bound.items():
        if k in ("dx", "dy"):
            b = b + ULP[typ] * (np.abs(want[k]) + b) + TINY[typ]
        assert np.all(np.abs(host(out[k]) - want[k]) <= b), k


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,per", [(20, 2056, 3), (20, 4096, 3), (20, 4097, 3), (24, 8192, 4), (9, 8191, 2),
                                           (9, 8184, 9), (5, 8200, 1)])
@pytest.mark.parametrize("pad", [0, 1])
def test_norm_gradient_where_its_forms_change(engine, typ, rows, cols, per, pad):
    # one pass or two, by columns, type, alignment and the rows of a gate
    check_gradient(engine, typ, rows, cols, per, pad)
