"""Operators around a linear layer against their definitions in 64 bits: microscaled casts,
read-back, the norm pass and its gradient, the product of a few tokens."""
import numpy as np
import pytest
import torch

import b2g
import linear_ops_ref as ref
from b2g._ops import block_shapes

pytestmark = pytest.mark.gpu

FMT = {"nvfp4": b2g.FMT_NVFP4, "mxf4": b2g.FMT_MXF4, "mxf8": b2g.FMT_MXF8}
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# one rounding to the type: half a unit in the last place (significands of 24, 8 and 11 bits),
# relative, and below the normal range
ULP = {k: torch.finfo(t).eps / 2 for k, t in TYPE.items()}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}


def dev(a, dtype, pad=0, fill=float("nan")):
    """`a` on the GPU as the left columns of a wider buffer (`fill` in the rest)."""
    a = torch.as_tensor(np.asarray(a))
    t = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=dtype, device="cuda")
    t[:, :a.shape[1]] = a.to(dtype)
    return t[:, :a.shape[1]]


def host(t):
    return t.double().cpu().numpy()


def u8(t):
    return t.cpu().numpy()


def code_buffers(fmt, rows, cols, fill=0xEE):
    c, s = block_shapes(FMT[fmt], rows, cols)
    return (torch.full(c, fill, dtype=torch.uint8, device="cuda"),
            torch.full(s, fill, dtype=torch.uint8, device="cuda"))


def rounded(a, typ):
    return host(torch.as_tensor(a).to(TYPE[typ]))


# ------------------------------------------------------------------ casts
def check_cast(codes, sf, x, fmt, rand=None):
    v, s = ref.decode(u8(codes), u8(sf), fmt)
    want, ws = ref.cast(x, fmt, rand)
    assert np.array_equal(s, ws, equal_nan=True)
    ok = np.repeat(np.isfinite(ws), ref.BLOCK[fmt], 1)
    assert np.array_equal(v[ok], want[ok])


SIZES = [(1, 1), (1, 17), (3, 32), (33, 65), (130, 250), (128, 64), (257, 1000), (64, 2048)]


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("typ", list(TYPE))
@pytest.mark.parametrize("rows,cols", SIZES)
def test_cast_both_ways_is_exact(engine, fmt, typ, rows, cols):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = rounded(rng.normal(size=(rows, cols)) * 10.0 ** rng.integers(-3, 3, size=(rows, 1)), typ)
    pad = (0, 8, 1)[(rows + cols) % 3]
    t = dev(x, TYPE[typ], pad)
    (c, s), (ct, st) = code_buffers(fmt, rows, cols), code_buffers(fmt, cols, rows)
    engine.quantize_block(FMT[fmt], t, c, s, codes_t=ct, sf_t=st)
    check_cast(c, s, x, fmt)
    check_cast(ct, st, x.T, fmt)
    # one way at a time: the same codes
    c1, s1 = code_buffers(fmt, rows, cols)
    engine.quantize_block(FMT[fmt], t, c1, s1)
    c2, s2 = code_buffers(fmt, cols, rows)
    engine.quantize_block(FMT[fmt], t, codes_t=c2, sf_t=s2)
    for a, b in ((c, c1), (s, s1), (ct, c2), (st, s2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("typ", list(TYPE))
@pytest.mark.parametrize("rows,cols", [(1, 5), (40, 96), (150, 333)])
def test_stochastic_cast_is_exact(engine, fmt, typ, rows, cols):
    rng = np.random.default_rng(5)
    x = rounded(rng.normal(size=(rows, cols)) * 0.02, typ)
    r = rng.integers(0, 256, size=(rows, cols))
    rand = dev(r, torch.uint8, (0, 8, 3)[rows % 3], 255)
    (c, s), (ct, st) = code_buffers(fmt, rows, cols), code_buffers(fmt, cols, rows)
    engine.quantize_block(FMT[fmt], dev(x, TYPE[typ]), c, s, codes_t=ct, sf_t=st, scale=64.0, rand=rand)
    check_cast(c, s, x * 64, fmt, r)
    check_cast(ct, st, x.T * 64, fmt, r.T)


def test_stochastic_cast_of_each_byte(engine):
    # a fraction of f steps goes up for the round(256 f) largest of the 256 bytes
    x = np.zeros((256, 32))
    x[:, 0], x[:, 1] = 6.0, 2.25  # scale 1; 2.25 lies a quarter of the way from 2 to 3
    c, s = code_buffers("mxf4", 256, 32)
    rand = torch.arange(256, dtype=torch.uint8, device="cuda").view(-1, 1).expand(-1, 32).contiguous()
    engine.quantize_block(FMT["mxf4"], dev(x, torch.bfloat16), c, s, rand=rand)
    got = ref.values(u8(c), u8(s), "mxf4")[:, 1]
    assert (got == 3).sum() == 64 and np.all(got[192:] == 3) and np.all(got[:192] == 2)


@pytest.mark.parametrize("scale", [0.25, 3.0])
def test_cast_with_a_scale(engine, scale):
    x = rounded(np.random.default_rng(6).normal(size=(48, 80)), "f32")
    # fp32 product, as the cast's first step
    y = (x.astype(np.float32) * np.float32(scale)).astype(np.float64)
    for fmt in FMT:
        (c, s), (ct, st) = code_buffers(fmt, 48, 80), code_buffers(fmt, 80, 48)
        engine.quantize_block(FMT[fmt], dev(x, torch.float32), c, s, codes_t=ct, sf_t=st, scale=scale)
        # x / s rounds to fp32 before it rounds to the element: a quotient within 2^-24 of a
        # boundary may land on it, which none of these does
        check_cast(c, s, y, fmt)
        check_cast(ct, st, y.T, fmt)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("typ", list(TYPE))
def test_cast_of_special_blocks(engine, fmt, typ):
    x = np.random.default_rng(7).normal(size=(40, 96))
    x[0, :32] = 0.0
    x[1, :32] = -0.0
    x[2, :32] *= 1e-7                      # scale at or below the smallest ue4m3
    x[3, 32:64] = np.linspace(-6, 6, 32)
    x[4, 5], x[4, 40], x[5, 70] = np.inf, -np.inf, np.nan
    x[6, :32] = 60000.0                    # beyond 6 * 448: ue4m3 scale saturates
    x[7, :32] = 2.0 ** -24 * (1 + np.arange(32) % 3)
    with np.errstate(over="ignore"):
        x = rounded(x, typ)
    t = dev(x, TYPE[typ])
    (c, s), (ct, st) = code_buffers(fmt, 40, 96), code_buffers(fmt, 96, 40)
    engine.quantize_block(FMT[fmt], t, c, s, codes_t=ct, sf_t=st)
    check_cast(c, s, x, fmt)
    check_cast(ct, st, x.T, fmt)
    out = torch.empty(40, 96, dtype=torch.float32, device="cuda")
    engine.dequantize_block(FMT[fmt], c, s, out)
    assert np.isnan(host(out)[4, 0]) and np.isnan(host(out)[5, 70]) and np.isfinite(host(out)[4, 95])


def test_cast_agrees_with_quantize(engine):
    x = torch.empty(64, 256, dtype=torch.float32, device="cuda")
    engine.fill(x, 21, 1)
    for fmt in FMT:
        (c, s), (c0, s0) = code_buffers(fmt, 64, 256), code_buffers(fmt, 64, 256)
        engine.quantize_block(FMT[fmt], x, c, s)
        engine.quantize(FMT[fmt], x, c0, s0)
        assert torch.equal(c, c0) and torch.equal(s, s0)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("typ", list(TYPE))
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (5, 33, 1), (70, 256, 8), (3, 1000, 0)])
def test_read_back(engine, fmt, typ, rows, cols, pad):
    rng = np.random.default_rng(8)
    cs, ss = block_shapes(FMT[fmt], rows, cols)
    codes, sf = rng.integers(0, 256, cs), rng.integers(0, 256, ss)
    if fmt == "mxf8":
        codes[(codes & 127) == 127] = 1
    if fmt == "nvfp4":
        sf &= 127
        sf[sf == 127] = 100
    else:
        sf = sf // 16 + 120  # 2^-7 .. 2^8: within every out type
    codes, sf = codes.astype(np.uint8), sf.astype(np.uint8)
    want = ref.values(codes, sf, fmt)[:, :cols] * 0.5
    out = dev(np.zeros((rows, cols)), TYPE[typ], pad)
    engine.dequantize_block(FMT[fmt], torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda(), out,
                            scale=0.5)
    # exact in fp32; one rounding
    exp = host(torch.as_tensor(want).to(torch.float32).to(TYPE[typ]))
    assert np.array_equal(host(out), exp)
    if pad:
        full = out.as_strided((rows, cols + pad), (cols + pad, 1))
        assert torch.isnan(full[:, cols:]).all()


@pytest.mark.parametrize("fmt", list(FMT))
def test_casts_feed_the_products_of_a_training_step(engine, fmt):
    T, N, K = 70, 96, 130
    rng = np.random.default_rng(9)
    x, w, dy = (rounded(rng.normal(size=s), "bf16") for s in ((T, K), (N, K), (T, N)))
    q = {}
    for name, a in (("x", x), ("w", w), ("dy", dy)):
        q[name] = code_buffers(fmt, *a.shape) + code_buffers(fmt, *a.shape[::-1])
        c, s, ct, st = q[name]
        engine.quantize_block(FMT[fmt], dev(a, torch.bfloat16), c, s, codes_t=ct, sf_t=st)

    def val(name, t):
        c, s = q[name][2 * t:2 * t + 2]
        return ref.values(u8(c), u8(s), fmt)

    for a, b, t, u, m, n in (("x", "w", 0, 0, T, N), ("dy", "w", 0, 1, T, K), ("dy", "x", 1, 1, N, K)):
        out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
        engine.gemm(q[a][2 * t], q[b][2 * u], out, FMT[fmt], sfa=q[a][2 * t + 1], sfb=q[b][2 * u + 1])
        engine.check()
        A, B = val(a, t), val(b, u)
        # fp32 sums of up to 160 products, one rounding to bf16
        bound = 160 * 2.0 ** -24 * (np.abs(A) @ np.abs(B).T) + 2.0 ** -8 * np.abs(A @ B.T) + 1e-30
        assert np.all(np.abs(host(out) - A @ B.T) <= bound)


def test_empty_casts_write_nothing(engine):
    for rows, cols in ((0, 64), (64, 0), (0, 0)):
        x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
        (c, s), (ct, st) = code_buffers("nvfp4", rows, cols), code_buffers("nvfp4", cols, rows)
        engine.quantize_block(FMT["nvfp4"], x, c, s, codes_t=ct, sf_t=st)
        engine.dequantize_block(FMT["nvfp4"], c, s, x)


# ------------------------------------------------------------------ the norm pass
def norm_case(typ, rows, cols, per, seed, gate=True):
    rng = np.random.default_rng(seed)
    a = {"x": rng.normal(size=(rows, cols)), "y": 3 * rng.normal(size=(rows, cols)),
         "w_post": 1 + 0.2 * rng.normal(size=cols), "w_pre": 1 + 0.2 * rng.normal(size=cols)}
    if gate:
        a["gate"] = rng.normal(size=(-(-rows // per), cols))
    return {k: rounded(v, typ) for k, v in a.items()}


def norm_bounds(a, per, v, h, r2, alpha, beta, typ, cols):
    """Bounds of x_out and h: the fp32 work before the one rounding.  rstd: the sum of cols
    squares is off by at most cols / 32 + 16 roundings in a thread and the tree, half of that
    relative in rstd; each element then sees at most 8 roundings of its terms."""
    e = (cols / 64 + 16) * 2.0 ** -24
    g = 1.0 if "gate" not in a else np.abs(a["gate"])[np.arange(len(v)) // per]
    terms = np.abs(alpha * a["x"])
    if "y" in a:
        z = a["y"]
        if "w_post" in a:
            z = z * ((z * z).mean(1, keepdims=True) + 1e-6) ** -0.5 * a["w_post"]
        terms = terms + np.abs(beta) * g * np.abs(z)
    bv = e * terms
    bx = bv + ULP[typ] * (np.abs(v) + bv) + TINY[typ]
    bh = None
    if h is not None:
        # h: its v, rstd(v), whose error is at most the largest relative error of v in the
        # 2-norm, and three roundings
        rel = np.linalg.norm(bv, axis=1, keepdims=True) / np.maximum(np.linalg.norm(v, axis=1, keepdims=True), 1e-30)
        bh = np.abs(r2[:, None] * a["w_pre"]) * bv + (e + rel) * np.abs(h)
        bh = bh, bh + ULP[typ] * (np.abs(h) + bh) + TINY[typ]
    return bx, bh


NORM_SIZES = [(1, 1), (1, 8), (3, 7), (5, 33), (2, 200), (301, 1000), (40, 1024), (4, 5000), (300, 8192),
              (2, 16384), (1, 32768)]


@pytest.mark.parametrize("typ", list(TYPE))
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_norm_pass(engine, typ, rows, cols):
    per = (1, 2, rows)[(rows + cols) % 3]
    a = norm_case(typ, rows, cols, per, rows + cols)
    v, h, r1, r2 = ref.norm_forward(**a, per=per, alpha=0.9, beta=0.7)
    pad = (0, 1, 8)[cols % 3]
    t = {k: dev(x, TYPE[typ], pad) if k in "xy" else torch.as_tensor(x).to(TYPE[typ]).cuda()
         for k, x in a.items()}
    xo, ho = (dev(np.zeros((rows, cols)), TYPE[typ], pad) for _ in range(2))
    s1, s2 = (torch.empty(rows, device="cuda") for _ in range(2))
    engine.residual_norm(t["x"], y=t["y"], gate=t["gate"], rows_per_gate=per, w_post=t["w_post"],
                         w_pre=t["w_pre"], x_out=xo, h=ho, rstd_post=s1, rstd_pre=s2, alpha=0.9, beta=0.7)
    bx, (_, bh) = norm_bounds(a, per, v, h, r2, 0.9, 0.7, typ, cols)
    assert np.all(np.abs(host(xo) - v) <= bx)
    assert np.all(np.abs(host(ho) - h) <= bh)
    e = (cols / 64 + 16) * 2.0 ** -24
    assert np.all(np.abs(host(s1) - r1) <= e * r1)
    rel = np.linalg.norm(bx, axis=1) / np.linalg.norm(v, axis=1)
    assert np.all(np.abs(host(s2) - r2) <= (e + rel) * r2)
    if pad:  # nothing beside the rows was written
        assert torch.isnan(ho.as_strided((rows, cols + pad), (cols + pad, 1))[:, cols:]).all()


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("typ", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (2, 200), (40, 1000), (300, 2048), (1, 8192)])
def test_norm_pass_into_codes(engine, fmt, typ, rows, cols):
    a = norm_case(typ, rows, cols, 1, 11)
    v, h, _, r2 = ref.norm_forward(**a, per=1)
    t = {k: torch.as_tensor(x).to(TYPE[typ]).cuda() for k, x in a.items()}
    c, s = code_buffers(fmt, rows, cols)
    ho = torch.empty_like(t["x"])
    engine.residual_norm(t["x"], y=t["y"], gate=t["gate"], w_post=t["w_post"], w_pre=t["w_pre"],
                         h=ho, codes=c, sf=s, h_format=FMT[fmt])
    _, (eh, bh) = norm_bounds(a, 1, v, h, r2, 1.0, 1.0, typ, cols)
    assert np.all(np.abs(host(ho) - h) <= bh)
    # each code is the element nearest to h over the stored scale, and that scale the one of
    # the block's largest magnitude, up to the fp32 error of h
    q, sc = ref.decode(u8(c), u8(s), fmt)
    kp, block = ref.up32(cols), ref.BLOCK[fmt]
    hp, ep = np.zeros((2, rows, kp))
    hp[:, :cols], ep[:, :cols] = h, eh
    assert np.all(q[:, cols:] == 0)
    amax = np.abs(hp).reshape(rows, -1, block).max(2)
    err = ep.reshape(rows, -1, block).max(2)
    lo, hi = (ref.cast(np.repeat(np.maximum(amax + d, 0), block, 1), fmt)[1] for d in (-err, err))
    assert np.all((sc >= lo) & (sc <= hi))
    sr = np.repeat(sc, block, 1)
    top = ref.GRID[fmt][-1]
    with np.errstate(divide="ignore", invalid="ignore"):
        x = np.where(sr > 0, hp / sr, 0)
        tol = np.where(sr > 0, ep / sr, 0) + 2.0 ** -22 * np.abs(x)
    # the distance to the code is the distance to the nearest element, within twice the error
    xc = np.clip(x, -top, top)
    best = np.abs(np.abs(xc) - ref.nearest(np.abs(xc), ref.GRID[fmt]))
    assert np.all(np.abs(q - xc) <= best + 2 * tol)


@pytest.mark.parametrize("typ", ["bf16", "f32"])
@pytest.mark.parametrize("drop", [("y", "gate", "w_post"), ("gate",), ("w_post",), ("gate", "w_post"),
                                  ("w_pre",)])
def test_norm_pass_without_parts(engine, typ, drop):
    a = norm_case(typ, 9, 72, 3, 12)
    for k in drop:
        del a[k]
    v, h, _, r2 = ref.norm_forward(**a, per=3, alpha=0.5, beta=2.0)
    t = {k: torch.as_tensor(x).to(TYPE[typ]).cuda() for k, x in a.items()}
    x, w_pre = t.pop("x"), t.pop("w_pre", None)
    ho = torch.empty_like(x) if w_pre is not None else None
    # x_out may be x
    engine.residual_norm(x, rows_per_gate=3, w_pre=w_pre, x_out=x, h=ho, alpha=0.5, beta=2.0, **t)
    bx, bh = norm_bounds(a, 3, v, h, r2, 0.5, 2.0, typ, 72)
    assert np.all(np.abs(host(x) - v) <= bx)
    if ho is not None:
        assert np.all(np.abs(host(ho) - h) <= bh[1])


def test_norm_pass_of_zero_and_bad_rows(engine):
    a = norm_case("f32", 4, 64, 1, 13)
    for k in ("x", "y"):
        a[k][0] = 0
    a["y"][2, 5], a["x"][3, 9] = np.inf, np.nan
    t = {k: torch.as_tensor(x).float().cuda() for k, x in a.items()}
    x = t.pop("x")
    ho, xo = torch.empty_like(x), torch.empty_like(x)
    c, s = code_buffers("mxf8", 4, 64)
    engine.residual_norm(x, x_out=xo, h=ho, codes=c, sf=s, h_format=FMT["mxf8"], **t)
    assert torch.all(ho[0] == 0) and torch.all(xo[0] == 0)  # rstd = 1 / sqrt(eps): finite
    assert torch.isfinite(ho[1]).all()
    assert torch.isnan(ho[2]).any() and torch.isnan(ho[3]).all()
    assert not np.any(np.isnan(ref.values(u8(c), u8(s), "mxf8")[:2]))
    assert np.all(u8(s)[3] == 255)


def test_no_rows(engine):
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    engine.residual_norm(x, w_pre=w, h=torch.empty_like(x))
    dw = torch.full((64,), 7.0, device="cuda")
    engine.residual_norm_backward(x, x, torch.empty(0, device="cuda"), w, torch.empty_like(x), dw_pre=dw)
    assert torch.all(dw == 0)


# ------------------------------------------------------------------ its gradient
def grad_bounds(a, v, dh, dxo, r1, r2, per, alpha, beta, typ, cols, rows):
    """Bounds of the gradients from the same formula on magnitudes: every term's size times
    the number of roundings on its way (sums over cols inside, over rows for weights)."""
    e = (cols / 32 + 32) * 2.0 ** -24
    p, vh = np.abs(a["w_pre"] * dh), np.abs(v * r2[:, None])
    mdv = np.abs(dxo) + r2[:, None] * (p + vh * (p * vh).mean(1, keepdims=True))
    g = np.abs(a["gate"])[np.arange(rows) // per]
    yh = np.abs(a["y"] * r1[:, None])
    mdz = abs(beta) * g * mdv
    u = mdz * np.abs(a["w_post"])
    # the mean of u yh goes through sums of both parts of dv, whose magnitudes mdv adds up
    mdy = r1[:, None] * (u + yh * (u * yh).mean(1, keepdims=True))
    out = {"dx": e * abs(alpha) * mdv, "dy": e * mdy}
    f = e + rows * 2.0 ** -24
    out["dw_pre"] = f * (np.abs(dh) * vh).sum(0)
    out["dw_post"] = f * (mdz * yh).sum(0)
    out["dgate"] = np.zeros(a["gate"].shape)
    np.add.at(out["dgate"], np.arange(rows) // per, f * abs(beta) * yh * np.abs(a["w_post"]) * mdv)
    return out


GRAD_SIZES = [(1, 1, 1), (1, 40, 1), (3, 7, 3), (5, 33, 2), (67, 200, 1), (130, 264, 50), (301, 1000, 301),
              (301, 1000, 3), (9, 5000, 9), (40, 8192, 40), (300, 4096, 100), (2, 20000, 1), (600, 136, 256)]


@pytest.mark.parametrize("typ", list(TYPE))
@pytest.mark.parametrize("rows,cols,per", GRAD_SIZES)
@pytest.mark.parametrize("pad", [0, 1])
def test_norm_gradient(engine, typ, rows, cols, per, pad):
    rng = np.random.default_rng(rows + cols + per)
    a = norm_case(typ, rows, cols, per, rows * 3 + cols)
    dh, dxo, v = (rounded(rng.normal(size=(rows, cols)), typ) for _ in range(3))
    r1, r2 = (rounded(1 / np.sqrt((m * m).mean(1) + 1e-6), "f32") for m in (a["y"], v))
    want = ref.norm_backward(dh, dxo, v, r2, a["w_pre"], a["y"], r1, a["w_post"], a["gate"], per, 0.9, 0.7)
    bound = grad_bounds(a, v, dh, dxo, r1, r2, per, 0.9, 0.7, typ, cols, rows)
    dt = TYPE[typ]
    w1, w2, g = (torch.as_tensor(a[k]).to(dt).cuda() for k in ("w_post", "w_pre", "gate"))
    f1, f2 = (torch.as_tensor(r).float().cuda() for r in (r1, r2))
    out = {k: dev(np.zeros((rows, cols)), dt, pad) for k in ("dx", "dy")}
    out.update({k: torch.full(want[k].shape, float("nan"), device="cuda") for k in ("dgate", "dw_post", "dw_pre")})

    def call():
        engine.residual_norm_backward(
            dev(dh, dt, pad), dev(v, dt, pad), f2, w2, out["dx"], dx_out=dev(dxo, dt, pad),
            y=dev(a["y"], dt, pad), rstd_post=f1, w_post=w1, gate=g, rows_per_gate=per, dy=out["dy"],
            dgate=out["dgate"], dw_post=out["dw_post"], dw_pre=out["dw_pre"], alpha=0.9, beta=0.7)
        return {k: o.clone() for k, o in out.items()}

    first = call()
    for k, b in bound.items():
        if k in ("dx", "dy"):
            b = b + ULP[typ] * (np.abs(want[k]) + b) + TINY[typ]
        assert np.all(np.abs(host(out[k]) - want[k]) <= b + 1e-37), k
    again = call()  # sums in a fixed order: the same bits
    for k in first:
        assert torch.equal(first[k], again[k])


@pytest.mark.parametrize("parts", ["no dh", "no dx_out", "no y", "no gate", "no w_post", "only weights"])
@pytest.mark.parametrize("cols", [40, 2048])
def test_norm_gradient_without_parts(engine, parts, cols):
    rows, per = 50, 20
    rng = np.random.default_rng(14)
    a = norm_case("f32", rows, cols, per, 15)
    dh, dxo, v = (rounded(rng.normal(size=(rows, cols)), "f32") for _ in range(3))
    r1, r2 = (rounded(1 / np.sqrt((m * m).mean(1) + 1e-6), "f32") for m in (a["y"], v))
    k = dict(dh=dh, dxo=dxo, v=v, r2=r2, w_pre=a["w_pre"], y=a["y"], r1=r1, w_post=a["w_post"], gate=a["gate"])
    if parts == "no dh":
        k.update(dh=None, v=None, r2=None, w_pre=None)
    elif parts == "no dx_out":
        k.update(dxo=None)
    elif parts == "no y":
        k.update(y=None, r1=None, w_post=None, gate=None)
    elif parts == "no gate":
        k.update(gate=None)
    elif parts == "no w_post":
        k.update(r1=None, w_post=None)
    want = ref.norm_backward(**k, per=per, alpha=0.9, beta=0.7)
    t = {n: None if m is None else torch.as_tensor(m).float().cuda() for n, m in k.items()}
    out = {n: torch.full(w.shape, float("nan"), device="cuda") for n, w in want.items()}
    if parts == "only weights":
        out = {n: o for n, o in out.items() if n[:2] == "dw"}
    engine.residual_norm_backward(
        t["dh"], t["v"], t["r2"], t["w_pre"], out.get("dx"), dx_out=t["dxo"], y=t["y"], rstd_post=t["r1"],
        w_post=t["w_post"], gate=t["gate"], rows_per_gate=per, dy=out.get("dy"), dgate=out.get("dgate"),
        dw_post=out.get("dw_post"), dw_pre=out.get("dw_pre"), alpha=0.9, beta=0.7)
    for n, o in out.items():
        # sums of at most 2048 columns and 50 rows of terms up to about 30 times the result's rms
        scale = np.sqrt((want[n] ** 2).mean()) + np.abs(want[n])
        assert np.all(np.abs(host(o) - want[n]) <= 30 * (2048 / 32 + 82) * 2.0 ** -24 * scale), n


def test_norm_gradient_against_differences(engine):
    # the kernels of both directions in fp32 against central differences of the forward kernel's
    # definition in 64 bits, whose own error is 1e-7 here; fp32 terms are of order 10
    rows, cols, per = 6, 48, 2
    a = norm_case("f32", rows, cols, per, 16)
    rng = np.random.default_rng(17)
    cv, ch = (rounded(rng.normal(size=(rows, cols)), "f32") for _ in range(2))
    t = {k: torch.as_tensor(x).float().cuda() for k, x in a.items()}
    xo, ho = torch.empty(rows, cols, device="cuda"), torch.empty(rows, cols, device="cuda")
    s1, s2 = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    engine.residual_norm(t["x"], y=t["y"], gate=t["gate"], rows_per_gate=per, w_post=t["w_post"],
                         w_pre=t["w_pre"], x_out=xo, h=ho, rstd_post=s1, rstd_pre=s2)
    out = {k: torch.empty_like(t[n]) for k, n in (("dx", "x"), ("dy", "y"), ("dgate", "gate"),
                                                  ("dw_post", "w_post"), ("dw_pre", "w_pre"))}
    f = torch.float32
    engine.residual_norm_backward(torch.as_tensor(ch).to(f).cuda(), xo, s2, t["w_pre"], out["dx"],
                                  dx_out=torch.as_tensor(cv).to(f).cuda(), y=t["y"], rstd_post=s1,
                                  w_post=t["w_post"], gate=t["gate"], rows_per_gate=per, dy=out["dy"],
                                  dgate=out["dgate"], dw_post=out["dw_post"], dw_pre=out["dw_pre"])

    def loss(q):
        v, h, _, _ = ref.norm_forward(**q, per=per)
        return (cv * v).sum() + (ch * h).sum()

    for key, name in (("dx", "x"), ("dy", "y"), ("dgate", "gate"), ("dw_post", "w_post"), ("dw_pre", "w_pre")):
        got = host(out[key])
        for at in list(np.ndindex(*a[name].shape))[::11]:
            q = {k: m.copy() for k, m in a.items()}
            q[name][at] += 1e-5
            hi = loss(q)
            q[name][at] -= 2e-5
            assert abs((hi - loss(q)) / 2e-5 - got[at]) < 2e-4, (key, at)


# ------------------------------------------------------------------ the product of a few tokens
def random_weights(fmt, N, K, seed, lo=118, hi=130):
    """Codes and scale bytes of N x K with zero padding, and their values."""
    rng = np.random.default_rng(seed)
    cs, ss = block_shapes(FMT[fmt], N, K)
    codes = rng.integers(0, 256, cs).astype(np.uint8)
    if fmt == "mxf8":
        codes[(codes & 127) == 127] = 1
        codes[:, K:] = 0
    else:
        nib = np.stack([codes & 15, codes >> 4], 2).reshape(N, -1)
        nib[:, K:] = 0
        codes = (nib[:, 0::2] | (nib[:, 1::2] << 4)).astype(np.uint8)
    sf = rng.integers(8, 100, ss) if fmt == "nvfp4" else rng.integers(lo, hi, ss)
    sf = sf.astype(np.uint8)
    return codes, sf, ref.values(codes, sf, fmt)[:, :K]


def check_linear(engine, x, codes, sf, w, fmt, typ, alpha=0.75, pad=0):
    T, N = x.shape[0], w.shape[0]
    out = dev(np.zeros((T, N)), TYPE[typ], pad)
    engine.linear(dev(x, TYPE[typ], pad), torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda(), out,
                  FMT[fmt], alpha=alpha)
    want = alpha * (x @ w.T)
    # fp32 sums of K products, x's error of 2^-40 of its row's largest, one rounding
    K = x.shape[1]
    bound = (K + 8) * 2.0 ** -24 * alpha * (np.abs(x) @ np.abs(w).T)
    bound += 2.0 ** -39 * alpha * np.abs(x).max(1, initial=0, keepdims=True) * np.abs(w).sum(1)
    bound += ULP[typ] * (np.abs(want) + bound) + TINY[typ]
    with np.errstate(over="ignore"):
        exp = want if typ == "f16" and np.abs(want).max(initial=0) > 65504 else want
    got = host(out)
    fine = np.abs(exp) < (65000 if typ == "f16" else 3e38)
    assert np.all(np.abs(got - exp)[fine] <= bound[fine])
    if pad:
        assert torch.isnan(out.as_strided((T, N + pad), (N + pad, 1))[:, N:]).all()


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("T,N,K", [(1, 1, 1), (1, 16, 32), (2, 15, 33), (5, 1001, 2050), (8, 17, 100),
                                   (9, 64, 4096), (16, 100, 777), (17, 33, 160), (33, 130, 512), (64, 128, 1024),
                                   (65, 40, 96), (130, 20, 300), (1, 300, 16384), (7, 4096, 2048)])
def test_few_tokens(engine, fmt, typ, T, N, K):
    x = rounded(np.random.default_rng(T + N + K).normal(size=(T, K)), typ)
    codes, sf, w = random_weights(fmt, N, K, K + 1)
    s = 1 / 64 if fmt == "mxf8" else 1.0
    check_linear(engine, rounded(x * s, typ), codes, sf, w, fmt, typ, pad=(0, 8, 1)[(T + N + K) % 3])


@pytest.mark.parametrize("fmt", ["mxf4", "mxf8"])
def test_few_tokens_with_scales_far_apart(engine, fmt):
    # neighbouring blocks whose scales differ by more than fp16's range, and x that makes up for it
    T, N, K = 3, 40, 512
    codes, sf, w = random_weights(fmt, N, K, 31, 90, 160)
    rng = np.random.default_rng(32)
    block_max = 2.0 ** (sf.astype(float).mean(0) - 127)
    x = rounded(rng.normal(size=(T, K)) / np.repeat(block_max, 32) ** 0.5, "bf16")
    check_linear(engine, x, codes, sf, w, fmt, "bf16")
    # one block that counts, behind far larger scales on blocks of zeros
    codes[:, :] = 0
    sf[:, :] = 200
    codes[:, 0] = 0x22 if fmt == "mxf4" else 0x38
    sf[:, 0] = 100
    w = ref.values(codes, sf, fmt)[:, :K]
    check_linear(engine, x, codes, sf, w, fmt, "bf16")


def test_few_tokens_with_x_of_a_wide_range(engine):
    T, N, K = 2, 64, 256
    rng = np.random.default_rng(33)
    x = rng.normal(size=(T, K)) * 2.0 ** rng.integers(-60, 60, size=(T, K))
    x[1] *= 2.0 ** -60
    for fmt in FMT:
        codes, sf, w = random_weights(fmt, N, K, 34)
        check_linear(engine, rounded(x, "bf16"), codes, sf, w, fmt, "bf16", alpha=2.0 ** -20)


@pytest.mark.parametrize("fmt", list(FMT))
def test_few_tokens_with_infinities_and_nan(engine, fmt):
    N, K = 32, 128
    codes, sf, w = random_weights(fmt, N, K, 35)
    x = np.random.default_rng(36).normal(size=(4, K))
    x[1, 7], x[2, 9] = np.inf, np.nan
    x = rounded(x / 64, "bf16")
    out = torch.empty(4, N, dtype=torch.bfloat16, device="cuda")
    engine.linear(dev(x, torch.bfloat16), torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda(), out, FMT[fmt])
    got = host(out)
    assert np.isfinite(got[[0, 3]]).all() and np.isnan(got[2]).all()
    inf = w[:, 7] != 0
    assert np.array_equal(got[1][inf], np.sign(w[inf, 7]) * np.inf) and np.isnan(got[1][~inf]).all()
    # a NaN scale reaches the outputs of its row alone
    sf[5, 0] = 127 if fmt == "nvfp4" else 255
    engine.linear(dev(x[:1], torch.bfloat16), torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda(),
                  out[:1], FMT[fmt])
    got = host(out[:1])
    assert np.isnan(got[0, 5]) and np.isfinite(np.delete(got[0], 5)).all()


def test_few_tokens_repeat_to_the_bit_on_another_stream(engine):
    codes, sf, w = random_weights("nvfp4", 48, 8192, 37)
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda()
    x = dev(np.random.default_rng(38).normal(size=(3, 8192)), torch.bfloat16)
    outs = [torch.empty(3, 48, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    engine.linear(x, c, s, outs[0], FMT["nvfp4"])
    engine.linear(x, c, s, outs[1], FMT["nvfp4"])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    engine.linear(x, c, s, outs[2], FMT["nvfp4"], stream=side)
    side.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_few_tokens_in_a_graph(engine):
    codes, sf, _ = random_weights("mxf4", 64, 4096, 39)
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda()
    x = dev(np.random.default_rng(40).normal(size=(2, 4096)), torch.float16)
    eager, out = (torch.empty(2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    engine.linear(x, c, s, eager, FMT["mxf4"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine.linear(x, c, s, out, FMT["mxf4"])
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_no_tokens(engine):
    codes, sf, _ = random_weights("nvfp4", 16, 64, 41)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    engine.linear(x, torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda(),
                  torch.empty(0, 16, dtype=torch.bfloat16, device="cuda"), FMT["nvfp4"])


# ------------------------------------------------------------------ tens of tokens
@pytest.mark.parametrize("fmt", ["mxf4", "mxf8"])
@pytest.mark.parametrize("T,N,K", [(9, 40, 512), (70, 131, 352), (130, 20, 2400)])
def test_tens_of_tokens_with_scales_far_apart(engine, fmt, T, N, K):
    # blocks outside fp16's range of their row's reference, here and there or nearly all
    rng = np.random.default_rng(T)
    for lo, hi in ((90, 160), (112, 134)):
        codes, sf, w = random_weights(fmt, N, K, 51 + lo, lo, hi)
        block_max = 2.0 ** (sf[:, :K // 32].astype(float).mean(0) - 127)
        x = rounded(rng.normal(size=(T, K)) / np.repeat(block_max, 32) ** 0.5, "bf16")
        check_linear(engine, x, codes, sf, w, fmt, "bf16")
    # one block that counts, behind far larger scales on blocks of zeros
    codes[:, :] = 0
    sf[:, :] = 200
    codes[:, 0] = 0x22 if fmt == "mxf4" else 0x38
    sf[:, 0] = 100
    check_linear(engine, x, codes, sf, ref.values(codes, sf, fmt)[:, :K], fmt, "bf16")


@pytest.mark.parametrize("fmt", list(FMT))
def test_tens_of_tokens_with_x_of_a_wide_range(engine, fmt):
    T, N, K = 20, 64, 256
    rng = np.random.default_rng(52)
    x = rng.normal(size=(T, K)) * 2.0 ** rng.integers(-60, 60, size=(T, K))
    x[1] *= 2.0 ** -60
    x[2] = 0
    codes, sf, w = random_weights(fmt, N, K, 53)
    check_linear(engine, rounded(x, "bf16"), codes, sf, w, fmt, "bf16", alpha=2.0 ** -20)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("T", [3, 12])
def test_products_of_infinities_and_nan(engine, fmt, T):
    N, K = 150, 320
    codes, sf, w = random_weights(fmt, N, K, 54)
    x = rounded(np.random.default_rng(55).normal(size=(T, K)) / 64, "bf16")
    x[1, 300], x[2, 9] = -np.inf, np.nan
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda()
    out = torch.empty(T, N, dtype=torch.bfloat16, device="cuda")
    engine.linear(dev(x, torch.bfloat16), c, s, out, FMT[fmt])
    got = host(out)
    assert np.isfinite(np.delete(got, (1, 2), 0)).all() and np.isnan(got[2]).all()
    some = w[:, 300] != 0
    assert np.array_equal(got[1][some], np.sign(w[some, 300]) * -np.inf) and np.isnan(got[1][~some]).all()
    # a NaN scale reaches the outputs of its row alone, where it is a row's first, and its last
    x[1, 300] = x[2, 9] = 0
    s[5, 0] = s[140, -1] = 127 if fmt == "nvfp4" else 255
    engine.linear(dev(x, torch.bfloat16), c, s, out, FMT[fmt])
    got = host(out)
    assert np.isnan(got[:, [5, 140]]).all() and np.isfinite(np.delete(got, (5, 140), 1)).all()
    # with blocks that are left out of the tensor product an infinity may become a NaN, not a number
    if fmt != "nvfp4":
        codes, sf, _ = random_weights(fmt, N, K, 56, 60, 190)
        x[0, 40] = np.inf
        engine.linear(dev(x, torch.bfloat16), torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda(), out,
                      FMT[fmt])
        got = host(out)
        assert not np.isfinite(got[0]).any() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("T", [1, 3, 7])
def test_few_tokens_with_many_weights(engine, fmt, T):
    # 2^26 weights, all of x in one CTA or not
    N, K = 4112, 16352
    rng = np.random.default_rng(63)
    x = rounded(rng.normal(size=(T, K)) / 64, "bf16")
    codes, sf, w = random_weights(fmt, N, K, 64)
    check_linear(engine, x, codes, sf, w, fmt, "bf16")


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("T", [5, 24])
def test_weights_and_scales_at_odd_places(engine, fmt, T):
    # codes on 16 bytes, scales on two, neither on the allocation's start
    N, K = 70, 1120
    codes, sf, w = random_weights(fmt, N, K, 57)
    c = torch.zeros(codes.size + 16, dtype=torch.uint8, device="cuda")[16:].view(codes.shape)
    s = torch.zeros(sf.size + 2, dtype=torch.uint8, device="cuda")[2:].view(sf.shape)
    c.copy_(torch.from_numpy(codes)), s.copy_(torch.from_numpy(sf))
    x = dev(np.random.default_rng(58).normal(size=(T, K)), torch.float16, 3)
    here, there = (torch.empty(T, N, dtype=torch.float16, device="cuda") for _ in range(2))
    engine.linear(x, c, s, here, FMT[fmt], alpha=1 / 64)
    engine.linear(x, torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda(), there, FMT[fmt], alpha=1 / 64)
    assert torch.equal(here, there) and torch.isfinite(here).all()


def test_tens_of_tokens_repeat_to_the_bit_on_another_stream_and_in_a_graph(engine):
    codes, sf, _ = random_weights("mxf8", 300, 8192, 59)
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda()
    x = dev(np.random.default_rng(60).normal(size=(40, 8192)) / 64, torch.bfloat16)
    first, out = (torch.empty(40, 300, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    engine.linear(x, c, s, first, FMT["mxf8"])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    engine.linear(x, c, s, out, FMT["mxf8"], stream=side)
    side.synchronize()
    assert torch.equal(first, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine.linear(x, c, s, out, FMT["mxf8"])
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, out)
    engine.check()


def test_tens_of_tokens_with_the_shortest_wait_limit(engine):
    # under a limit of a microsecond a call either is right or reports that a wait ran out; nothing
    # is left behind, and the next call with the usual limit is right
    codes, sf, _ = random_weights("nvfp4", 1000, 8192, 65)
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda()
    x = dev(np.random.default_rng(66).normal(size=(20, 8192)) / 64, torch.bfloat16)
    first, out = (torch.empty(20, 1000, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    engine.linear(x, c, s, first, FMT["nvfp4"])
    engine.check()
    for _ in range(20):
        engine.set_wait_limit(1000)
        try:
            out.zero_()
            engine.linear(x, c, s, out, FMT["nvfp4"])
            engine.check()
            assert torch.equal(first, out)
        except b2g.B2GError as e:
            assert e.status == b2g._lib.B2G_ERR_TIMEOUT
        finally:
            engine.set_wait_limit(0)
        out.zero_()
        engine.linear(x, c, s, out, FMT["nvfp4"])
        engine.check()
        assert torch.equal(first, out)


@pytest.mark.parametrize("typ", list(TYPE))
@pytest.mark.parametrize("cols", [1, 2, 7, 9, 15, 17, 31, 257])
def test_norm_passes_of_narrow_rows_at_odd_places(engine, typ, cols):
    # the words that hold a row's ends may hold its neighbours' too, and what lies outside
    rows, per = 9, 2
    a = norm_case(typ, rows, cols, per, 61 + cols)
    v, h, r1, r2 = ref.norm_forward(**a, per=per)
    dt = TYPE[typ]

    def odd(m):  # contiguous, one element behind an aligned place
        flat = torch.full((m.size + 2,), float("nan"), dtype=dt, device="cuda")
        flat[1:-1] = torch.as_tensor(m.reshape(-1)).to(dt)
        return flat, flat[1:-1].view(m.shape)

    t = {k: odd(m)[1] for k, m in a.items()}
    t["w_pre"], t["w_post"] = t["w_pre"].view(-1), t["w_post"].view(-1)
    xo, ho, dx, dy = (odd(np.zeros((rows, cols))) for _ in range(4))
    s1, s2 = (torch.empty(rows, device="cuda") for _ in range(2))
    engine.residual_norm(t["x"], y=t["y"], gate=t["gate"], rows_per_gate=per, w_post=t["w_post"],
                         w_pre=t["w_pre"], x_out=xo[1], h=ho[1], rstd_post=s1, rstd_pre=s2)
    bx, (_, bh) = norm_bounds(a, per, v, h, r2, 1.0, 1.0, typ, cols)
    assert np.all(np.abs(host(xo[1]) - v) <= bx) and np.all(np.abs(host(ho[1]) - h) <= bh)

    rng = np.random.default_rng(cols)
    dh, dxo, v = (rounded(rng.normal(size=(rows, cols)), typ) for _ in range(3))
    r1, r2 = (rounded(1 / np.sqrt((m * m).mean(1) + 1e-6), "f32") for m in (a["y"], v))
    want = ref.norm_backward(dh, dxo, v, r2, a["w_pre"], a["y"], r1, a["w_post"], a["gate"], per, 1.0, 1.0)
    out = {k: torch.empty(want[k].shape, device="cuda") for k in ("dgate", "dw_post", "dw_pre")}
    engine.residual_norm_backward(
        odd(dh)[1], odd(v)[1], torch.as_tensor(r2).float().cuda(), t["w_pre"], dx[1], dx_out=odd(dxo)[1],
        y=t["y"], rstd_post=torch.as_tensor(r1).float().cuda(), w_post=t["w_post"], gate=t["gate"],
        rows_per_gate=per, dy=dy[1], **out)
    out.update(dx=dx[1], dy=dy[1])
    for k, b in grad_bounds(a, v, dh, dxo, r1, r2, per, 1.0, 1.0, typ, cols, rows).items():
        if k in ("dx", "dy"):
            b = b + ULP[typ] * (np.abs(want[k]) + b) + TINY[typ]
        assert np.all(np.abs(host(out[k]) - want[k]) <= b + 1e-37), k
    for flat, _ in (xo, ho, dx, dy):
        assert torch.isnan(flat[[0, -1]]).all()


# ------------------------------------------------------------------ refusals
def test_refusals(engine):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    r = torch.ones(4, device="cuda")
    c, s = code_buffers("nvfp4", 4, 64)
    fmt = FMT["nvfp4"]

    def refuses(status, f, *args, **kw):
        with pytest.raises(b2g.B2GError) as e:
            f(*args, **kw)
        assert e.value.status == status

    q = engine.quantize_block
    refuses(4, q, b2g.FMT_E4M3, x, c, s)                    # no block scales
    refuses(1, q, fmt, x)                                   # no output
    refuses(1, q, fmt, x, c)                                # codes without scales
    refuses(1, q, fmt, x, c[:, :16], s)                     # too few codes
    refuses(1, q, fmt, x.t(), c, s)                         # strided rows
    refuses(1, q, fmt, x.double(), c, s)                    # type
    refuses(1, q, fmt, x, c, s, scale=0.0)
    refuses(1, q, fmt, x, c, s, scale=float("nan"))
    refuses(1, q, fmt, x, c, s, rand=x)                     # not bytes
    odd = torch.zeros(4 * 32 + 1, dtype=torch.uint8, device="cuda")[1:].view(4, 32)
    refuses(1, q, fmt, x, odd, s)                           # codes off 16 bytes
    refuses(1, engine.dequantize_block, fmt, c, s, torch.empty(4, 96, device="cuda"))
    refuses(1, engine.dequantize_block, fmt, c.cpu(), s, x)
    n = engine.residual_norm
    refuses(1, n, x)                                        # no output
    refuses(1, n, x, h=x)                                   # h without w_pre
    refuses(1, n, x, w_pre=w, h=x, gate=x)                  # gate without y
    refuses(1, n, x, y=x, gate=x, rows_per_gate=2, x_out=x)  # gate rows
    refuses(1, n, x, y=x, gate=x, rows_per_gate=0, x_out=x)
    refuses(1, n, x, w_pre=w.float(), h=x)
    refuses(1, n, x, w_pre=w, h=x, eps=-1.0)
    refuses(4, n, x, w_pre=w, codes=c, sf=s, h_format=b2g.FMT_E4M3)
    wide = torch.zeros(1, 32776, dtype=torch.bfloat16, device="cuda")
    refuses(4, n, wide, x_out=wide)
    b = engine.residual_norm_backward
    refuses(1, b, None, None, None, None, x)                # no gradient
    refuses(1, b, x, None, r, w, x)                         # dh without x_out
    refuses(1, b, x, x, r, w, None)                         # no output
    refuses(1, b, x, x, r, w, x, y=x, w_post=w)             # w_post without rstd_post
    refuses(1, b, x, x, r, w, x, y=x, dgate=x.float())      # dgate without gate
    refuses(1, b, x, x, r, w, x, dy=x)                      # dy without y
    lin = engine.linear
    out = torch.empty(4, 4, dtype=torch.bfloat16, device="cuda")
    refuses(4, lin, x.float(), c, s, out.float(), fmt)      # x not 16-bit
    refuses(4, lin, x, c, s, out, b2g.FMT_BF16)
    refuses(1, lin, x, c[:2], s[:2], out, fmt)              # N
    refuses(1, lin, x[:, :32], c, s, out, fmt)              # K
    refuses(1, lin, x, c, None, out, fmt)
    engine.check()  # nothing was launched, and the handle still works
    engine.quantize_block(fmt, x, c, s)
