"""Definitions, in 64 bits, of the operators around a linear layer, for their tests: grids
of the element formats, casts, the norm pass and its gradient.  numpy only."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6.0])
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)]
                + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1])
BLOCK = {"nvfp4": 16, "mxf4": 32, "mxf8": 32}
EMAX = {"mxf4": 2, "mxf8": 8}
GRID = {"nvfp4": E2M1, "mxf4": E2M1, "mxf8": E4M3}


def up32(n):
    return (n + 31) // 32 * 32


def nearest(q, grid):
    """The grid value nearest to q >= 0, of two equally near the one with the even index."""
    lo = np.clip(np.searchsorted(grid, q, side="right") - 1, 0, len(grid) - 2)
    d = (q - grid[lo]) - (grid[lo + 1] - q)
    return np.where((d > 0) | ((d == 0) & (lo % 2 == 1)), grid[lo + 1], grid[lo])


def cast(x, fmt, rand=None):
    """(values over their scale, scales) of x (rows x cols), blocks along the rows; rows
    padded with zeros to a multiple of 32."""
    rows, cols = x.shape
    kp, block, grid = up32(cols), BLOCK[fmt], GRID[fmt]
    b = np.zeros((rows, kp))
    b[:, :cols] = x
    b = b.reshape(-1, block)
    with np.errstate(invalid="ignore"):
        amax = np.abs(b).max(1)
    bad = ~np.isfinite(amax)
    b = np.where(bad[:, None], 0, b)
    amax = np.where(bad, 0, amax)
    if fmt == "nvfp4":
        s = nearest(np.minimum(amax / 6, 448), E4M3)
    else:
        e = np.frexp(amax)[1] - 1 - EMAX[fmt]
        s = 2.0 ** np.clip(np.where(amax > 0, e, -127), -127, 127)
    q = np.minimum(np.divide(np.abs(b), s[:, None], out=np.zeros_like(b), where=s[:, None] > 0),
                   grid[-1])
    if rand is None:
        m = nearest(q, grid)
    else:
        r = np.zeros((rows, kp))
        r[:, :cols] = rand
        lo = np.clip(np.searchsorted(grid, q, side="right") - 1, 0, len(grid) - 2)
        step = grid[lo + 1] - grid[lo]
        up = (q - grid[lo]) / step + (r.reshape(-1, block) + 0.5) / 256 >= 1
        m = np.where(up, grid[lo + 1], grid[lo])
    s = np.where(bad, np.nan, s)
    return (np.sign(b) * m).reshape(rows, kp), s.reshape(rows, -1)


def decode(codes, sf, fmt):
    """(values over their scale, scales) of stored uint8 codes and scale bytes."""
    rows = codes.shape[0]
    e4 = np.concatenate([E4M3, [np.nan]])
    if fmt == "mxf8":
        v = e4[codes & 127] * np.where(codes >> 7, -1.0, 1.0)
    else:
        c = np.stack([codes & 15, codes >> 4], 2).reshape(rows, -1)
        v = E2M1[c & 7] * np.where(c >> 3, -1.0, 1.0)
    if fmt == "nvfp4":
        s = e4[sf & 127]
    else:
        s = np.where(sf == 255, np.nan, 2.0 ** (sf.astype(np.float64) - 127))
    return v, s


def values(codes, sf, fmt):
    """What stored codes stand for (rows x padded cols)."""
    v, s = decode(codes, sf, fmt)
    return v * np.repeat(s, BLOCK[fmt], 1)


def norm_forward(x, y=None, gate=None, per=1, w_post=None, w_pre=None, eps=1e-6, alpha=1.0, beta=1.0):
    r1 = r2 = h = None
    v = alpha * x
    if y is not None:
        z = y
        if w_post is not None:
            r1 = ((y * y).mean(1) + eps) ** -0.5
            z = y * r1[:, None] * w_post
        v = v + beta * (1.0 if gate is None else gate[np.arange(len(x)) // per]) * z
    if w_pre is not None:
        r2 = ((v * v).mean(1) + eps) ** -0.5
        h = v * r2[:, None] * w_pre
    return v, h, r1, r2


def norm_backward(dh, dxo, v, r2, w_pre, y=None, r1=None, w_post=None, gate=None, per=1,
                  alpha=1.0, beta=1.0):
    """Gradients of norm_forward from its saved v, r1 and r2 (None: not computed)."""
    rows, cols = (dh if dh is not None else dxo).shape
    dv = np.zeros((rows, cols)) if dxo is None else dxo.copy()
    out = {}
    if dh is not None:
        vh = v * r2[:, None]
        p = w_pre * dh
        dv += r2[:, None] * (p - vh * (p * vh).mean(1, keepdims=True))
        out["dw_pre"] = (dh * vh).sum(0)
    out["dx"] = alpha * dv
    if y is not None:
        g = np.ones((rows, cols)) if gate is None else gate[np.arange(rows) // per]
        yh = y if r1 is None else y * r1[:, None]
        z = yh if w_post is None else yh * w_post
        if gate is not None:
            out["dgate"] = np.zeros(gate.shape)
            np.add.at(out["dgate"], np.arange(rows) // per, beta * z * dv)
        dz = beta * g * dv
        if w_post is None:
            out["dy"] = dz
        else:
            out["dw_post"] = (dz * yh).sum(0)
            u = dz * w_post
            out["dy"] = r1[:, None] * (u - yh * (u * yh).mean(1, keepdims=True))
    return out
