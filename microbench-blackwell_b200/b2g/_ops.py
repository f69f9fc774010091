"""Operators around a linear layer of a language model: microscaled casts, the norms,
gate and residual addition between blocks, and the product of a few tokens.

Methods of ``Engine``.  Every tensor is on the engine's device and every result goes
into a tensor the caller passes; a shape, type or layout that does not fit raises
``B2GError`` before anything is launched.  Formats are FMT_NVFP4, FMT_MXF4 and FMT_MXF8,
laid out as ``Engine.gemm`` reads them.
"""
from __future__ import annotations

from . import _lib
from ._errors import B2GError


class _Torch:
    """torch in a module's names, imported at its first use: the package loads without it."""

    def __init__(self, names):
        self._names = names

    def __getattr__(self, name):
        import torch as module

        self._names["torch"] = module
        return getattr(module, name)


torch = _Torch(globals())
_TYPES = {}  # b2g_dtype of a torch dtype
_BLOCK = {_lib.FMT_NVFP4: 16, _lib.FMT_MXF4: 32, _lib.FMT_MXF8: 32}


def _refuse(msg: str):
    raise B2GError(1, msg)


def _up32(n: int) -> int:
    return (n + 31) // 32 * 32


def block_shapes(fmt: int, rows: int, cols: int):
    """Shapes of the uint8 tensors (codes, scales) of a rows x cols matrix in `fmt`, blocks
    along the rows: cols are padded to a multiple of 32."""
    if fmt not in _BLOCK:
        raise B2GError(4, f"format {fmt} has no block scales")
    kp = _up32(cols)
    return (rows, kp if fmt == _lib.FMT_MXF8 else kp // 2), (rows, kp // _BLOCK[fmt])


def _mat(t, name, shape, dtype, device):
    """(pointer, leading dimension) of a matrix with contiguous rows; (0, 0) for None."""
    if t is None:
        return 0, 0
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device:
        _refuse(f"{name} is {t.dtype} {tuple(t.shape)} on {t.device}, not {dtype} {tuple(shape)} "
                f"on cuda:{device}")
    ld, one = t.stride()
    if one != 1 and shape[1] > 1:
        _refuse(f"{name}: elements of a row must be contiguous")
    return t.data_ptr(), ld if shape[0] > 1 else max(ld, shape[1])


def _flat(t, name, shape, dtype, device):
    """Pointer of a contiguous tensor; 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{device}")
    return t.data_ptr()


def _pair(fmt, codes, sf, name, rows, cols, device):
    """Pointers of codes and scales of a rows x cols matrix."""
    if codes is None and sf is None:
        return 0, 0
    if codes is None or sf is None:
        _refuse(f"{name}: codes and scales go together")
    cs, ss = block_shapes(fmt, rows, cols)
    u8 = torch.uint8
    return _flat(codes, name, cs, u8, device), _flat(sf, f"the scales of {name}", ss, u8, device)


def _type(t, name):
    if not _TYPES:
        _TYPES.update({torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16})
    kind = _TYPES.get(t.dtype)
    if kind is None or t.dim() != 2:
        _refuse(f"{name} must be a float32, bfloat16 or float16 matrix")
    return kind


class LinearOps:
    # A descriptor is packed in one step from its values (ctypes would set field by field).

    def _stream_of(self, stream):
        if stream is None:
            return torch._C._cuda_getCurrentRawStream(self.device)
        return stream.cuda_stream

    def quantize_block(self, fmt: int, x, codes=None, sf=None, *, codes_t=None, sf_t=None,
                       scale: float = 1.0, rand=None, stream=None):
        """b2g_block_quantize: x (rows x cols, fp32 / bf16 / fp16), times `scale`, to codes
        with one scale per block along the rows and / or (codes_t, sf_t) along the columns;
        shapes from ``block_shapes(fmt, rows, cols)`` and ``(fmt, cols, rows)``.  `rand`
        (uint8, x's shape): stochastic rounding with these random bytes."""
        kind, dev = _type(x, "x"), self.device
        shape = rows, cols = x.shape
        px, ld = _mat(x, "x", shape, x.dtype, dev)
        pc, ps = _pair(fmt, codes, sf, "codes", rows, cols, dev)
        pct, pst = _pair(fmt, codes_t, sf_t, "codes_t", cols, rows, dev)
        pr, ldr = _mat(rand, "rand", shape, torch.uint8, dev)
        d = _lib.BLOCK_QUANT(fmt, kind, rows, cols, ld, px, pc, ps, pct, pst, pr, ldr, scale, 0)
        st = self.lib.b2g_block_quantize(self.h, d, self._stream_of(stream))
        if st:
            self._ok(st, "b2g_block_quantize")
        return codes if codes is not None else codes_t

    def dequantize_block(self, fmt: int, codes, sf, out, *, scale: float = 1.0, stream=None):
        """b2g_block_dequantize: out (rows x cols) = code * block scale * scale."""
        kind, dev = _type(out, "out"), self.device
        shape = rows, cols = out.shape
        po, ld = _mat(out, "out", shape, out.dtype, dev)
        if codes is None:
            _refuse("codes missing")
        pc, ps = _pair(fmt, codes, sf, "codes", rows, cols, dev)
        st = self.lib.b2g_block_dequantize(self.h, fmt, pc, ps, rows, cols, kind, po, ld, scale,
                                           self._stream_of(stream))
        if st:
            self._ok(st, "b2g_block_dequantize")
        return out

    def residual_norm(self, x, *, y=None, gate=None, rows_per_gate: int = 1, w_post=None,
                      w_pre=None, x_out=None, h=None, codes=None, sf=None, h_format: int = 0,
                      rstd_post=None, rstd_pre=None, eps: float = 1e-6, alpha: float = 1.0,
                      beta: float = 1.0, stream=None):
        """b2g_residual_norm: v = alpha * x + beta * gate * norm(y) * w_post, x_out = v and
        h = norm(v) * w_pre, as it is (h) and / or as codes and scales of h_format.  gate has
        one row for each rows_per_gate rows of x."""
        kind, dt, dev = _type(x, "x"), x.dtype, self.device
        shape = rows, cols = x.shape
        px, ldx = _mat(x, "x", shape, dt, dev)
        py, ldy = _mat(y, "y", shape, dt, dev)
        po, ldo = _mat(x_out, "x_out", shape, dt, dev)
        ph, ldh = _mat(h, "h", shape, dt, dev)
        pg = 0
        if gate is not None:
            if rows_per_gate < 1:
                _refuse("rows_per_gate < 1")
            pg = _flat(gate, "gate", (-(-rows // rows_per_gate), cols), dt, dev)
        pc, ps = _pair(h_format, codes, sf, "codes", rows, cols, dev)
        f32, col, row = torch.float32, (cols,), (rows,)
        d = _lib.RESIDUAL_NORM(
            kind, h_format, rows, cols, ldx, ldy, ldo, ldh, rows_per_gate, px, py, pg,
            _flat(w_post, "w_post", col, dt, dev), _flat(w_pre, "w_pre", col, dt, dev), po, ph, pc,
            ps, _flat(rstd_post, "rstd_post", row, f32, dev),
            _flat(rstd_pre, "rstd_pre", row, f32, dev), eps, alpha, beta, 0)
        st = self.lib.b2g_residual_norm(self.h, d, self._stream_of(stream))
        if st:
            self._ok(st, "b2g_residual_norm")
        return x_out

    def residual_norm_backward(self, dh, x_out, rstd_pre, w_pre, dx, *, dx_out=None, y=None,
                               rstd_post=None, w_post=None, gate=None, rows_per_gate: int = 1,
                               dy=None, dgate=None, dw_post=None, dw_pre=None,
                               alpha: float = 1.0, beta: float = 1.0, stream=None):
        """b2g_residual_norm_backward: from dh and dx_out (gradients of h and x_out; either
        may be None) and what the forward pass had, dx and dy in the operands' type, dgate,
        dw_post and dw_pre in fp32.  Each output may be None."""
        some = dh if dh is not None else dx_out
        if some is None:
            _refuse("neither dh nor dx_out")
        kind, dt, dev = _type(some, "dh"), some.dtype, self.device
        shape = rows, cols = some.shape
        pdh, ldh = _mat(dh, "dh", shape, dt, dev)
        pdo, ldo = _mat(dx_out, "dx_out", shape, dt, dev)
        pv, ldv = _mat(x_out, "x_out", shape, dt, dev)
        py, ldy = _mat(y, "y", shape, dt, dev)
        pdx, lddx = _mat(dx, "dx", shape, dt, dev)
        pdy, lddy = _mat(dy, "dy", shape, dt, dev)
        f32, col, row = torch.float32, (cols,), (rows,)
        pg = pdg = 0
        if gate is not None:
            if rows_per_gate < 1:
                _refuse("rows_per_gate < 1")
            gates = -(-rows // rows_per_gate), cols
            pg = _flat(gate, "gate", gates, dt, dev)
            pdg = _flat(dgate, "dgate", gates, f32, dev)
        elif dgate is not None:
            _refuse("dgate needs gate")
        d = _lib.RESIDUAL_NORM_GRAD(
            kind, 0, rows, cols, ldh, ldo, ldv, ldy, lddx, lddy, rows_per_gate, pdh, pdo, pv, py,
            pg, _flat(w_post, "w_post", col, dt, dev), _flat(w_pre, "w_pre", col, dt, dev),
            _flat(rstd_post, "rstd_post", row, f32, dev),
            _flat(rstd_pre, "rstd_pre", row, f32, dev), pdx, pdy, pdg,
            _flat(dw_post, "dw_post", col, f32, dev), _flat(dw_pre, "dw_pre", col, f32, dev),
            alpha, beta)
        st = self.lib.b2g_residual_norm_backward(self.h, d, self._stream_of(stream))
        if st:
            self._ok(st, "b2g_residual_norm_backward")
        return dx

    def linear(self, x, w, sfw, out, fmt: int, *, alpha: float = 1.0, stream=None):
        """b2g_linear: out (T x N) = alpha * x (T x K, bf16 or fp16) . W^T for a few tokens,
        W (N x K) as codes and scales of quantize_block's shapes."""
        kind, dt, dev = _type(x, "x"), x.dtype, self.device
        T, K = x.shape
        if out.dim() != 2:
            _refuse("out must be a matrix")
        N = out.shape[1]
        px, ldx = _mat(x, "x", (T, K), dt, dev)
        po, ldo = _mat(out, "out", (T, N), dt, dev)
        if w is None:
            _refuse("w missing")
        pw, ps = _pair(fmt, w, sfw, "w", N, K, dev)
        d = _lib.LINEAR(fmt, kind, T, N, K, ldx, ldo, px, pw, ps, po, alpha, 0)
        st = self.lib.b2g_linear(self.h, d, self._stream_of(stream))
        if st:
            self._ok(st, "b2g_linear")
        return out
