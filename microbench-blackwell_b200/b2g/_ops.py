"""Operators around a linear layer of a language model: microscaled casts, the norms,
gate and residual addition between blocks, and the product of a few tokens.

Methods of ``Engine``.  Every tensor is on the engine's device and every result goes
into a tensor the caller passes; a shape, type or layout that does not fit raises
``B2GError`` before anything is launched.  Formats are FMT_NVFP4, FMT_MXF4 and FMT_MXF8,
laid out as ``Engine.gemm`` reads them.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._errors import B2GError


class _Torch:
    """torch, imported at its first use: the package itself loads without it."""

    def __getattr__(self, name):
        import torch as module

        globals()["torch"] = module
        return getattr(module, name)


torch = _Torch()
_TYPES = {}  # b2g_dtype of a torch dtype
_BLOCK = {_lib.FMT_NVFP4: 16, _lib.FMT_MXF4: 32, _lib.FMT_MXF8: 32}
_byref = C.byref


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


class LinearOps:
    def _here(self, t, name):
        if t.get_device() != self.device:
            _refuse(f"{name} is not on cuda:{self.device}")
        return t.data_ptr()

    def _mat(self, t, name, rows, cols, dtype):
        """(pointer, leading dimension) of a rows x cols tensor with contiguous rows."""
        if t is None:
            return None, 0
        if t.dtype != dtype:
            _refuse(f"{name} is {t.dtype}, not {dtype}")
        if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols:
            _refuse(f"{name} is {tuple(t.shape)}, not {(rows, cols)}")
        ld, one = t.stride()
        if one != 1 and cols > 1:
            _refuse(f"{name}: elements of a row must be contiguous")
        return self._here(t, name), ld if rows > 1 else max(ld, cols)

    def _flat(self, t, name, shape, dtype):
        """Pointer of a contiguous tensor of that shape."""
        if t is None:
            return None
        if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
            _refuse(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
        return self._here(t, name)

    def _pair(self, fmt, codes, sf, name, rows, cols):
        if codes is None and sf is None:
            return None, None
        if codes is None or sf is None:
            _refuse(f"{name}: codes and scales go together")
        cs, ss = block_shapes(fmt, rows, cols)
        return (self._flat(codes, name, cs, torch.uint8),
                self._flat(sf, f"scales of {name}", ss, torch.uint8))

    def _raw_stream(self, stream):
        if stream is None:
            return torch._C._cuda_getCurrentRawStream(self.device)
        return stream.cuda_stream

    def _type(self, t, name):
        if not _TYPES:
            _TYPES.update({torch.float32: _lib.F32, torch.bfloat16: _lib.BF16,
                           torch.float16: _lib.F16})
        if t.dtype not in _TYPES or t.dim() != 2:
            _refuse(f"{name} must be a float32, bfloat16 or float16 matrix")
        return _TYPES[t.dtype]

    def quantize_block(self, fmt: int, x, codes=None, sf=None, *, codes_t=None, sf_t=None,
                       scale: float = 1.0, rand=None, stream=None):
        """b2g_block_quantize: x (rows x cols, fp32 / bf16 / fp16), times `scale`, to codes
        with one scale per block along the rows and / or (codes_t, sf_t) along the columns;
        shapes from ``block_shapes(fmt, rows, cols)`` and ``(fmt, cols, rows)``.  `rand`
        (uint8, x's shape): stochastic rounding with these random bytes."""
        kind = self._type(x, "x")
        rows, cols = x.shape
        px, ld = self._mat(x, "x", rows, cols, x.dtype)
        pc, ps = self._pair(fmt, codes, sf, "codes", rows, cols)
        pct, pst = self._pair(fmt, codes_t, sf_t, "codes_t", cols, rows)
        pr, ldr = self._mat(rand, "rand", rows, cols, torch.uint8)
        d = _lib.BlockQuantDesc(fmt, kind, rows, cols, ld, px, pc, ps, pct, pst, pr, ldr, scale)
        self._ok(self.lib.b2g_block_quantize(self.h, _byref(d), self._raw_stream(stream)),
                 "b2g_block_quantize")
        return codes if codes is not None else codes_t

    def dequantize_block(self, fmt: int, codes, sf, out, *, scale: float = 1.0, stream=None):
        """b2g_block_dequantize: out (rows x cols) = code * block scale * scale."""
        kind = self._type(out, "out")
        rows, cols = out.shape
        po, ld = self._mat(out, "out", rows, cols, out.dtype)
        if codes is None:
            _refuse("codes missing")
        pc, ps = self._pair(fmt, codes, sf, "codes", rows, cols)
        self._ok(self.lib.b2g_block_dequantize(self.h, fmt, pc, ps, rows, cols, kind, po, ld,
                                               scale, self._raw_stream(stream)),
                 "b2g_block_dequantize")
        return out

    def residual_norm(self, x, *, y=None, gate=None, rows_per_gate: int = 1, w_post=None,
                      w_pre=None, x_out=None, h=None, codes=None, sf=None, h_format: int = 0,
                      rstd_post=None, rstd_pre=None, eps: float = 1e-6, alpha: float = 1.0,
                      beta: float = 1.0, stream=None):
        """b2g_residual_norm: v = alpha * x + beta * gate * norm(y) * w_post, x_out = v and
        h = norm(v) * w_pre, as it is (h) and / or as codes and scales of h_format.  gate has
        one row for each rows_per_gate rows of x."""
        kind, dt = self._type(x, "x"), x.dtype
        rows, cols = x.shape
        px, ldx = self._mat(x, "x", rows, cols, dt)
        py, ldy = self._mat(y, "y", rows, cols, dt)
        po, ldo = self._mat(x_out, "x_out", rows, cols, dt)
        ph, ldh = self._mat(h, "h", rows, cols, dt)
        pg = None
        if gate is not None:
            if rows_per_gate < 1:
                _refuse("rows_per_gate < 1")
            pg = self._flat(gate, "gate", (-(-rows // rows_per_gate), cols), dt)
        pc, ps = self._pair(h_format, codes, sf, "codes", rows, cols)
        f32 = torch.float32
        d = _lib.ResidualNormDesc(
            kind, h_format, rows, cols, ldx, ldy, ldo, ldh, rows_per_gate, px, py, pg,
            self._flat(w_post, "w_post", (cols,), dt), self._flat(w_pre, "w_pre", (cols,), dt),
            po, ph, pc, ps, self._flat(rstd_post, "rstd_post", (rows,), f32),
            self._flat(rstd_pre, "rstd_pre", (rows,), f32), eps, alpha, beta)
        self._ok(self.lib.b2g_residual_norm(self.h, _byref(d), self._raw_stream(stream)),
                 "b2g_residual_norm")
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
        kind, dt = self._type(some, "dh"), some.dtype
        rows, cols = some.shape
        pdh, ldh = self._mat(dh, "dh", rows, cols, dt)
        pdo, ldo = self._mat(dx_out, "dx_out", rows, cols, dt)
        pv, ldv = self._mat(x_out, "x_out", rows, cols, dt)
        py, ldy = self._mat(y, "y", rows, cols, dt)
        pdx, lddx = self._mat(dx, "dx", rows, cols, dt)
        pdy, lddy = self._mat(dy, "dy", rows, cols, dt)
        f32 = torch.float32
        pg = pdg = None
        if gate is not None:
            if rows_per_gate < 1:
                _refuse("rows_per_gate < 1")
            shape = (-(-rows // rows_per_gate), cols)
            pg = self._flat(gate, "gate", shape, dt)
            pdg = self._flat(dgate, "dgate", shape, f32)
        elif dgate is not None:
            _refuse("dgate needs gate")
        d = _lib.ResidualNormGradDesc(
            kind, 0, rows, cols, ldh, ldo, ldv, ldy, lddx, lddy, rows_per_gate, pdh, pdo, pv, py,
            pg, self._flat(w_post, "w_post", (cols,), dt), self._flat(w_pre, "w_pre", (cols,), dt),
            self._flat(rstd_post, "rstd_post", (rows,), f32),
            self._flat(rstd_pre, "rstd_pre", (rows,), f32), pdx, pdy, pdg,
            self._flat(dw_post, "dw_post", (cols,), f32),
            self._flat(dw_pre, "dw_pre", (cols,), f32), alpha, beta)
        self._ok(self.lib.b2g_residual_norm_backward(self.h, _byref(d), self._raw_stream(stream)),
                 "b2g_residual_norm_backward")
        return dx

    def linear(self, x, w, sfw, out, fmt: int, *, alpha: float = 1.0, stream=None):
        """b2g_linear: out (T x N) = alpha * x (T x K, bf16 or fp16) . W^T for a few tokens,
        W (N x K) as codes and scales of quantize_block's shapes."""
        kind, dt = self._type(x, "x"), x.dtype
        T, K = x.shape
        if out.dim() != 2:
            _refuse("out must be a matrix")
        N = out.shape[1]
        px, ldx = self._mat(x, "x", T, K, dt)
        po, ldo = self._mat(out, "out", T, N, dt)
        if w is None:
            _refuse("w missing")
        pw, ps = self._pair(fmt, w, sfw, "w", N, K)
        d = _lib.LinearDesc(fmt, kind, T, N, K, ldx, ldo, px, pw, ps, po, alpha)
        self._ok(self.lib.b2g_linear(self.h, _byref(d), self._raw_stream(stream)), "b2g_linear")
        return out
