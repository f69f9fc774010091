"""Host side of the operators around a linear layer: struct layouts, refusals that need no
device, and the arithmetic their kernels rely on."""
import ctypes as C
import itertools

import numpy as np
import pytest

import b2g
import linear_ops_ref as ref
from b2g import _lib
from b2g._ops import LinearOps, block_shapes
from test_abi import _compile_and_run


@pytest.mark.parametrize("struct,ctype", [
    ("b2g_block_quant_desc", "BlockQuantDesc"), ("b2g_residual_norm_desc", "ResidualNormDesc"),
    ("b2g_residual_norm_grad_desc", "ResidualNormGradDesc"), ("b2g_linear_desc", "LinearDesc")])
def test_structs_match_the_c_layout(tmp_path, struct, ctype):
    cls = getattr(_lib, ctype)
    names = [n for n, _ in cls._fields_]
    lines = [f'  printf("{n} %zu\\n", offsetof({struct}, {n}));' for n in names]
    src = ("#include <stddef.h>\n#include <stdio.h>\n#include \"b2g.h\"\nint main(void) {\n"
           f'  printf("sizeof %zu\\n", sizeof({struct}));\n' + "\n".join(lines) + "\n  return 0;\n}\n")
    got = dict(line.split() for line in _compile_and_run(tmp_path, src).splitlines())
    assert int(got["sizeof"]) == C.sizeof(cls)
    for n in names:
        assert int(got[n]) == getattr(cls, n).offset, n


@pytest.mark.parametrize("pack,ctype", [
    (_lib.BLOCK_QUANT, "BlockQuantDesc"), (_lib.RESIDUAL_NORM, "ResidualNormDesc"),
    (_lib.RESIDUAL_NORM_GRAD, "ResidualNormGradDesc"), (_lib.LINEAR, "LinearDesc")])
def test_packed_descriptors_match_the_structs(pack, ctype):
    cls = getattr(_lib, ctype)
    values = [i + 1 for i in range(len(cls._fields_))]
    data = pack(*values)
    assert len(data) == C.sizeof(cls)
    d = cls.from_buffer_copy(data)
    assert [getattr(d, n) for n, _ in cls._fields_] == values


def test_a_null_handle_or_descriptor_is_refused():
    lib = _lib.load()
    assert lib.b2g_block_quantize(None, None, None) == 1
    assert lib.b2g_block_dequantize(None, 6, None, None, 1, 1, 1, None, 1, 1.0, None) == 1
    assert lib.b2g_residual_norm(None, None, None) == 1
    assert lib.b2g_residual_norm_backward(None, None, None) == 1
    assert lib.b2g_linear(None, None, None) == 1


def test_block_shapes():
    assert block_shapes(b2g.FMT_NVFP4, 3, 33) == ((3, 32), (3, 4))
    assert block_shapes(b2g.FMT_MXF4, 0, 32) == ((0, 16), (0, 1))
    assert block_shapes(b2g.FMT_MXF8, 5, 1) == ((5, 32), (5, 1))
    with pytest.raises(b2g.B2GError) as e:
        block_shapes(b2g.FMT_BF16, 1, 1)
    assert e.value.status == 4


def test_tensors_that_do_not_fit_are_refused_before_a_launch():
    import torch

    ops = LinearOps()  # no handle: a call that got as far as the library would fail otherwise
    ops.device = 0
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for bad in (dict(x=x.to(torch.int32)), dict(x=x[0]), dict(x=x)):  # type, rank, device
        with pytest.raises(b2g.B2GError) as e:
            ops.quantize_block(b2g.FMT_NVFP4, **bad)
        assert e.value.status == 1


def _bf16_values():
    bits = np.arange(1 << 15, dtype=np.uint32) << 16
    v = bits.view(np.float32)
    return v[np.isfinite(v)]


def _f16_values():
    v = np.arange(1 << 15, dtype=np.uint16).view(np.float16).astype(np.float32)
    return v[np.isfinite(v)]


@pytest.mark.parametrize("values", [_bf16_values, _f16_values])
def test_the_short_quotient_crosses_no_boundary(values):
    # e2m1(x / s) through fma(x, 1/s, 48) - 48, for every 16-bit x and every ue4m3 s, over the
    # magnitudes where the code is not 0 or saturated anyway.  x * (1/s) is exact in 64 bits
    # (11 + 24 bits), so the sum below rounds once, as the fma does.
    x = values()
    for s in ref.E4M3[1:].astype(np.float32):
        inv = np.float32(1.0) / s
        # beside the range the quotient is far from any boundary; keep a margin around it
        xs = x[(x > 0.2 * s) & (x < 8 * s)]
        snap = (xs.astype(np.float64) * np.float64(inv) + 48.0).astype(np.float32) - np.float32(48.0)
        exact = xs.astype(np.float64) / np.float64(s)
        got, want = ref.nearest(np.minimum(snap, 6.0), ref.E2M1), ref.nearest(np.minimum(exact, 6), ref.E2M1)
        assert np.array_equal(got, want), float(s)


def test_the_gradient_formula_agrees_with_differences():
    rng = np.random.default_rng(3)
    rows, cols, per = 5, 12, 2
    p = {"x": rng.normal(size=(rows, cols)), "y": rng.normal(size=(rows, cols)),
         "gate": rng.normal(size=(3, cols)), "w_post": 1 + 0.3 * rng.normal(size=cols),
         "w_pre": 1 + 0.3 * rng.normal(size=cols)}
    cv, ch = rng.normal(size=(rows, cols)), rng.normal(size=(rows, cols))
    kw = dict(eps=1e-3, alpha=0.9, beta=0.6, per=per)

    def loss(q):
        v, h, _, _ = ref.norm_forward(**q, **kw)
        return (cv * v).sum() + (ch * h).sum()

    v, _, r1, r2 = ref.norm_forward(**p, **kw)
    got = ref.norm_backward(ch, cv, v, r2, p["w_pre"], p["y"], r1, p["w_post"], p["gate"], per,
                            alpha=0.9, beta=0.6)
    for name, key in (("x", "dx"), ("y", "dy"), ("gate", "dgate"), ("w_post", "dw_post"),
                      ("w_pre", "dw_pre")):
        for at in itertools.islice(np.ndindex(*p[name].shape), 0, None, 3):
            q = {k: a.copy() for k, a in p.items()}
            e = 1e-5
            q[name][at] += e
            hi = loss(q)
            q[name][at] -= 2 * e
            # central difference: error e^2 times the third derivative, and 2^-53 / e
            assert abs((hi - loss(q)) / (2 * e) - got[key][at]) < 1e-7, (name, at)


def test_differences_without_a_norm_or_gate():
    rng = np.random.default_rng(4)
    x, y, c = (rng.normal(size=(3, 5)) for _ in range(3))
    got = ref.norm_backward(None, c, None, None, None, y=y, alpha=0.5, beta=2.0)
    assert np.allclose(got["dx"], 0.5 * c) and np.allclose(got["dy"], 2 * c)
    assert "dgate" not in got and "dw_pre" not in got
    assert np.allclose(ref.norm_forward(x, y, alpha=0.5, beta=2.0)[0], 0.5 * x + 2 * y)
