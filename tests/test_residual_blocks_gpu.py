"""The example that trains and decodes a stack of residual blocks with the operators around a
linear layer (microbench-blackwell_b200/examples/residual_blocks.py)."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import linear_ops_ref as ref

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "microbench-blackwell_b200", "examples",
                    "residual_blocks.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("residual_blocks", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def norm(a, w):
    return a / np.sqrt((a * a).mean(1, keepdims=True) + 1e-6) * w


@pytest.mark.parametrize("fmt", ["nvfp4", "mxf4", "mxf8"])
def test_stack_learns_and_decodes(engine, example, fmt):
    tokens, width, blocks = 90, 160, 3
    net = example.Stack(engine, example.FORMATS[fmt], tokens=tokens, width=width, blocks=blocks, sequences=3)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(tokens, width, generator=g).bfloat16().cuda()
    target = (x.float() + x.float().roll(1, 1)).bfloat16()
    losses = [net.step(x, target, 0.02) for _ in range(15)]
    engine.check()
    assert np.isfinite(losses).all() and losses[-1] < 0.7 * losses[0]
    # few tokens through the same codes, against 64 bits with the codes' values: each block rounds
    # three times to bf16 and passes an error of its input on with a gain of at most two
    for T in (1, 5, 11):
        got = net.decode(x[30:30 + T].contiguous(), sequence=1).double().cpu().numpy()
        v = x[30:30 + T].double().cpu().numpy()
        for b in net.blocks:
            w = ref.values(b.wq.codes.cpu().numpy(), b.wq.sf.cpu().numpy(), fmt)[:, :width]
            p = {k: getattr(b, k).double().cpu().numpy() for k in ("gate", "w_pre", "w_post")}
            v = v + p["gate"][1] * norm(norm(v, p["w_pre"]) @ w.T, p["w_post"])
        bound = sum(3 * 2.0 ** -8 * 2 ** i for i in range(blocks))
        assert np.linalg.norm(got - v) <= bound * np.linalg.norm(v)
    with pytest.raises(ValueError):
        example.Stack(engine, example.FORMATS[fmt], tokens=10, width=32, blocks=1, sequences=3)


def test_stack_gradient_against_differences(engine, example):
    # along one direction of each parameter that stays in bf16, MXFP8 operands: the products' casts
    # have 4 significant bits, 2^-5 of an element at most and random in sign, so the derivative is
    # right to a few percent; the differences are taken in 64 bits of the same function
    tokens, width, blocks = 64, 96, 2
    net = example.Stack(engine, example.FORMATS["mxf8"], tokens=tokens, width=width, blocks=blocks)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(tokens, width, generator=g).bfloat16().cuda()
    c = torch.randn(tokens, width, generator=g).bfloat16().cuda()
    net.forward(x)
    net.backward(c, 1.0, False)
    engine.check()
    params = [{k: getattr(b, k).double().cpu().numpy() for k in ("w", "gate", "w_pre", "w_post")}
              for b in net.blocks]
    v0, c0 = x.double().cpu().numpy(), c.double().cpu().numpy()

    def loss():
        v = v0
        for p in params:
            v = v + p["gate"] * norm(norm(v, p["w_pre"]) @ p["w"].T, p["w_post"])
        return (c0 * v).sum()

    names = {"w": "dw", "gate": "dgate", "w_pre": "dw_pre", "w_post": "dw_post"}
    for i, b in enumerate(net.blocks):
        for key, grad in names.items():
            got = getattr(b, grad).double().cpu().numpy().reshape(params[i][key].shape)
            step = 1e-4 * got / np.linalg.norm(got)
            keep = params[i][key]
            params[i][key] = keep + step
            hi = loss()
            params[i][key] = keep - step
            lo = loss()
            params[i][key] = keep
            # the derivative along its own direction is its length
            assert abs((hi - lo) / 2e-4 / np.linalg.norm(got) - 1) < 0.06, (i, key)
