"""The handle's workspaces behind the operators around a linear layer: the first call of a
handle on a side stream."""
import numpy as np
import pytest
import torch

import b2g
from test_linear_ops_gpu import FMT, dev, random_weights

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh():
    eng = b2g.Engine(0)
    yield eng
    torch.cuda.synchronize()
    eng.close()


def few(engine, T, N, K, seed, fmt="mxf4"):
    """A call's operands and its result by the shared engine."""
    codes, sf, _ = random_weights(fmt, N, K, seed)
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda()
    x = dev(np.random.default_rng(seed).normal(size=(T, K)) / 64, torch.bfloat16)
    want = torch.empty(T, N, dtype=torch.bfloat16, device="cuda")
    engine.linear(x, c, s, want, FMT[fmt])
    return (x, c, s, torch.empty_like(want), FMT[fmt]), want


@pytest.mark.parametrize("T", [2, 24])
def test_the_first_call_is_on_a_side_stream_of_a_busy_device(engine, fresh, T):
    # K is cut among CTAs, whose arrivals are counted from zero
    args, want = few(engine, T, 300, 16384, 80)
    a = torch.randn(8192, 8192, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(8):
        a = a @ a * 1e-2
    for _ in range(3):
        fresh.linear(*args, stream=side)
    side.synchronize()
    assert torch.equal(args[3], want)
