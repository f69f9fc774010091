"""The handle's workspaces behind the operators around a linear layer: the first call of a
handle on a side stream, growth under captured graphs."""
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


def captured(f):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    return graph


def test_graphs_outlive_the_growth_of_the_workspace(engine, fresh):
    # 128 row tiles leave no SMs to cut K, 16 do: the smaller product needs the larger workspace,
    # and counters, for the first time within its capture
    large, want_large = few(engine, 16, 16384, 8192, 81)
    small, want_small = few(engine, 16, 2048, 8192, 82)
    one, want_one = few(engine, 1, 300, 16384, 83)
    fresh.linear(*large)
    assert torch.equal(large[3], want_large)
    graphs = [captured(lambda: fresh.linear(*a)) for a in (small, one, large)]
    # an eager call that needs more than all of them, and buffers where freed ones would have been
    more, want_more = few(engine, 128, 2048, 8192, 84)
    fresh.linear(*more)
    assert torch.equal(more[3], want_more)
    rubbish = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for n in [1 << 16, 1 << 20, 1 << 21] * 8]
    for _ in range(2):
        for g, (args, want) in zip(graphs, ((small, want_small), (one, want_one), (large, want_large))):
            args[3].zero_()
            g.replay()
            fresh.linear(*more)
            torch.cuda.synchronize()
            assert torch.equal(args[3], want) and torch.equal(more[3], want_more)
    assert all((r == 0xFF).all() for r in rubbish)
    fresh.check()


@pytest.mark.parametrize("rows,cols", [(40, 1024), (64, 9000)])
def test_gradient_in_graphs_before_any_call(engine, fresh, rows, cols):
    rng = np.random.default_rng(85)
    dh, v = (dev(rng.normal(size=(rows, cols)), torch.float32) for _ in range(2))
    w, r2 = torch.ones(cols, device="cuda"), torch.ones(rows, device="cuda")

    def grad(eng, n):
        out = torch.zeros(n, cols, device="cuda"), torch.zeros(cols, device="cuda")
        return out, lambda: eng.residual_norm_backward(dh[:n], v[:n], r2[:n], w, out[0], dw_pre=out[1])

    few_rows, all_rows = grad(fresh, rows // 4), grad(fresh, rows)
    graphs = [captured(f) for _, f in (few_rows, all_rows)]
    for g in graphs * 2:
        g.replay()
    torch.cuda.synchronize()
    for (out, _), n in ((few_rows, rows // 4), (all_rows, rows)):
        want, call = grad(engine, n)
        call()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
