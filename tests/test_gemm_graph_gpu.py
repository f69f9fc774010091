"""b2g_gemm in captured graphs: the handle's workspaces while a graph holds them."""
import pytest
import torch

import b2g

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh():
    eng = b2g.Engine(0)
    yield eng
    torch.cuda.synchronize()
    eng.close()


def captured(f):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    return graph


def block_scaled(engine, M, N, K, seed):
    """Operands and result buffer of an NVFP4 product."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ops = []
    for rows in (M, N):
        x = torch.randn(rows, K, generator=g, device="cuda")
        q = [torch.empty(s, dtype=torch.uint8, device="cuda") for s in b2g.block_shapes(b2g.FMT_NVFP4, rows, K)]
        engine.quantize_block(b2g.FMT_NVFP4, x, *q)
        ops.append(q)
    return ops, torch.empty(M, N, dtype=torch.bfloat16, device="cuda")


def multiply(eng, ops, out):
    (a, sa), (b, sb) = ops
    return eng.gemm(a, b, out, b2g.FMT_NVFP4, sfa=sa, sfb=sb)


def test_graphs_outlive_the_growth_of_the_workspaces(engine, fresh):
    # scales in the engine's layout, and the split tail's partial tiles
    cases = [block_scaled(engine, *size, seed) for seed, size in
             enumerate([(130, 256, 512), (500, 1024, 2048), (1024, 1024, 8192)])]
    wants = [multiply(engine, ops, torch.empty_like(out)) for ops, out in cases]
    graphs = [captured(lambda: multiply(fresh, *c)) for c in cases]
    more = block_scaled(engine, 2500, 2048, 16384, 9)
    multiply(fresh, *more)  # an eager call that needs more
    rubbish = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for n in [1 << 16, 1 << 20, 1 << 21] * 8]
    for g, (_, out), want in zip(graphs, cases, wants):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all((r == 0xFF).all() for r in rubbish)
    fresh.check()


@pytest.mark.parametrize("M,N,K", [(500, 1024, 2048), (512, 512, 8192), (2500, 2048, 2048)])
def test_replays_of_a_split_tail_use_their_own_partial_sums(engine, fresh, M, N, K):
    # every replay has other inputs: sums that the last one left would show
    assert b2g.plan_gemm(b2g.FMT_BF16, M, N, K)["tail_split"] > 1
    a, b = (torch.empty(r, K, dtype=torch.bfloat16, device="cuda") for r in (M, N))
    out, want = (torch.empty(M, N, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    graph = captured(lambda: [fresh.gemm(a, b, out, b2g.FMT_BF16) for _ in range(2)])
    g = torch.Generator(device="cuda").manual_seed(11)
    for _ in range(6):
        for t in (a, b):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        engine.gemm(a, b, want, b2g.FMT_BF16)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        fresh.gemm(a, b, out, b2g.FMT_BF16)
        assert torch.equal(out, want)
    fresh.check()
