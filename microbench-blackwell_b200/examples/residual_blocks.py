"""A stack of residual blocks with microscaled weights, trained and then decoded.

Each block is  x <- x + gate * norm(W . norm(x) * w_pre) * w_post  with one gate row per
sequence.  Training keeps bf16 weights and casts every operand of its three products
(Engine.quantize_block, along both dimensions in one pass); the norms, gate, residual
addition and the cast of the next product's input are one pass (Engine.residual_norm), as
is their gradient (Engine.residual_norm_backward).  Decoding feeds a few tokens through the
same weights' codes (Engine.linear), without casting the activations.

    python microbench-blackwell_b200/examples/residual_blocks.py --format mxf8
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import torch  # noqa: E402

import b2g  # noqa: E402

FORMATS = {"nvfp4": b2g.FMT_NVFP4, "mxf4": b2g.FMT_MXF4, "mxf8": b2g.FMT_MXF8}


class Cast:
    """Codes and scales of a matrix, along its rows and its columns."""

    def __init__(self, eng, fmt, rows, cols, device):
        self.eng, self.fmt = eng, fmt
        u8 = dict(dtype=torch.uint8, device=device)
        (a, b), (c, d) = b2g.block_shapes(fmt, rows, cols), b2g.block_shapes(fmt, cols, rows)
        self.codes, self.sf = torch.empty(a, **u8), torch.empty(b, **u8)
        self.codes_t, self.sf_t = torch.empty(c, **u8), torch.empty(d, **u8)

    def __call__(self, x, scale=1.0, rand=None):
        self.eng.quantize_block(self.fmt, x, self.codes, self.sf, codes_t=self.codes_t, sf_t=self.sf_t,
                                scale=scale, rand=rand)
        return self


class Block:
    """Parameters of one block, what its backward pass needs, and its gradients."""

    def __init__(self, eng, fmt, tokens, width, sequences, device, generator):
        bf16, f32 = (dict(dtype=t, device=device) for t in (torch.bfloat16, torch.float32))
        self.eng, self.fmt = eng, fmt
        self.w = (torch.randn(width, width, generator=generator) / width ** 0.5).to(**bf16)
        self.gate = torch.full((sequences, width), 0.5, **bf16)
        self.w_pre, self.w_post = torch.ones(width, **bf16), torch.ones(width, **bf16)
        self.wq = Cast(eng, fmt, width, width, device)(self.w)
        self.hq, self.dyq = (Cast(eng, fmt, tokens, width, device) for _ in range(2))
        self.h, self.y, self.x_out, self.dh, self.dy, self.dx = (
            torch.empty(tokens, width, **bf16) for _ in range(6))
        self.dw = torch.empty(width, width, **bf16)
        self.dgate = torch.empty(sequences, width, **f32)
        self.dw_pre, self.dw_post = (torch.empty(width, **f32) for _ in range(2))
        self.rstd_pre, self.rstd_post = (torch.empty(tokens, **f32) for _ in range(2))

    def product(self):
        """y = W . h, both cast."""
        self.hq(self.h)
        self.eng.gemm(self.hq.codes, self.wq.codes, self.y, self.fmt, sfa=self.hq.sf, sfb=self.wq.sf)

    def product_backward(self, scale, rand):
        """dh and dw of dy, which is cast once for both; `scale` keeps it in the format's range."""
        q = self.dyq(self.dy, scale, rand)
        self.eng.gemm(q.codes, self.wq.codes_t, self.dh, self.fmt, sfa=q.sf, sfb=self.wq.sf_t, alpha=1 / scale)
        self.eng.gemm(q.codes_t, self.hq.codes_t, self.dw, self.fmt, sfa=q.sf_t, sfb=self.hq.sf_t,
                      alpha=1 / scale)

    def update(self, rate):
        for p, g in ((self.w, self.dw), (self.gate, self.dgate), (self.w_pre, self.dw_pre),
                     (self.w_post, self.dw_post)):
            p.copy_(p.float() - rate * g.float())
        self.wq(self.w)


class Stack:
    def __init__(self, eng, fmt, *, tokens, width, blocks, sequences=1, device="cuda:0", seed=0):
        if tokens % sequences:
            raise ValueError("tokens must be a multiple of sequences")
        g = torch.Generator().manual_seed(seed)
        self.eng, self.fmt, self.tokens, self.width = eng, fmt, tokens, width
        self.per = tokens // sequences
        self.blocks = [Block(eng, fmt, tokens, width, sequences, device, g) for _ in range(blocks)]
        self.ones = torch.ones(width, dtype=torch.bfloat16, device=device)
        self.rand = torch.empty(tokens, width, dtype=torch.uint8, device=device)

    def forward(self, x):
        """x (tokens x width, bf16) through the blocks; the last one's output."""
        first = self.blocks[0]
        self.eng.residual_norm(x, w_pre=first.w_pre, h=first.h, rstd_pre=first.rstd_pre)
        first.x_in = x
        for i, b in enumerate(self.blocks):
            b.product()
            after = self.blocks[i + 1] if i + 1 < len(self.blocks) else None
            # the end of this block and the norm before the next in one pass
            self.eng.residual_norm(b.x_in, y=b.y, gate=b.gate, rows_per_gate=self.per, w_post=b.w_post,
                                   w_pre=after.w_pre if after else self.ones, x_out=b.x_out,
                                   h=after.h if after else None, rstd_post=b.rstd_post,
                                   rstd_pre=after.rstd_pre if after else None)
            if after:
                after.x_in = b.x_out
        return self.blocks[-1].x_out

    def backward(self, dx_out, scale, stochastic):
        """Gradients of every parameter from the output's."""
        dh = None
        for i in reversed(range(len(self.blocks))):
            b = self.blocks[i]
            after = self.blocks[i + 1] if i + 1 < len(self.blocks) else None
            self.eng.residual_norm_backward(
                dh, b.x_out if after else None, after.rstd_pre if after else None,
                after.w_pre if after else None, b.dx, dx_out=dx_out, y=b.y, rstd_post=b.rstd_post,
                w_post=b.w_post, gate=b.gate, rows_per_gate=self.per, dy=b.dy, dgate=b.dgate,
                dw_post=b.dw_post, dw_pre=after.dw_pre if after else None)
            rand = self.rand.random_(0, 256) if stochastic else None
            b.product_backward(scale, rand)
            dx_out, dh = b.dx, b.dh
        first = self.blocks[0]
        self.eng.residual_norm_backward(dh, first.x_in, first.rstd_pre, first.w_pre, None, dx_out=dx_out,
                                        dw_pre=first.dw_pre)

    def step(self, x, target, rate, scale=2.0 ** 12, stochastic=True):
        """One step of gradient descent on the squared distance (sum over the columns, mean
        over the tokens); the mean over the elements, before the step."""
        diff = self.forward(x).float() - target.float()
        self.backward((diff * (2 / self.tokens)).bfloat16(), scale, stochastic)
        for b in self.blocks:
            b.update(rate)
        return float((diff * diff).mean())

    def decode(self, x, sequence=0):
        """A few tokens of one sequence (T x width, bf16) through the same weights."""
        h, y = torch.empty_like(x), torch.empty_like(x)
        self.eng.residual_norm(x, w_pre=self.blocks[0].w_pre, h=h)
        x = x.clone()
        for i, b in enumerate(self.blocks):
            self.eng.linear(h, b.wq.codes, b.wq.sf, y, self.fmt)
            last = i + 1 == len(self.blocks)
            self.eng.residual_norm(x, y=y, gate=b.gate[sequence:sequence + 1], rows_per_gate=len(x),
                                   w_post=b.w_post, w_pre=self.ones if last else self.blocks[i + 1].w_pre,
                                   x_out=x, h=None if last else h)
        return x


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--format", choices=list(FORMATS), default="mxf8")
    p.add_argument("--tokens", type=int, default=2048)
    p.add_argument("--width", type=int, default=1024)
    p.add_argument("--blocks", type=int, default=4)
    p.add_argument("--sequences", type=int, default=4)
    p.add_argument("--steps", type=int, default=40)
    p.add_argument("--rate", type=float, default=0.02)
    o = p.parse_args(argv)
    eng = b2g.Engine(0)
    net = Stack(eng, FORMATS[o.format], tokens=o.tokens, width=o.width, blocks=o.blocks, sequences=o.sequences)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(o.tokens, o.width, generator=g).bfloat16().cuda()
    # something the stack can learn: a fixed mixing of the columns
    target = (x.float() + x.float().roll(1, 1)).bfloat16()
    for i in range(o.steps):
        loss = net.step(x, target, o.rate)
        if i % 10 == 0 or i + 1 == o.steps:
            print(f"step {i}: loss {loss:.4f}")
    eng.check()
    few = net.decode(x[:4].contiguous())
    far = (few.float() - net.forward(x)[:4].float()).norm() / few.float().norm()
    print(f"four tokens decoded; {100 * float(far):.2f} % from the pass with cast activations")
    eng.close()


if __name__ == "__main__":
    main()
