"""One training step of a layer with experts, and one of its decode, on an MI355X.

    python examples/expert_layer.py [--tokens 2048] [--experts 8] [--hidden 1024] [--inner 2048]

Forward: tokens go to their expert (sorted by expert, the row offsets stay on the device), through an up
projection with its activation and a down projection onto the residual stream.  Backward: the
gradients of both experts' weights and of the input.  Update: the weights' gradients, brought near orthogonal
matrices by Newton-Schulz steps, are subtracted.  Decode: one token through the same experts.
Each stage prints its time, and how far the forward pass is from plain torch operations in fp32.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import rocm_wmma_gemm_amd as R  # noqa: E402


class ExpertLayer:
    """x + W2[e] silu(W1[e] x + b1[e]) for the rows of every expert e."""

    def __init__(self, experts, hidden, inner, dtype=torch.bfloat16, device="cuda"):
        self.E, self.H, self.I = experts, hidden, inner
        new = lambda *s: torch.randn(s, device=device, dtype=torch.float32)  # noqa: E731
        self.w1 = (new(experts, inner, hidden) / hidden ** 0.5).to(dtype)  # stored out x in
        self.w2 = (new(experts, hidden, inner) / inner ** 0.5).to(dtype)
        self.b1 = (0.1 * new(experts, inner)).to(dtype)
        self.loader = R.Loader()

    @staticmethod
    def dispatch(choice, experts):
        """Rows sorted by expert: (order, offsets).  Nothing leaves the device."""
        order = torch.argsort(choice, stable=True)
        counts = torch.zeros(experts, dtype=torch.int32, device=choice.device)
        counts.scatter_add_(0, choice, torch.ones_like(choice, dtype=torch.int32))
        offsets = torch.zeros(experts + 1, dtype=torch.int32, device=choice.device)
        offsets[1:] = counts.cumsum(0)
        return order, offsets

    def forward(self, x, offsets):
        T = x.shape[0]
        z, h, y = (torch.empty((T, n), dtype=x.dtype, device=x.device) for n in (self.I, self.I, self.H))
        self.loader.grouped(h, x, self.w1, offsets, T, self.I, self.H, bias=self.b1, preact=z,
                            activation=R.activation.silu)
        self.loader.grouped(y, h, self.w2, offsets, T, self.H, self.I, residual=x)
        return y, (x, z, h)

    def backward(self, dy, kept, offsets):
        x, z, h = kept
        T = x.shape[0]
        dh, dx = torch.empty_like(h), torch.empty_like(x)
        dw1, dw2, db1 = torch.empty_like(self.w1), torch.empty_like(self.w2), torch.empty_like(self.b1)
        self.loader.grouped_backward(dh, dw2, None, dy, h, self.w2, offsets, T, self.H, self.I)
        self.loader.grouped_backward(dx, dw1, db1, dh, x, self.w1, offsets, T, self.I, self.H, preact=z,
                                     activation=R.activation.silu)
        return dx + dy, dw1, dw2, db1

    def update(self, dw1, dw2, db1, rate=0.02):
        for w, dw in ((self.w1, dw1), (self.w2, dw2)):
            step = torch.empty_like(dw)
            self.loader.orthogonalize(step, dw, w.shape[1], w.shape[2], self.E)
            w.add_(step, alpha=-rate)
        self.b1.add_(db1, alpha=-rate)

    def plain(self, x, offsets):
        y, ends = x.float().clone(), offsets.tolist()
        for e in range(self.E):
            at = slice(ends[e], ends[e + 1])
            z = x[at].float() @ self.w1[e].float().t() + self.b1[e].float()
            y[at] += (z * torch.sigmoid(z)) @ self.w2[e].float().t()
        return y


def timed(name, f, *args):
    f(*args)
    torch.cuda.synchronize()
    start = time.perf_counter()
    out = f(*args)
    torch.cuda.synchronize()
    print(f"{name:10s} {(time.perf_counter() - start) * 1e6:9.1f} us")
    return out


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("tokens", 2048), ("experts", 8), ("hidden", 1024), ("inner", 2048)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    torch.manual_seed(0)
    layer = ExpertLayer(a.experts, a.hidden, a.inner)
    x = torch.randn((a.tokens, a.hidden), device="cuda").to(torch.bfloat16)
    order, offsets = layer.dispatch(torch.randint(a.experts, (a.tokens,), device="cuda"), a.experts)
    x = x[order].contiguous()

    y, kept = timed("forward", layer.forward, x, offsets)
    off = (y.float() - layer.plain(x, offsets)).norm() / y.float().norm()
    print(f"forward against plain operations in fp32: relative difference {off.item():.2e}")
    dy = y / y.numel()  # the gradient of half the mean square
    grads = timed("backward", layer.backward, dy, kept, offsets)
    timed("update", layer.update, *grads[1:])
    after = layer.forward(x, offsets)[0].float().square().mean()
    print(f"mean square of the output: {y.float().square().mean().item():.4f} -> {after.item():.4f}")

    token = x[:1].contiguous()
    _, one = layer.dispatch(torch.randint(a.experts, (1,), device="cuda"), a.experts)
    timed("decode", layer.forward, token, one)
    assert off < 1e-2, off


if __name__ == "__main__":
    main()
