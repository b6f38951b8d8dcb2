"""One training step of a model with experts, from its router to its loss, and one of its decode, on an MI355X.

    python examples/expert_model.py [--tokens 1000] [--experts 16] [--choices 4] [--hidden 512] [--inner 768] [--vocabulary 8003]

Forward: the router's logits choose the experts of every token, the tokens' rows go to them sorted by expert, through an up
projection with its activation and a down projection, and come back as a weighted sum onto the residual stream; a projection
onto the vocabulary ends in the cross entropy against every token's target, without its logits being kept.  Backward: the
gradients of all of it, the router's through the weights of the experts it chose.  Nothing travels to the host.
Each stage prints its time, and every gradient how far it is from the same model in fp64.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import rocm_wmma_gemm_amd as R  # noqa: E402

HOW = dict(score=R.score.sigmoid, renormalize=True, scale=1.5)


class ExpertModel:
    """loss(head(x + sum_j w_j W2[e_j] silu(W1[e_j] x))), (e_j, w_j) = route(router x)."""

    def __init__(self, experts, choices, hidden, inner, vocabulary, dtype=torch.bfloat16, seed=0):
        self.E, self.k, self.H, self.I, self.V, self.dtype = experts, choices, hidden, inner, vocabulary, dtype
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        new = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
        self.router = (new(experts, hidden) / hidden ** 0.5).to(dtype)
        self.w1 = (new(experts, inner, hidden) / hidden ** 0.5).to(dtype)  # stored out x in
        self.w2 = (new(experts, hidden, inner) / inner ** 0.5).to(dtype)
        self.head = (new(vocabulary, hidden) * 2 / hidden ** 0.5).to(dtype)
        self.balance = 0.1 * new(experts)
        self.loader = R.Loader()

    def _empty(self, *shape, dtype=None):
        return torch.empty(shape, dtype=dtype or self.dtype, device="cuda")

    def experts(self, x, real=None):
        """The layer: its output, and what its backward pass needs.  real: tokens that are no padding."""
        L, T, S, i32, f32 = self.loader, x.shape[0], x.shape[0] * self.k, torch.int32, torch.float32
        logits, chosen, weights = self._empty(T, self.E, dtype=f32), self._empty(T, self.k, dtype=i32), self._empty(T, self.k, dtype=f32)
        L.linear(logits, x, self.router, T, self.E, self.H)
        L.route(chosen, weights, logits, T, self.E, self.k, bias=self.balance, mask=real, **HOW)
        offsets, places = self._empty(self.E + 1, dtype=i32), self._empty(T, self.k, dtype=i32)
        rows, z, h, y = self._empty(S, self.H), self._empty(S, self.I), self._empty(S, self.I), self._empty(S, self.H)
        L.dispatch(rows, offsets, places, x, chosen, T, self.H, self.k)
        L.grouped(h, rows, self.w1, offsets, S, self.I, self.H, preact=z, activation=R.activation.silu)
        L.grouped(y, h, self.w2, offsets, S, self.H, self.I)
        out = self._empty(T, self.H)
        L.combine(out, y, places, T, self.H, self.k, weights=weights, residual=x)
        return out, (x, logits, chosen, weights, offsets, places, rows, z, h, y)

    def loss(self, out, targets):
        T = out.shape[0]
        loss, lse = self._empty(T, dtype=torch.float32), self._empty(T, dtype=torch.float32)
        self.loader.linear_cross_entropy(loss, lse, out, self.head, targets, T, self.V, self.H)
        return loss, lse

    def backward(self, dloss, lse, out, targets, kept):
        """The gradients of the states, the router, both weights of the experts and the head."""
        L = self.loader
        x, logits, chosen, weights, offsets, places, rows, z, h, y = kept
        T, S = x.shape[0], rows.shape[0]
        dout, dhead = self._empty(T, self.H), torch.empty_like(self.head)
        L.linear_cross_entropy_backward(dout, dhead, dloss, lse, out, self.head, targets, T, self.V, self.H)
        dy, dweights = torch.empty_like(y), torch.empty_like(weights)
        L.combine_backward(dy, dweights, dout, y, places, T, self.H, self.k, weights=weights)
        dh, drows, dw1, dw2 = torch.empty_like(h), torch.empty_like(rows), torch.empty_like(self.w1), torch.empty_like(self.w2)
        L.grouped_backward(dh, dw2, None, dy, h, self.w2, offsets, S, self.H, self.I)
        L.grouped_backward(drows, dw1, None, dh, rows, self.w1, offsets, S, self.I, self.H, preact=z, activation=R.activation.silu)
        dx, dlogits = self._empty(T, self.H), torch.empty_like(logits)
        L.combine(dx, drows, places, T, self.H, self.k, residual=dout)  # of the dispatch, and of the residual stream
        L.route_backward(dlogits, dweights, chosen, logits, T, self.E, self.k, **HOW)
        by_router, drouter = self._empty(T, self.H), torch.empty_like(self.router)
        L.linear_backward(by_router, drouter, None, dlogits.to(self.dtype), x, self.router, T, self.E, self.H)
        return {"states": dx + by_router, "router": drouter, "up": dw1, "down": dw2, "head": dhead}

    def exact(self, x, targets, chosen, real=None):
        """Loss by token and gradients of the mean over the tokens with a target, in fp64 by differentiation of plain operations,
        for the experts that were chosen."""
        leaves = {n: v.double().requires_grad_(True) for n, v in
                  (("states", x), ("router", self.router), ("up", self.w1), ("down", self.w2), ("head", self.head))}
        s = leaves["states"]
        at = chosen.clamp_min(0).long()
        score = torch.sigmoid(s @ leaves["router"].t()).gather(1, at)
        w = HOW["scale"] * score / score.sum(1, keepdim=True) * (chosen >= 0)
        out = s
        for j in range(self.k):
            for e in range(self.E):
                t = ((at[:, j] == e) & (chosen[:, j] >= 0)).nonzero()[:, 0]
                zz = s[t] @ leaves["up"][e].t()
                out = out.index_add(0, t, w[t, j:j + 1] * ((zz * torch.sigmoid(zz)) @ leaves["down"][e].t()))
        log_p = torch.log_softmax(out @ leaves["head"].t(), 1)
        counts = targets >= 0
        loss = -log_p.gather(1, targets.clamp_min(0)[:, None])[:, 0] * counts
        (loss.sum() / counts.sum()).backward()
        return loss.detach(), {n: v.grad for n, v in leaves.items()}


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
    for name, value in (("tokens", 1000), ("experts", 16), ("choices", 4), ("hidden", 512), ("inner", 768), ("vocabulary", 8003)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    model = ExpertModel(a.experts, a.choices, a.hidden, a.inner, a.vocabulary)
    torch.manual_seed(1)
    x = torch.randn((a.tokens, a.hidden), device="cuda").to(torch.bfloat16)
    real = torch.arange(a.tokens, device="cuda") < a.tokens - a.tokens // 8  # the batch's end is padding
    targets = torch.where(real, torch.randint(a.vocabulary, (a.tokens,), device="cuda"), -100)

    out, kept = timed("experts", model.experts, x, real)
    loss, lse = timed("loss", model.loss, out, targets)
    dloss = real.float() / real.sum()
    grads = timed("backward", model.backward, dloss, lse, out, targets, kept)
    want_loss, want = model.exact(x, targets, kept[2], real)
    worst = 0.0
    for name, got, right in [("loss", loss, want_loss)] + [(n, grads[n], want[n]) for n in grads]:
        off = ((got.double() - right).norm() / right.norm()).item()
        worst = max(worst, off)
        print(f"{name:10s} relative difference from fp64 {off:.2e}")
    timed("decode", model.experts, x[:1].contiguous())
    # a state passes some eight roundings to bf16 (2^-9 of a norm each) on its way to a gradient
    assert worst < 8 * 2.0 ** -9 * 2, worst


if __name__ == "__main__":
    main()
