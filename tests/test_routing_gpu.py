"""From a router's logits to rows sorted by expert and back, on the GPU, against the definitions in 64 bits.

What is chosen, and where rows go, has to be equal.  Numbers have bounds, element by element: weights are worked out in
64 bits and rounded once; a gradient of the logits is worked out in fp32, where a score is off by |x - top| + 48
roundings of 2^-24 (the argument of the exponential, the exponential, a sum of 36 additions, a division) and what is made of
scores by a few of those; a sum over k rows takes k + 2 roundings, a product of rows one for each of its elements.
"""
import math

import pytest
import torch

import rocm_wmma_gemm_amd as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
LEAST = {F16: 2.0 ** -25, BF16: 2.0 ** -133, F32: 2.0 ** -149}
E32 = 2.0 ** -24
SOFTMAX, SIGMOID = R.score.softmax, R.score.sigmoid


@pytest.fixture(scope="module")
def loader():
    return R.Loader()


def _id(v):
    return str(v).replace("torch.", "").replace("score.", "")


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=F32) * scale).to(dtype)


def odd_start(t):
    """The same values one element further on in memory."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    over = (got.double() - want).abs() - tol
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3g} over its bound at {int(over.argmax())}"


def scores64(x, score):
    x = x.double()
    if score == SIGMOID:
        return 1 / (1 + torch.exp(-x))
    top = x.max(1, keepdim=True)[0]
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def choice64(x, k, score, bias, groups, kept, best):
    """Expert by expert: the largest that is left, the first of equal ones."""
    M, E = x.shape
    s = scores64(x, score)
    value = s if bias is None else s + bias.double()
    rank = (x.double() if bias is None else value).clone()
    rank = torch.where(torch.isnan(rank), torch.full_like(rank, -1.7e308), rank).clamp(-1.7e308, 1.7e308)
    if groups > 1:
        each = E // groups
        of = torch.stack([v.sort(1, descending=True)[0][:, :best].sum(1) for v in value.split(each, 1)], 1)
        for t in range(M):
            order = sorted(range(groups), key=lambda g: (-of[t, g].item(), g))
            for g in order[kept:]:
                rank[t, g * each:(g + 1) * each] = -math.inf
    chosen = torch.empty((M, k), dtype=torch.int64, device=x.device)
    for j in range(k):
        top = rank.max(1, keepdim=True)[0]
        chosen[:, j] = torch.where(rank == top, torch.arange(E, device=x.device), E).min(1)[0]
        rank.scatter_(1, chosen[:, j:j + 1], -math.inf)
    return chosen, s


def weights64(s, chosen, renormalize, scale):
    w = s.gather(1, chosen)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / torch.where(total == 0, torch.ones_like(total), total))
    return w * scale


def routed(loader, x, k, **how):
    M, E = x.shape
    chosen = torch.full((M, k), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((M, k), math.nan, dtype=F32, device="cuda")
    loader.route(chosen, weights, x, M, E, k, **how)
    return chosen, weights


ROUTES = [  # M, E, k, groups, kept, best
    (1, 1, 1, 1, 1, 1), (1, 64, 2, 1, 1, 2), (3, 7, 7, 1, 1, 2), (17, 8, 2, 2, 1, 2), (33, 16, 4, 4, 2, 1), (65, 33, 5, 3, 2, 2),
    (100, 128, 8, 1, 1, 2), (257, 256, 8, 8, 4, 2), (50, 512, 32, 1, 1, 2), (19, 512, 17, 16, 16, 2), (21, 504, 16, 9, 5, 1),
    (40, 160, 6, 5, 3, 2), (16, 48, 3, 16, 3, 2), (9, 15, 3, 15, 15, 2), (1000, 60, 4, 1, 1, 2)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=_id)
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID], ids=_id)
@pytest.mark.parametrize("size", ROUTES, ids=_id)
def test_route_and_its_gradient(loader, size, score, dtype):
    M, E, k, groups, kept, best = size
    x, dw = rnd((M, E), dtype, 1, 2.0), rnd((M, k), F32, 2)
    for bias, renormalize, scale in ((None, True, 1.0), (rnd((E,), F32, 3, 0.05), True, 2.5), (None, False, 1.0),
                                     (rnd((E,), F32, 4, 0.3), False, 0.5)):
        how = dict(score=score, renormalize=renormalize, scale=scale)
        chosen, weights = routed(loader, x, k, bias=bias, groups=groups, kept_groups=kept, group_best=best, **how)
        want, s = choice64(x, k, score, bias, groups, kept, best)
        assert torch.equal(chosen.long(), want)
        w = weights64(s, want, renormalize, scale)
        within(weights, w, E32 * w.abs() * 1.001 + LEAST[F32], "weights")
        dx = torch.full((M, E), math.nan, dtype=dtype, device="cuda")
        loader.route_backward(dx, dw, chosen, x, M, E, k, **how)
        check_route_gradient(dx, dw, want, x, s, **how)


def check_route_gradient(dx, dw, chosen, x, s, score, renormalize, scale):
    dtype, p = x.dtype, s.gather(1, chosen)
    total = p.sum(1, keepdim=True) if renormalize else torch.ones_like(p[:, :1])
    total = torch.where(total == 0, torch.full_like(total, math.inf), total)
    ds, size = scale * dw.double() / total, scale * dw.double().abs() / total
    if renormalize:
        ds, size = ds - (ds * p).sum(1, keepdim=True) / total, size + (size * p).sum(1, keepdim=True) / total
    full, full_size = (torch.zeros_like(s).scatter_add_(1, chosen, v) for v in (ds, size))
    if score == SIGMOID:
        want, size = full * s * (1 - s), full_size * s * (1 - s)
    else:
        # (renormalised, sum_j s_j ds_j = scale sum_j s_j (dw_j - sum_i dw_i s_i / total) / total is 0 exactly: in 64 bits it
        # comes out as a rounding of 1e-17, which the logits that were not chosen would show)
        want = s * (full - (0 if renormalize else (full * s).sum(1, keepdim=True)))
        size = s * (full_size + (0 if renormalize else (full_size * s).sum(1, keepdim=True)))
    finite = torch.where(torch.isfinite(x), x.double(), torch.zeros_like(s))
    spread = (finite.abs().max(1, keepdim=True)[0] * 2 + 48) * 4
    within(dx, want, UNIT[dtype] * want.abs() + LEAST[dtype] + E32 * spread * size * 1.01 + 1e-37, "gradient of the logits")


def test_gradient_of_the_weights_against_differences(loader):
    """Steps of 2^-6 in fp32 logits: the difference of the weights, worked out in 64 bits, against the gradient."""
    M, E, k = 6, 12, 3
    x = rnd((M, E), F32, 5)
    dw = rnd((M, k), F32, 6)
    for score in (SOFTMAX, SIGMOID):
        for renormalize in (True, False):
            how = dict(score=score, renormalize=renormalize, scale=1.5)
            chosen, _ = routed(loader, x, k, **how)
            dx = torch.empty_like(x)
            loader.route_backward(dx, dw, chosen, x, M, E, k, **how)
            step = 2.0 ** -12
            for e in range(E):
                moved = []
                for sign in (1, -1):
                    y = x.double().clone()
                    y[:, e] += sign * step
                    moved.append((weights64(scores64(y, score), chosen.long(), renormalize, 1.5) * dw.double()).sum(1))
                want = (moved[0] - moved[1]) / (2 * step)
                # central differences of functions whose third derivatives are below 10: 10 step^2 / 6, and fp32's own
                assert (dx[:, e].double() - want).abs().max() < 10 * step * step * 3 * 4 + 1e-5


def test_route_ties_masks_and_extremes(loader):
    inf, nan = math.inf, math.nan
    x = torch.zeros((8, 20), device="cuda")
    x[1, 7:] = 1.0  # ties of two values
    x[2] = -inf  # nothing left
    x[3] = -inf
    x[3, 11] = 2.0  # one left
    x[4, 5] = nan
    x[5] = torch.finfo(F32).min
    x[6, 19], x[6, 18] = 100.0, 100.0
    x[7] = -0.0
    x[7, 3] = 0.0
    for score in (SOFTMAX, SIGMOID):
        for bias in (None, torch.zeros(20, device="cuda")):
            chosen, weights = routed(loader, x, 4, score=score, bias=bias)
            rows = [0, 1, 2, 3, 5, 6, 7]
            want, s = choice64(x, 4, score, bias, 1, 1, 2)
            assert torch.equal(chosen[rows].long(), want[rows]), (score, bias)
            w = weights64(s, want, True, 1.0)
            within(weights[rows], w[rows], E32 * w[rows].abs() * 1.001 + LEAST[F32], "weights")
            assert sorted(chosen[4].tolist()) == [0, 1, 2, 3]  # (no number: last)
            if score == SOFTMAX:
                assert (weights[2] == 0).all()
    dx = torch.full((8, 20), nan, device="cuda")
    chosen, weights = routed(loader, x, 4)
    loader.route_backward(dx, torch.ones((8, 4), device="cuda"), chosen, x, 8, 20, 4)
    assert (dx[2] == 0).all() and torch.isfinite(dx[[0, 1, 3, 5, 6, 7]]).all()
    # a padded batch: tokens that go nowhere
    for dtype in (torch.bool, torch.uint8):
        mask = torch.tensor([1, 0, 1, 0, 1, 1, 0, 1], device="cuda").to(dtype)
        got, gone = routed(loader, x, 4, mask=mask)
        off = mask == 0
        assert (got[off] == -1).all() and (gone[off] == 0).all() and torch.equal(got[~off], chosen[~off])
        loader.route_backward(dx, torch.ones((8, 4), device="cuda"), got, x, 8, 20, 4, renormalize=False)
        assert (dx[off] == 0).all()


def test_route_scores_next_to_each_other(loader):
    """Sums of score and bias that fp32 cannot tell apart are told apart."""
    x = torch.tensor([[0.5, 0.5, 0.25, 0.25]], device="cuda")
    s = scores64(x, SIGMOID)[0]
    # expert 2's bias lifts it to just above expert 0, by less than a rounding of fp32
    up = (s[0] - s[2]).item()
    bias = torch.tensor([0.0, 0.0, up, up], dtype=F32, device="cuda")
    want, _ = choice64(x, 2, SIGMOID, bias, 1, 1, 2)
    chosen, _ = routed(loader, x, 2, score=SIGMOID, bias=bias)
    assert torch.equal(chosen.long(), want)


def sorted64(chosen, E):
    flat = chosen.flatten().tolist()
    places, offsets, at = [-1] * len(flat), [0], 0
    for e in range(E):
        for i, c in enumerate(flat):
            if c == e:
                places[i] = at
                at += 1
        offsets.append(at)
    return torch.tensor(places, dtype=torch.int32).view(chosen.shape), torch.tensor(offsets, dtype=torch.int32)


def choices(M, k, E, seed, outside=0.0):
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, E, (M, k), generator=g).to(torch.int32)
    if outside:
        c[torch.rand((M, k), generator=g) < outside] = -1
        c[torch.rand((M, k), generator=g) < outside / 4] = E  # (no expert either)
    return c.cuda()


DISPATCHES = [(1, 8, 1, 1), (1, 5120, 8, 64), (5, 7, 3, 2), (32, 4096, 8, 64), (63, 100, 2, 512), (129, 33, 32, 5), (512, 64, 8, 16), (128, 1000, 8, 11), (129, 520, 8, 11),
              (513, 8, 8, 17), (2000, 24, 6, 130), (3, 1, 1, 300), (4097, 3, 3, 9)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=_id)
@pytest.mark.parametrize("size", DISPATCHES, ids=_id)
def test_dispatch(loader, size, dtype):
    M, N, k, E = size
    for outside, odd in ((0.0, False), (0.3, True)):
        chosen, x = choices(M, k, E, 1, outside), rnd((M, N), dtype, 2)
        x = odd_start(x) if odd else x
        rows = torch.full((M * k, N), 77.0, dtype=dtype, device="cuda")
        places = torch.full((M, k), -7, dtype=torch.int32, device="cuda")
        offsets = torch.full((E + 1,), -7, dtype=torch.int32, device="cuda")
        loader.dispatch(rows, offsets, places, x, chosen, M, N, k)
        want, ends = sorted64(chosen, E)
        assert torch.equal(offsets.cpu(), ends) and torch.equal(places.cpu(), want)
        there = want.flatten() >= 0
        assert torch.equal(rows[want.flatten()[there].long().cuda()], x.repeat_interleave(k, 0)[there.cuda()])
        assert (rows[int(ends[-1]):] == 77.0).all()  # behind the last: as they were
        again, also = torch.empty_like(offsets), torch.empty_like(places)
        loader.dispatch(None, again, also, None, chosen, M, N, k)
        assert torch.equal(again, offsets) and torch.equal(also, places)
        # the gradient of x: every token's rows summed
        dx = torch.full((M, N), math.nan, dtype=dtype, device="cuda")
        loader.combine(dx, rows, places, M, N, k)
        sums = (x.double()[:, None] * (places >= 0).double()[:, :, None])
        within(dx, sums.sum(1), (UNIT[dtype] + (k + 2) * E32) * sums.abs().sum(1) + LEAST[dtype], "gradient of x")


@pytest.mark.parametrize("size", [(70001, 8, 8, 256), (30000, 8, 8, 100), (3000, 8, 31, 512)], ids=_id)
def test_dispatch_of_many_choices(loader, size):
    """Tables of counts that the scan adds up and that every workgroup does, against a stable sort."""
    M, N, k, E = size
    chosen, x = choices(M, k, E, 3, 0.1), rnd((M, N), F16, 4)
    rows, places = torch.zeros((M * k, N), dtype=F16, device="cuda"), torch.empty((M, k), dtype=torch.int32, device="cuda")
    offsets = torch.empty(E + 1, dtype=torch.int32, device="cuda")
    loader.dispatch(rows, offsets, places, x, chosen, M, N, k)
    flat = torch.where((chosen < 0) | (chosen >= E), E, chosen).flatten().long()
    order = torch.argsort(flat, stable=True)
    n = int((flat < E).sum())
    want = torch.full_like(flat, -1)
    want[order[:n]] = torch.arange(n, device="cuda")
    assert torch.equal(places.flatten().long(), want)
    assert torch.equal(offsets.long(), torch.searchsorted(flat[order], torch.arange(E + 1, device="cuda")))
    assert torch.equal(rows[:n], x[order[:n] // k]) and (rows[n:] == 0).all()


@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F32, F32), (F16, F32), (BF16, F32)], ids=_id)
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (1, 5120, 8, 64), (33, 7, 5, 4), (50, 264, 32, 40), (300, 2056, 3, 9), (7, 8200, 2, 3)],
                         ids=_id)
def test_combine_and_its_gradients(loader, size, types):
    M, N, k, E = size
    kind, out = types
    for outside, odd, weighted, added in ((0.0, False, True, True), (0.3, True, True, False), (0.3, False, False, True)):
        move = odd_start if odd else lambda t: t
        chosen, y = choices(M, k, E, 1, outside), rnd((M * k, N), kind, 2)
        places = sorted64(chosen, E)[0].cuda()
        there = (places >= 0)[:, :, None]
        # rows that no place names must not be read: a number that would show
        unnamed = torch.ones(M * k, dtype=torch.bool, device="cuda")
        unnamed[places[places >= 0].long()] = False
        y[unnamed] = math.nan
        y = move(y)
        w, res = rnd((M, k), F32, 3) if weighted else None, move(rnd((M, N), out, 4)) if added else None
        C = move(torch.full((M, N), math.nan, dtype=out, device="cuda"))
        loader.combine(C, y, places, M, N, k, weights=w, residual=res)
        w64 = torch.ones((M, k, 1), dtype=torch.float64, device="cuda") if w is None else w.double()[:, :, None]
        terms = torch.where(there, w64 * torch.where(there, y[places.clamp_min(0).long()].double(), 0.0), 0.0)
        want, size64 = terms.sum(1), terms.abs().sum(1)
        if added:
            want, size64 = want + res.double(), size64 + res.double().abs()
        within(C, want, UNIT[out] * want.abs() + LEAST[out] + (k + 3) * E32 * size64, "sum")
        if added:
            loader.combine(res, y, places, M, N, k, weights=w, residual=res)  # onto itself
            assert torch.equal(res, C)
        dC = move(rnd((M, N), out, 5))
        drows, dw = move(torch.full((M * k, N), 77.0, dtype=kind, device="cuda")), torch.full((M, k), math.nan, device="cuda")
        loader.combine_backward(drows, dw, dC, y, places, M, N, k, weights=w)
        named = places[places >= 0].long()
        d64 = (w64 * dC.double()[:, None, :])[places >= 0]
        within(drows[named], d64, (UNIT[kind] + E32) * 1.01 * d64.abs() + LEAST[kind], "gradient of the rows")
        assert (drows[unnamed] == 77.0).all()
        dots = torch.where(there, dC.double()[:, None, :] * torch.where(there, y[places.clamp_min(0).long()].double(), 0.0), 0.0)
        within(dw, dots.sum(2), (N + 8) * E32 * dots.abs().sum(2), "gradient of the weights")
        only = torch.full_like(drows, 77.0)
        loader.combine_backward(only, None, dC, None, places, M, N, k, weights=w)
        assert torch.equal(only, drows)
        alone = torch.empty_like(dw)
        loader.combine_backward(None, alone, dC, y, places, M, N, k, weights=w)
        assert torch.equal(alone, dw)


def test_places_outside_the_rows_add_nothing(loader):
    M, N, k = 4, 16, 2
    y = rnd((M * k, N), BF16, 1)
    places = torch.tensor([[0, 8], [-5, 1], [2, 1 << 30], [-(1 << 31), 3]], dtype=torch.int32, device="cuda")
    C = torch.empty((M, N), dtype=BF16, device="cuda")
    loader.combine(C, y, places, M, N, k)
    assert torch.equal(C, y[[0, 1, 2, 3]])
    dw = torch.full((M, k), math.nan, device="cuda")
    drows = torch.zeros_like(y)
    loader.combine_backward(drows, dw, C, y, places, M, N, k)
    assert (dw[[0, 1, 2, 3], [1, 0, 1, 0]] == 0).all() and torch.equal(drows[:4], C) and (drows[4:] == 0).all()


def test_routing_of_nothing(loader):
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
    f32 = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    loader.route(i32(0, 2), f32(0, 2), f32(0, 8), 0, 8, 2)
    loader.route(i32(3, 0), f32(3, 0), f32(3, 8), 3, 8, 0)
    dx = torch.full((3, 8), math.nan, device="cuda")
    loader.route_backward(dx, f32(3, 0), i32(3, 0), f32(3, 8), 3, 8, 0)
    assert (dx == 0).all()
    offsets = torch.full((5,), -7, dtype=torch.int32, device="cuda")
    loader.dispatch(f32(0, 8), offsets, i32(0, 2), f32(0, 8), i32(0, 2), 0, 8, 2)
    assert (offsets == 0).all()
    offsets = torch.full((1,), -7, dtype=torch.int32, device="cuda")
    places = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    loader.dispatch(None, offsets, places, None, torch.zeros((3, 2), dtype=torch.int32, device="cuda"), 3, 8, 2)
    assert (offsets == 0).all() and (places == -1).all()  # no experts: every choice is outside
    C = torch.full((3, 8), math.nan, device="cuda")
    loader.combine(C, f32(0, 8), i32(3, 0), 3, 8, 0)
    assert (C == 0).all()
    dw = torch.full((3, 2), math.nan, device="cuda")
    loader.combine_backward(None, dw, f32(3, 0), f32(6, 0), torch.zeros((3, 2), dtype=torch.int32, device="cuda"), 3, 0, 2)
    assert (dw == 0).all()


def test_routing_on_a_side_stream_and_in_a_graph(loader):
    """The calls of a layer recorded once and replayed with new logits and rows, against the eager calls."""
    M, N, k, E = 1500, 72, 4, 24  # (several blocks of choices: the scratch buffer is used)
    x, h = rnd((M, E), BF16, 1), rnd((M, N), BF16, 2)
    chosen, places = (torch.empty((M, k), dtype=torch.int32, device="cuda") for _ in range(2))
    weights, offsets = torch.empty((M, k), device="cuda"), torch.empty(E + 1, dtype=torch.int32, device="cuda")
    rows, out = torch.zeros((M * k, N), dtype=BF16, device="cuda"), torch.empty((M, N), dtype=BF16, device="cuda")

    def layer(stream=None):
        loader.route(chosen, weights, x, M, E, k, stream=stream)
        loader.dispatch(rows, offsets, places, h, chosen, M, N, k, stream=stream)
        loader.combine(out, rows, places, M, N, k, weights=weights, stream=stream)

    layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    before = out.clone()
    out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    layer(side)
    side.synchronize()
    assert torch.equal(out, before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for seed in (3, 4, 5):
        x.copy_(rnd((M, E), BF16, seed)), h.copy_(rnd((M, N), BF16, seed + 10))
        layer()
        torch.cuda.synchronize()
        want = [t.clone() for t in (chosen, weights, offsets, places, rows, out)]
        for t in (chosen, weights, offsets, places, rows, out):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (chosen, weights, offsets, places, rows, out)))


def test_routing_refuses(loader):
    x, i, w = rnd((4, 8), F32, 1), torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.zeros((4, 2), device="cuda")
    with pytest.raises(TypeError):
        loader.route(i.long(), w, x, 4, 8, 2)
    with pytest.raises(TypeError):
        loader.route(i, w, x.double(), 4, 8, 2)
    with pytest.raises(ValueError):
        loader.route(i, w, x, 5, 8, 2)
    with pytest.raises(ValueError):
        loader.route(i, w, x.cpu(), 4, 8, 2)
    with pytest.raises(ValueError):
        loader.route(i, w, x.t().contiguous().t(), 4, 8, 2)
    with pytest.raises(TypeError):
        loader.route(i, w, x, 4, 8, 2, mask=torch.ones(4, device="cuda"))
    for bad in (dict(groups=3), dict(groups=0), dict(groups=2, kept_groups=3), dict(group_best=3), dict(scale=math.inf),
                dict(groups=8, kept_groups=1)):
        with pytest.raises(R.GemmLibraryError):
            loader.route(i, w, x, 4, 8, 2, **bad)
    with pytest.raises(ValueError):
        loader.dispatch(w, torch.zeros(9, dtype=torch.int32, device="cuda"), i, None, i, 4, 1, 2)
    with pytest.raises(ValueError):
        loader.combine_backward(None, None, x, None, i, 4, 8, 2)
    with pytest.raises(R.GemmLibraryError):
        loader.combine(x.half(), rnd((8, 8), BF16, 1), i, 4, 8, 2)


def test_rows_past_32_bits(loader):
    """More than 2^31 elements of sorted rows, 4.6 GB: dispatch, combine and its gradients, all of it or both ends."""
    M, N, k, E, dtype = 70001, 8192, 4, 64, BF16
    assert M * k * N > 1 << 31
    chosen, x = choices(M, k, E, 1, 0.02), rnd((M, N), dtype, 2)
    rows = torch.zeros((M * k, N), dtype=dtype, device="cuda")
    places, offsets = torch.empty((M, k), dtype=torch.int32, device="cuda"), torch.empty(E + 1, dtype=torch.int32, device="cuda")
    loader.dispatch(rows, offsets, places, x, chosen, M, N, k)
    flat = torch.where((chosen < 0) | (chosen >= E), E, chosen).flatten().long()
    order = torch.argsort(flat, stable=True)
    n = int((flat < E).sum())
    assert n * N > 1 << 31 and int(offsets[-1]) == n
    want = torch.full_like(flat, -1)
    want[order[:n]] = torch.arange(n, device="cuda")
    assert torch.equal(places.flatten().long(), want)
    for at in range(0, n, 32768):
        assert torch.equal(rows[at:min(at + 32768, n)], x[order[at:min(at + 32768, n)] // k]), at
    assert (rows[n:] == 0).all()
    w, dC = rnd((M, k), F32, 3), rnd((M, N), dtype, 5)
    C = torch.full((M, N), math.nan, dtype=dtype, device="cuda")
    loader.combine(C, rows, places, M, N, k, weights=w)
    drows, dw = torch.full_like(rows, 77.0), torch.full((M, k), math.nan, device="cuda")
    loader.combine_backward(drows, dw, dC, rows, places, M, N, k, weights=w)
    assert (drows[n:] == 77.0).all()
    for token in range(0, M, 8192):
        at = slice(token, min(token + 8192, M))
        there = (places[at] >= 0).double()
        # (every row is its token's: the sum is the token's row times its weights')
        factor, x64, d64 = w[at].double() * there, x[at].double(), dC[at].double()
        total = factor.sum(1, keepdim=True) * x64
        within(C[at], total, UNIT[dtype] * total.abs() + LEAST[dtype] + (k + 3) * E32 * factor.abs().sum(1, keepdim=True) * x64.abs(), "sum")
        dot = (x64 * d64).sum(1, keepdim=True) * there
        within(dw[at], dot, (N + 8) * E32 * (x64 * d64).abs().sum(1, keepdim=True) * there, "gradient of the weights")
        for j in range(k):
            is_there = places[at][:, j] >= 0
            d = (factor[:, j:j + 1] * d64)[is_there]
            within(drows[places[at][:, j][is_there].long()], d, (UNIT[dtype] + E32) * 1.01 * d.abs() + LEAST[dtype], "gradient of the rows")


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=_id)
@pytest.mark.parametrize("centre", [-640.0, -100.0, -90.0, -88.0, -86.0, -80.0, 0.0, 30.0, 600.0])
def test_gradient_of_sigmoid_weights_wherever_the_logits_lie(loader, centre, dtype):
    """All of a token's logits near `centre`, gradients as large as a scaled loss has them: a token's weights are shares of the
    sum of its scores, which is far below fp32's least number for most of these, and so is 1 - s for the last.

    The kernel works in fp64 and rounds to fp32, then to the logits' type; what is made of differences (dw_j - D) is off by
    some 2^-48 of the numbers subtracted."""
    M, E, k, size = 65, 40, 6, 4096.0 if dtype is not F16 else 256.0
    x, dw = (rnd((M, E), F32, 1, 1.5) + centre).to(dtype), rnd((M, k), F32, 2, size)
    s, rest = (1 / (1 + torch.exp(-v * x.double())) for v in (1, -1))  # s and 1 - s
    for renormalize, scale in ((True, 2.5), (False, 0.5)):
        chosen, weights = routed(loader, x, k, score=SIGMOID, renormalize=renormalize, scale=scale)
        p, q = s.gather(1, chosen.long()), rest.gather(1, chosen.long())
        w = p / p.sum(1, keepdim=True) if renormalize else p
        within(weights, scale * w, E32 * scale * w * 1.001 + LEAST[F32], "weights")
        dot, most = ((w * v).sum(1, keepdim=True) if renormalize else 0.0 for v in (dw.double(), dw.double().abs()))
        want = torch.zeros_like(s).scatter_(1, chosen.long(), scale * w * (dw.double() - dot) * q)
        part = torch.zeros_like(s).scatter_(1, chosen.long(), scale * w * (dw.double().abs() + most) * q)
        dx = torch.full((M, E), math.nan, dtype=dtype, device="cuda")
        loader.route_backward(dx, dw, chosen, x, M, E, k, score=SIGMOID, renormalize=renormalize, scale=scale)
        within(dx, want, (UNIT[dtype] + E32) * 1.01 * want.abs() + 2.0 ** -48 * part + LEAST[dtype] + LEAST[F32], "gradient of the logits")


@pytest.mark.parametrize("sizes", [(20, 1), (24, 4), (512, 1), (48, 16)], ids=_id)
def test_a_logit_that_is_no_number_is_chosen_last(loader, sizes):
    """The other experts are chosen as without it: by their scores among the numbers, with a bias, in groups, by every score."""
    E, groups = sizes
    M, k, each = 50, 6, E // groups
    kept = max(1, groups // 2) if each * (groups // 2) >= k + 2 else groups
    for score in (SOFTMAX, SIGMOID):
        for bias in (None, rnd((E,), F32, 3, 0.05 if score == SIGMOID else 0.01)):
            x = rnd((M, E), F32, 1, 1.5)
            gone = torch.randint(E, (M,), generator=torch.Generator().manual_seed(2)).cuda()
            bad = x.scatter(1, gone[:, None], math.nan)
            s = scores64(x.scatter(1, gone[:, None], -math.inf), score)  # (of the numbers; the one that is none counts 0 in their sum)
            value = (s if bias is None else s + bias.double()).scatter(1, gone[:, None], -math.inf)
            rank = value if bias is not None else x.double().scatter(1, gone[:, None], -math.inf)
            if groups > 1:
                of = value.view(M, groups, each).sort(2, descending=True)[0][:, :, :2].sum(2)
                best = of.sort(dim=1, descending=True, stable=True)[1][:, :kept]
                allowed = torch.zeros((M, groups), dtype=torch.bool, device="cuda").scatter_(1, best, True)
                rank = torch.where(allowed.repeat_interleave(each, 1), rank, -math.inf)
            want = rank.sort(dim=1, descending=True, stable=True)[1][:, :k]
            chosen, _ = routed(loader, bad, k, score=score, bias=bias, groups=groups, kept_groups=kept)
            assert torch.equal(chosen.long(), want), (score, bias is not None)
    if groups == 1 and E <= 32:
        for bias in (None, torch.zeros(E, device="cuda")):
            chosen, _ = routed(loader, bad, E, score=SOFTMAX, bias=bias)
            assert torch.equal(chosen[:, -1].long(), gone)


def test_no_more_groups_are_kept_than_asked_for(loader):
    """A group whose two best biased scores are infinite both ways has no sum: it is the lowest, not one more."""
    E, groups, kept, k = 16, 8, 1, 2
    x = rnd((40, E), F32, 1)
    bias = torch.zeros(E, device="cuda")
    bias[4], bias[5] = math.inf, -math.inf
    for score in (SOFTMAX, SIGMOID):
        chosen, _ = routed(loader, x, k, score=score, bias=bias, groups=groups, kept_groups=kept)
        assert (chosen // 2 == chosen[:, :1] // 2).all() and (chosen // 2 != 2).all(), score
