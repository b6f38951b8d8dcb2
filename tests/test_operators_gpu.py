"""The operators next to the GEMM on the GPU: linear layers with their epilogue, groups of rows
with a weight each, the gradients of both, and Newton-Schulz steps, against their definitions in
64 bits.

Tolerances are bounds, element by element: an output is rounded once (u_out of its own size), sums
are added up in fp32 (K + 8 roundings of 2^-23 of the sum of the absolute products), the logistic
function costs a few units of 2^-22, and what a backward pass multiplies, dZ, is rounded to 16
bits first where there is an activation.
"""
import itertools
import math
import random

import pytest
import torch

import rocm_wmma_gemm_amd as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
PAIRS = [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]  # (A and B, C)
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
LEAST = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}  # half the smallest subnormal
SUM = 2.0 ** -23
LOGISTIC = 16 * 2.0 ** -22
ACTS = list(R.activation)


@pytest.fixture(scope="module")
def loader():
    return R.Loader()


def _id(v):
    return str(v).replace("torch.", "").replace("activation.", "")


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=F32) * scale).to(dtype)


def act64(z, act):
    if act == R.activation.relu:
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == R.activation.silu:
        return z / (1 + torch.exp(-z))
    if act == R.activation.gelu:
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope64(z, act):
    if act == R.activation.relu:
        return (z > 0).double()
    if act == R.activation.silu:
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == R.activation.gelu:
        r = math.sqrt(2 / math.pi)
        t = torch.tanh(r * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * r * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    over = (got.double() - want).abs() - tol
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3g} over its bound at {int(over.argmax())}"


def weight64(B, layout):
    """As K x N (with a leading group dimension kept)."""
    return B.double().transpose(-1, -2) if layout == R.col_major else B.double()


def check_forward(C, kept, A, W, bias, residual, act, out, what):
    """A (M x K) and W (K x N) in 64 bits."""
    K = A.shape[1]
    z = A @ W
    size = A.abs() @ W.abs()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    err = (K + 8) * SUM * size
    if kept is not None:
        within(kept, z, UNIT[kept.dtype] * (z.abs() + err) + LEAST[kept.dtype] + err, what + " preact")
    y = act64(z, act)
    err = 1.2 * err + (LOGISTIC * z.abs() if act in (R.activation.silu, R.activation.gelu) else 0)
    if residual is not None:
        y = y + residual.double()
        err = err + 2.0 ** -23 * y.abs()
    within(C, y, UNIT[out] * (y.abs() + err) + LEAST[out] + err, what)


def weights(shape_kn, layout, dtype, seed, groups=None, scale=None):
    k, n = shape_kn
    shape = (k, n) if layout == R.row_major else (n, k)
    if groups is not None:
        shape = (groups,) + shape
    return rnd(shape, dtype, seed, 1 / math.sqrt(max(k, 1)) if scale is None else scale)


SIZES = [(1, 1, 1), (1, 8, 8), (1, 1024, 64), (2, 40, 1000), (3, 17, 5), (7, 256, 513), (16, 32, 128), (17, 96, 264),
         (33, 40, 72), (64, 64, 64), (65, 129, 200), (100, 512, 8), (128, 256, 64), (129, 136, 320), (257, 264, 136),
         (300, 513, 77), (511, 768, 192), (640, 1024, 1088)]


@pytest.mark.parametrize("types", PAIRS, ids=_id)
@pytest.mark.parametrize("size", SIZES, ids=_id)
def test_linear(loader, size, types):
    M, N, K = size
    ab, out = types
    combos = itertools.cycle(itertools.product((True, False), (False, True), (True, False)))
    for layout, act in itertools.product((R.col_major, R.row_major), ACTS):
        with_bias, with_residual, with_preact = next(combos)
        A, B = rnd((M, K), ab, 1), weights((K, N), layout, ab, 2)
        bias = rnd((N,), ab, 3) if with_bias else None
        residual = rnd((M, N), out, 4) if with_residual else None
        kept = torch.full((M, N), math.nan, dtype=ab, device="cuda") if with_preact else None
        C = torch.full((M, N), math.nan, dtype=out, device="cuda")
        loader.linear(C, A, B, M, N, K, layout, bias=bias, residual=residual, preact=kept, activation=act)
        check_forward(C, kept, A.double(), weight64(B, layout), bias, residual, act, out,
                      f"{size} {layout.name} {act.name}")


@pytest.mark.parametrize("types", PAIRS, ids=_id)
def test_linear_empty_sizes(loader, types):
    ab, out = types
    bias = rnd((24,), ab, 1)
    C = torch.full((5, 24), math.nan, dtype=out, device="cuda")
    loader.linear(C, torch.empty(0, dtype=ab, device="cuda"), torch.empty(0, dtype=ab, device="cuda"), 5, 24, 0,
                  bias=bias, activation=R.activation.relu)
    assert torch.equal(C, bias.clamp_min(0).to(out).expand(5, 24))
    nothing = torch.empty(0, dtype=out, device="cuda")
    empty = torch.empty(0, dtype=ab, device="cuda")
    loader.linear(nothing, empty, rnd((24, 8), ab, 1), 0, 24, 8)
    loader.linear(nothing, rnd((5, 8), ab, 1), empty, 5, 0, 8)
    # no rows: a gradient of zeros; accumulated: what was there
    dB, dbias = (torch.full(s, 3.0, dtype=out, device="cuda") for s in ((24, 8), (24,)))
    loader.linear_backward(None, dB, dbias, empty, empty, None, 0, 24, 8, accumulate=True)
    assert (dB == 3).all() and (dbias == 3).all()
    loader.linear_backward(None, dB, dbias, empty, empty, None, 0, 24, 8, preact=empty, activation=R.activation.silu)
    assert (dB == 0).all() and (dbias == 0).all()
    dA = torch.full((5, 8), 3.0, dtype=out, device="cuda")
    loader.linear_backward(dA, None, None, empty, None, empty, 5, 0, 8)
    assert (dA == 0).all()


@pytest.mark.parametrize("types", PAIRS, ids=_id)
def test_linear_in_place_residual_and_side_stream(loader, types):
    ab, out = types
    M, N, K = 200, 264, 136
    A, B, C = rnd((M, K), ab, 1), weights((K, N), R.col_major, ab, 2), rnd((M, N), out, 3)
    before = C.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    loader.linear(C, A, B, M, N, K, residual=C, stream=stream)
    stream.synchronize()
    check_forward(C, None, A.double(), weight64(B, R.col_major), None, before, R.activation.none, out, "in place")


def odd_start(t):
    """The same values one element further on in memory, so that no row starts on 16 bytes."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("types", PAIRS, ids=_id)
def test_operands_that_start_anywhere(loader, types, which):
    ab, out = types
    M, N, K = 150, 264, 200
    for layout in (R.col_major, R.row_major):
        t = [rnd((M, K), ab, 1), weights((K, N), layout, ab, 2), rnd((N,), ab, 3), rnd((M, N), out, 4),
             torch.empty((M, N), dtype=ab, device="cuda"), torch.empty((M, N), dtype=out, device="cuda")]
        t[which] = odd_start(t[which])
        A, B, bias, residual, kept, C = t
        loader.linear(C, A, B, M, N, K, layout, bias=bias, residual=residual, preact=kept,
                      activation=R.activation.gelu)
        check_forward(C, kept, A.double(), weight64(B, layout), bias, residual, R.activation.gelu, out, f"odd {which}")
        dA, dB, dbias = (torch.empty_like(x, dtype=out) for x in (A, B, bias))
        loader.linear_backward(dA, dB, dbias, kept, A, B, M, N, K, layout)
        check_backward(dA, dB, dbias, kept, None, A, B, layout, R.activation.none, out, f"odd {which}")


def check_backward(dA, dB, dbias, dC, Z, A, B, layout, act, out, what, before=None):
    """One problem: rows of one weight.  before: (dB, dbias) that were added to."""
    M, N = dC.shape
    W = weight64(B, layout)
    dz = dC.double()
    rounded, err = 0.0, torch.zeros_like(dz)
    if act != R.activation.none:
        dz = dz * slope64(Z.double(), act)
        # the slope's own error is a few units of 2^-22 of the terms it is made of (|z| to about 8 matters)
        err = dC.double().abs() * (8 * LOGISTIC if act != R.activation.relu else 0)
        rounded = UNIT[dC.dtype]
        err = err + rounded * (dz.abs() + err) + LEAST[dC.dtype]
    def bound(x, e):
        return UNIT[out] * (x.abs() + e) + LEAST[out] + e
    if dA is not None:
        want = dz @ W.t()
        e = (N + 8) * SUM * (dz.abs() @ W.abs().t()) + err @ W.abs().t()
        within(dA, want, bound(want, e), what + " dA")
    if dB is not None:
        a = A.double()
        want = a.t() @ dz
        e = (M + 8) * SUM * (a.abs().t() @ dz.abs()) + a.abs().t() @ err
        if layout == R.col_major:
            want, e = want.t(), e.t()
        if before is not None:
            want = want + before[0].double()
            e = e + SUM * want.abs()
        within(dB, want, bound(want, e), what + " dB")
    if dbias is not None:
        want = dz.sum(0)
        e = (M + 8) * SUM * dz.abs().sum(0) + err.sum(0)
        if before is not None:
            want = want + before[1].double()
            e = e + SUM * want.abs()
        within(dbias, want, bound(want, e), what + " dbias")


@pytest.mark.parametrize("types", PAIRS, ids=_id)
@pytest.mark.parametrize("size", SIZES, ids=_id)
def test_linear_backward(loader, size, types):
    M, N, K = size
    ab, out = types
    accumulate = itertools.cycle((False, True, False))
    for layout, act in itertools.product((R.col_major, R.row_major), ACTS):
        add = next(accumulate)
        A, B, dC, Z = rnd((M, K), ab, 1), weights((K, N), layout, ab, 2), rnd((M, N), ab, 3), rnd((M, N), ab, 4, 2.0)
        dA = torch.full((M, K), math.nan, dtype=out, device="cuda")
        dB = rnd(B.shape, out, 5) if add else torch.full(B.shape, math.nan, dtype=out, device="cuda")
        dbias = rnd((N,), out, 6) if add else torch.full((N,), math.nan, dtype=out, device="cuda")
        before = (dB.clone(), dbias.clone()) if add else None
        loader.linear_backward(dA, dB, dbias, dC, A, B, M, N, K, layout, preact=Z, activation=act, accumulate=add)
        check_backward(dA, dB, dbias, dC, Z, A, B, layout, act, out, f"{size} {layout.name} {act.name}", before)


def test_each_gradient_alone(loader):
    M, N, K = 130, 72, 200
    A, B, dC, Z = rnd((M, K), BF16, 1), weights((K, N), R.col_major, BF16, 2), rnd((M, N), BF16, 3), rnd((M, N), BF16, 4)
    whole = [torch.empty_like(A), torch.empty_like(B), torch.empty((N,), dtype=BF16, device="cuda")]
    loader.linear_backward(*whole, dC, A, B, M, N, K, preact=Z, activation=R.activation.silu)
    for i in range(3):
        one = [None, None, None]
        one[i] = torch.empty_like(whole[i])
        loader.linear_backward(*one, dC, A if i == 1 else None, B if i == 0 else None, M, N, K, preact=Z,
                               activation=R.activation.silu)
        assert torch.equal(one[i], whole[i])


# ---------------------------------------------------------------------------------------------
# groups of rows
# ---------------------------------------------------------------------------------------------
def routing(groups, rows, seed):
    rng = random.Random(seed)
    popular = [math.exp(rng.gauss(0, 1)) for _ in range(groups)]
    counts = [0] * groups
    for e in rng.choices(range(groups), popular, k=rows):
        counts[e] += 1
    return counts


GROUPS = [  # (rows of each group, N, K)
    ([1], 8, 8),
    ([0, 0, 3, 0], 64, 64),
    ([5, 0, 1, 17, 0], 40, 72),
    ([128, 128], 128, 64),
    ([0, 257, 64, 1, 129, 0], 136, 200),
    ([31, 2, 65], 33, 17),
    ([0, 0, 0], 64, 64),
    (routing(64, 16, 1), 256, 512),
    (routing(70, 900, 2), 72, 136),
    (routing(200, 333, 3), 64, 40),
    (routing(9, 2000, 4), 264, 520),
    ([700, 1], 513, 130),
]


def offsets_of(counts, start=0):
    ends = [start]
    for c in counts:
        ends.append(ends[-1] + c)
    return ends, torch.tensor(ends, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("types", PAIRS, ids=_id)
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_grouped(loader, case, types):
    counts, N, K = GROUPS[case]
    ab, out = types
    E = len(counts)
    before, behind = (3, 5) if case % 2 else (0, 0)  # rows of nobody
    ends, offsets = offsets_of(counts, before)
    M = ends[-1] + behind
    for layout, act in ((R.col_major, ACTS[case % 4]), (R.row_major, ACTS[(case + 1) % 4])):
        A, B = rnd((M, K), ab, 1), weights((K, N), layout, ab, 2, E)
        bias = rnd((E, N), ab, 3) if case % 3 else None
        residual = rnd((M, N), out, 4) if case % 2 else None
        kept = torch.full((M, N), -7.0, dtype=ab, device="cuda")
        C = torch.full((M, N), -7.0, dtype=out, device="cuda")
        # what no row of a group may see: the weights of groups without rows, the rows of nobody
        for e, c in enumerate(counts):
            if c == 0:
                B[e] = math.nan
        A[:before] = math.nan
        A[ends[-1]:] = math.nan
        loader.grouped(C, A, B, offsets, M, N, K, layout, bias=bias, residual=residual, preact=kept, activation=act)
        assert (C[:before] == -7).all() and (C[ends[-1]:] == -7).all()
        assert (kept[:before] == -7).all() and (kept[ends[-1]:] == -7).all()
        for e in range(E):
            at = slice(ends[e], ends[e + 1])
            if counts[e]:
                check_forward(C[at], kept[at], A[at].double(), weight64(B[e], layout),
                              None if bias is None else bias[e], None if residual is None else residual[at], act, out,
                              f"case {case} group {e} {layout.name} {act.name}")


@pytest.mark.parametrize("types", PAIRS, ids=_id)
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_grouped_backward(loader, case, types):
    counts, N, K = GROUPS[case]
    ab, out = types
    E = len(counts)
    before, behind = (2, 3) if case % 2 else (0, 0)
    ends, offsets = offsets_of(counts, before)
    M = ends[-1] + behind
    for layout, act, add in ((R.col_major, ACTS[case % 4], False), (R.row_major, ACTS[(case + 1) % 4], bool(case % 3))):
        A, B, dC, Z = rnd((M, K), ab, 1), weights((K, N), layout, ab, 2, E), rnd((M, N), ab, 3), rnd((M, N), ab, 4, 2.0)
        for t in (A, dC, Z):
            t[:before] = math.nan
            t[ends[-1]:] = math.nan
        dA = torch.full((M, K), -7.0, dtype=out, device="cuda")
        dB = rnd(B.shape, out, 5) if add else torch.full(B.shape, math.nan, dtype=out, device="cuda")
        dbias = rnd((E, N), out, 6) if add else torch.full((E, N), math.nan, dtype=out, device="cuda")
        old = (dB.clone(), dbias.clone())
        loader.grouped_backward(dA, dB, dbias, dC, A, B, offsets, M, N, K, layout, preact=Z, activation=act,
                                accumulate=add)
        assert (dA[:before] == -7).all() and (dA[ends[-1]:] == -7).all()
        for e in range(E):
            at = slice(ends[e], ends[e + 1])
            check_backward(dA[at] if counts[e] else None, dB[e], dbias[e], dC[at], Z[at], A[at], B[e], layout, act, out,
                           f"case {case} group {e} {layout.name} {act.name}",
                           (old[0][e], old[1][e]) if add else None)


def test_a_group_of_nan_rows_stays_alone(loader):
    """NaN and infinity in one group's rows and weights reach nothing of the other groups."""
    counts, N, K = [70, 5, 130, 64, 9], 136, 72
    ends, offsets = offsets_of(counts)
    M, E = ends[-1], len(counts)
    for poison in (math.nan, math.inf):
        A, B, dC = rnd((M, K), F16, 1), weights((K, N), R.col_major, F16, 2, E), rnd((M, N), F16, 3)
        for bad in (1, 3):
            A[ends[bad]:ends[bad + 1]] = poison
            dC[ends[bad]:ends[bad + 1]] = poison
            B[bad] = poison
        C, dA, dB, dbias = (torch.empty(s, dtype=F32, device="cuda") for s in ((M, N), (M, K), B.shape, (E, N)))
        loader.grouped(C, A, B, offsets, M, N, K)
        loader.grouped_backward(dA, dB, dbias, dC, A, B, offsets, M, N, K)
        for e in range(E):
            at = slice(ends[e], ends[e + 1])
            if e in (1, 3):
                assert not torch.isfinite(C[at]).any() and not torch.isfinite(dB[e]).any()
            else:
                check_forward(C[at], None, A[at].double(), weight64(B[e], R.col_major), None, None,
                              R.activation.none, F32, f"group {e}")
                check_backward(dA[at], dB[e], dbias[e], dC[at], None, A[at], B[e], R.col_major, R.activation.none, F32,
                               f"group {e}")


@pytest.mark.parametrize("act", ACTS, ids=_id)
def test_activations_of_special_values(loader, act):
    """Infinities, NaN and large values through the epilogue and the slope."""
    special = torch.tensor([0.0, -0.0, 1e-4, -1e-4, 20.0, -20.0, 3e4, -3e4, math.inf, math.nan, 1e30, -1e30],
                           device="cuda").to(BF16)
    M = special.numel()
    A = special.view(M, 1).contiguous()
    B = torch.ones((8, 1), dtype=BF16, device="cuda")
    C = torch.empty((M, 8), dtype=F32, device="cuda")
    loader.linear(C, A, B, M, 8, 1, activation=act)
    want = act64(special.double(), act).clamp(-1e38, math.inf)  # (the double's own overflow is not at issue)
    got = C[:, 3].double()
    big = special.double() == -1e30
    want = torch.where(special.double() < -1e29, torch.zeros_like(want) if act != R.activation.none else want, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (got, want)
    ok = torch.isfinite(want)
    assert ((got - want).abs()[ok] <= 2.0 ** -20 * (want.abs() + special.double().abs().clamp(max=1))[ok]).all(), (got, want)
    assert (got[~ok & ~torch.isnan(want)] == want[~ok & ~torch.isnan(want)]).all()
    # the slope, as the gradient of one column
    dC, Z = torch.ones((M, 8), dtype=BF16, device="cuda"), special.view(M, 1).expand(M, 8).contiguous()
    dA = torch.empty((M, 1), dtype=F32, device="cuda")
    eighth = torch.full((8, 1), 0.125, dtype=BF16, device="cuda")
    loader.linear_backward(dA, None, None, dC, None, eighth, M, 8, 1, preact=Z, activation=act)
    finite = special.double().clamp(-64, 64)
    want = slope64(finite, act)
    if act == R.activation.relu:
        want = torch.where(torch.isnan(special), torch.ones_like(want), want)  # (the gradient passes, as z <= 0 is false)
    got = dA[:, 0].double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (got, want)
    ok = torch.isfinite(want)
    assert ((got - want).abs()[ok] <= (2.0 ** -8 * want.abs() + 2.0 ** -18)[ok]).all(), (got, want)


@pytest.mark.parametrize("act", ACTS, ids=_id)
def test_gradients_against_differences(loader, act):
    """<dA, D> and <dB, D> against the change of the layer's own output along D (fp32 outputs;
    inputs on a grid that the steps keep exact)."""
    counts, N, K = [40, 0, 23, 66], 48, 64
    ends, offsets = offsets_of(counts)
    M, E = ends[-1], len(counts)
    grid = 2.0 ** -5  # values k / 32, |k| < 64, and steps of 1 / 32: sums of both are exact in f16
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    def on_grid(*shape):
        return (torch.randint(-32, 33, shape, generator=g, device="cuda") * grid).to(F16)
    A, B, bias = on_grid(M, K), on_grid(E, N, K) * 0.25, on_grid(E, N)
    if act == R.activation.relu:
        bias = bias + 2.0 ** -9  # no sum lies on the kink (sums are multiples of 2^-12 ... of the grid's square)
    W = rnd((M, N), F16, 7)

    def outputs(a, b, c):
        C, Z = torch.empty((M, N), dtype=F32, device="cuda"), torch.empty((M, N), dtype=F16, device="cuda")
        loader.grouped(C, a, b, offsets, M, N, K, bias=c, preact=Z, activation=act)
        return C.double(), Z

    _, Z = outputs(A, B, bias)
    dA, dB, dbias = (torch.empty(s, dtype=F16, device="cuda") for s in ((M, K), (E, N, K), (E, N)))
    loader.grouped_backward(dA, dB, dbias, W, A, B, offsets, M, N, K, preact=Z, activation=act)
    for name, grad in (("A", dA), ("B", dB), ("bias", dbias)):
        D = torch.zeros(grad.shape, device="cuda")
        at = torch.randperm(grad.numel(), generator=g, device="cuda")[:max(8, grad.numel() // 64)]
        D.view(-1)[at] = torch.where(torch.rand(at.numel(), generator=g, device="cuda") < 0.5, -1.0, 1.0)
        step = (D * grid).to(F16) * (1.0 if name != "B" else 0.25)
        size = step.float().abs().max().item()
        moved = lambda s: (A + s * step if name == "A" else A, B + s * step if name == "B" else B,  # noqa: E731
                           bias + s * step if name == "bias" else bias)
        up, down = outputs(*moved(1))[0], outputs(*moved(-1))[0]
        change = ((up - down) * W.double()).sum().item() / (2 * size)
        along = (grad.double() * D.double()).sum().item()
        # the third derivative over a step, the rounding of the gradients, kinks that a step of relu crosses
        scale = ((up - down).abs() * W.double().abs()).sum().item() / (2 * size)
        assert abs(change - along) <= (0.06 if act == R.activation.relu else 0.02) * scale + 1e-3, (name, change, along, scale)


def test_results_repeat_bit_for_bit(loader):
    counts, N, K = routing(16, 1500, 8), 512, 384
    ends, offsets = offsets_of(counts)
    M, E = ends[-1], len(counts)
    A, B, dC = rnd((M, K), BF16, 1), weights((K, N), R.col_major, BF16, 2, E), rnd((M, N), BF16, 3)
    G = rnd((3, 200, 136), F32, 4)
    seen = []
    for _ in range(3):
        C, dA, dB, dbias = (torch.empty(s, dtype=F32, device="cuda") for s in ((M, N), (M, K), B.shape, (E, N)))
        O = torch.empty(G.shape, dtype=BF16, device="cuda")
        loader.grouped(C, A, B, offsets, M, N, K, activation=R.activation.silu)
        loader.grouped_backward(dA, dB, dbias, dC, A, B, offsets, M, N, K)
        loader.orthogonalize(O, G, 200, 136, 3)
        seen.append((C, dA, dB, dbias, O))
    for other in seen[1:]:
        assert all(torch.equal(x, y) for x, y in zip(seen[0], other))


@pytest.mark.parametrize("kind", ["linear", "grouped"])
def test_more_elements_than_32_bits_count(loader, kind):
    """Rows past the 2^32nd byte and the 2^31st element of C (and of A)."""
    M, N, K = 70001, 32768, 32
    A, B = rnd((M, K), F16, 1), weights((K, N), R.col_major, F16, 2)
    C = torch.empty((M, N), dtype=F16, device="cuda")
    if kind == "linear":
        loader.linear(C, A, B, M, N, K)
    else:
        _, offsets = offsets_of([69000, 0, 1001])
        loader.grouped(C, A, torch.stack((B, B, B)), offsets, M, N, K)
    for at in (slice(0, 3), slice(65534, 65539), slice(M - 4, M)):
        check_forward(C[at], None, A[at].double(), weight64(B, R.col_major), None, None, R.activation.none, F16,
                      f"rows {at.start}")
    dA = torch.empty((M, K), dtype=F16, device="cuda")
    dB = torch.empty((N, K), dtype=F32, device="cuda")
    loader.linear_backward(dA, None, None, C, None, B, M, N, K)
    at = slice(M - 4, M)
    check_backward(dA[at], None, None, C[at], None, None, B, R.col_major, R.activation.none, F16, "last rows")
    del dB


def test_captured_in_a_graph(loader):
    """Forward, backward and update recorded once, replayed on new data between eager calls."""
    counts, N, K = [100, 0, 37, 60], 128, 64
    ends, offsets = offsets_of(counts)
    M, E = ends[-1], len(counts)
    A, B, dC = rnd((M, K), BF16, 1), weights((K, N), R.col_major, BF16, 2, E), rnd((M, N), BF16, 3)
    def outputs():
        return [torch.empty(s, dtype=BF16, device="cuda") for s in ((M, N), (M, N), (M, K), B.shape, (E, N), B.shape)]
    def step(C, Z, dA, dB, dbias, O):
        loader.grouped(C, A, B, offsets, M, N, K, preact=Z, activation=R.activation.gelu)
        loader.grouped_backward(dA, dB, dbias, dC, A, B, offsets, M, N, K, preact=Z, activation=R.activation.gelu)
        loader.orthogonalize(O, dB, N, K, E)
    eager, recorded = outputs(), outputs()
    step(*eager)  # sizes the scratch buffer
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*recorded)
    for replay in range(4):
        A.copy_(rnd((M, K), BF16, 10 + replay))
        dC.copy_(rnd((M, N), BF16, 20 + replay))
        offsets.copy_(offsets_of([100 - 20 * replay, 5 * replay, 37 + 10 * replay, 60])[1])
        step(*eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        last = int(offsets[-1])
        for i, (x, y) in enumerate(zip(eager, recorded)):
            same = torch.equal(x[:last], y[:last]) if i < 3 else torch.equal(x, y)
            assert same, (replay, i)


# ---------------------------------------------------------------------------------------------
# every kernel form, at sizes that the library's own choice sends there
# ---------------------------------------------------------------------------------------------
COVERED = [  # (product, M, N, K, groups, layout of B, types)
    ("forward", 2048, 4096, 512, 8, 1, 2), ("forward", 2048, 4096, 999, 8, 1, 0), ("forward", 512, 520, 512, 64, 0, 3),
    ("forward", 384, 520, 16384, 0, 0, 1), ("forward", 100, 8192, 512, 8, 0, 2), ("forward", 384, 1024, 16384, 0, 1, 0),
    ("forward", 1024, 1001, 512, 8, 0, 3), ("forward", 384, 1001, 16384, 0, 1, 2), ("forward", 1, 14336, 4096, 0, 1, 1),
    ("forward", 48, 520, 16384, 0, 1, 2), ("forward", 1, 4096, 16384, 0, 0, 0), ("forward", 24, 1024, 16384, 0, 0, 3),
    ("forward", 16, 8192, 1000, 8, 1, 2), ("forward", 64, 520, 8192, 0, 0, 0), ("forward", 24, 4096, 16384, 0, 0, 2),
    ("forward", 256, 1001, 999, 8, 0, 1), ("forward", 48, 14336, 4096, 0, 1, 0), ("forward", 48, 4096, 16384, 0, 1, 3),
    ("forward", 48, 8192, 1000, 8, 1, 0), ("forward", 384, 520, 16384, 0, 1, 2), ("forward", 1, 520, 16384, 0, 1, 1),
    ("forward", 1, 520, 999, 0, 1, 2), ("forward", 32, 1001, 512, 64, 0, 0), ("forward", 1, 520, 999, 64, 1, 3),
    ("forward", 4096, 5120, 5120, 0, 1, 2), ("forward", 1024, 1024, 999, 8, 0, 0),
    ("gradient_a", 2048, 1001, 4096, 8, 1, 2), ("gradient_a", 384, 14336, 512, 0, 1, 0), ("gradient_a", 2048, 4096, 512, 8, 1, 1),
    ("gradient_a", 384, 14336, 999, 0, 1, 2), ("gradient_a", 24, 14336, 1000, 0, 1, 3), ("gradient_a", 100, 14336, 999, 0, 0, 0),
    ("gradient_b", 4096, 520, 999, 0, 1, 3), ("gradient_b", 2048, 520, 512, 0, 1, 2), ("gradient_b", 4096, 4096, 512, 0, 0, 0),
    ("gradient_b", 777, 14336, 512, 0, 1, 1), ("gradient_b", 2048, 1024, 1000, 37, 0, 2), ("gradient_b", 3000, 2048, 1024, 11, 1, 3),
]


@pytest.mark.parametrize("case", range(len(COVERED)))
def test_sizes_of_every_form(loader, case):
    product, M, N, K, groups, layout, types = COVERED[case]
    ab, out = PAIRS[types]
    layout = R.m_layout(layout)
    counts = routing(groups, M, case) if groups else [M]
    ends, offsets = offsets_of(counts)
    A, B = rnd((M, K), ab, 1), weights((K, N), layout, ab, 2, groups or None)
    each = B if groups else B[None]
    act = ACTS[case % 4] if product == "forward" else R.activation.none
    if product == "forward":
        bias = rnd((groups or 1, N), ab, 3)
        residual = rnd((M, N), out, 4) if case % 2 else None
        kept = torch.full((M, N), math.nan, dtype=ab, device="cuda") if case % 3 else None
        C = torch.full((M, N), math.nan, dtype=out, device="cuda")
        if groups:
            loader.grouped(C, A, B, offsets, M, N, K, layout, bias=bias, residual=residual, preact=kept, activation=act)
        else:
            loader.linear(C, A, B, M, N, K, layout, bias=bias, residual=residual, preact=kept, activation=act)
    else:
        dC = rnd((M, N), ab, 3)
        result = torch.full((M, K) if product == "gradient_a" else B.shape, math.nan, dtype=out, device="cuda")
        wanted = (result, None, None) if product == "gradient_a" else (None, result, None)
        if groups:
            loader.grouped_backward(*wanted, dC, A, B, offsets, M, N, K, layout)
        else:
            loader.linear_backward(*wanted, dC, A, B, M, N, K, layout)
    for e, count in enumerate(counts):
        at, what = slice(ends[e], ends[e + 1]), f"{COVERED[case]} group {e}"
        if product == "forward":
            if count:
                check_forward(C[at], None if kept is None else kept[at], A[at].double(), weight64(each[e], layout),
                              bias[e], None if residual is None else residual[at], act, out, what)
        elif product == "gradient_a":
            if count:
                check_backward(result[at], None, None, dC[at], None, None, each[e], layout, act, out, what)
        else:
            check_backward(None, result[e] if groups else result, None, dC[at], None, A[at], each[e], layout, act, out, what)


def test_the_sizes_above_cover_the_forms(loader):
    seen = {}
    for product, M, N, K, groups, layout, types in COVERED:
        p = loader.product_select(product, M, N, K, groups, types, R.m_layout(layout))
        for what in (("form", p.form), ("cut", p.form if p.cut_tail else 0), ("slices", p.k_slices), ("once", p.once),
                     ("copies", p.copies)):
            seen.setdefault(what[0], set()).add(what[1])
    assert seen["form"] >= {0, 1, 2, 3, 4, 6, 7, 8, 9, 10, 11, 12, 13}, seen
    assert seen["cut"] >= {2, 3, 4, 6}, seen
    assert seen["slices"] >= {1, 2, 4} and seen["once"] == {0, 1} and seen["copies"] >= {0, 1, 2, 3}, seen


# ---------------------------------------------------------------------------------------------
# Newton-Schulz steps
# ---------------------------------------------------------------------------------------------
def steps64(G, steps=5, coefficients=(3.4445, -4.7750, 2.0315), epsilon=1e-7):
    a, b, c = coefficients
    X = G.double()
    X = X / (X.square().sum((1, 2), keepdim=True).sqrt() + epsilon)
    tall = X.shape[1] > X.shape[2]
    X = X.transpose(1, 2).contiguous() if tall else X
    for _ in range(steps):
        S = torch.matmul(X, X.transpose(1, 2).contiguous())
        X = a * X + torch.matmul(b * S + c * torch.matmul(S, S), X)
    return X.transpose(1, 2) if tall else X


#: what the f16 operands of the products may leave (2^-11 an operand; a step on noise shrinks
#: what the one before left, so that a few of them remain) and the rounding of the output
STEPS_TOLERANCE = {F16: 8 * 2.0 ** -11 + 2.0 ** -11, BF16: 8 * 2.0 ** -11 + 2.0 ** -8 / math.sqrt(3)}


@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 40), (2, 8, 8), (3, 7, 5), (1, 64, 64), (2, 65, 130), (2, 300, 72),
                                   (1, 128, 512), (1, 513, 257), (5, 96, 96), (1, 640, 640)], ids=_id)
@pytest.mark.parametrize("types", list(itertools.product((F32, BF16, F16), (BF16, F16))), ids=_id)
@pytest.mark.parametrize("spectrum", ["noise", "few strong directions"])
def test_orthogonalize(loader, shape, types, spectrum):
    batch, M, N = shape
    given, out = types
    G = rnd(shape, F32, 1)
    if spectrum != "noise":
        rank = max(1, min(M, N) // 32)
        G = 0.1 * G + rnd((batch, M, rank), F32, 2) @ rnd((batch, rank, N), F32, 3)
    G = G.to(given)
    O = torch.full(shape, math.nan, dtype=out, device="cuda")
    loader.orthogonalize(O, G, M, N, batch)
    want = steps64(G)
    for i in range(batch):
        off = (O[i].double() - want[i]).norm() / want[i].norm()
        assert off <= STEPS_TOLERANCE[out], (i, off)


def test_orthogonalize_other_steps_and_scales(loader):
    G = rnd((2, 96, 160), F32, 1)
    for steps, coefficients, scale in ((1, (1.5, -0.5, 0.0), 1.0), (2, (1.875, -1.25, 0.375), 1e-6),
                                       (9, (1.5, -0.5, 0.0), 1e6)):
        O = torch.empty(G.shape, dtype=F16, device="cuda")
        loader.orthogonalize(O, G * scale, 96, 160, 2, steps=steps, coefficients=coefficients)
        want = steps64(G * scale, steps, coefficients)
        assert (O.double() - want).norm() / want.norm() <= STEPS_TOLERANCE[F16]
    # a matrix of zeros stays one, next to one that is not
    G[0] = 0
    O = torch.empty(G.shape, dtype=BF16, device="cuda")
    loader.orthogonalize(O, G, 96, 160, 2)
    assert (O[0] == 0).all() and torch.isfinite(O[1].float()).all() and O[1].float().abs().max() > 0
    # a gradient with a NaN in it says so everywhere, and only in its own matrix
    G[0, 5, 7] = math.nan
    loader.orthogonalize(O, G, 96, 160, 2)
    assert torch.isnan(O[0]).all() and torch.isfinite(O[1].float()).all()


# ---------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------
def test_refusals(loader):
    A, B, C = (torch.zeros(s, dtype=BF16, device="cuda") for s in ((4, 8), (16, 8), (4, 16)))
    with pytest.raises(ValueError, match="holds"):
        loader.linear(C, A, B, 5, 16, 8)
    with pytest.raises(ValueError, match="31 bits"):
        loader.linear(C, A, B, -1, 16, 8)
    with pytest.raises(TypeError):
        loader.linear(C.half(), A, B, 4, 16, 8)
    with pytest.raises(TypeError, match="B must be"):
        loader.linear(C, A, B.half(), 4, 16, 8)
    with pytest.raises(ValueError, match="packed"):
        loader.linear(C, A.t(), B, 4, 16, 8)
    with pytest.raises(ValueError, match="device"):
        loader.linear(C, A.cpu(), B, 4, 16, 8)
    with pytest.raises(TypeError, match="residual"):
        loader.linear(C, A, B, 4, 16, 8, residual=C.float())
    with pytest.raises(ValueError):
        loader.linear(C, A, B, 4, 16, 8, activation=9)
    with pytest.raises(ValueError):
        loader.linear(C, A, B, 4, 16, 8, 2)
    with pytest.raises(ValueError, match="preact"):
        loader.linear_backward(torch.zeros_like(A), None, None, C, None, B, 4, 16, 8, activation=R.activation.relu)
    with pytest.raises(ValueError, match="wanted"):
        loader.linear_backward(None, None, None, C, A, B, 4, 16, 8)
    with pytest.raises(ValueError, match="needs"):
        loader.linear_backward(torch.zeros_like(A), None, None, C, A, None, 4, 16, 8)
    with pytest.raises(TypeError, match="share"):
        loader.linear_backward(torch.zeros_like(A), torch.zeros_like(B).float(), None, C, A, B, 4, 16, 8)
    offsets = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError, match="offsets"):
        loader.grouped(C, A, B, offsets.long(), 4, 16, 8)
    with pytest.raises(ValueError, match="offsets"):
        loader.grouped(C, A, B, offsets.cpu(), 4, 16, 8)
    with pytest.raises(ValueError, match="groups"):
        loader.grouped(C, A, B, torch.zeros(1026, dtype=torch.int32, device="cuda"), 4, 16, 8)
    with pytest.raises(ValueError, match="holds"):
        loader.grouped(C, A, B, torch.zeros(3, dtype=torch.int32, device="cuda"), 4, 16, 8)
    with pytest.raises(TypeError):
        loader.orthogonalize(torch.zeros(4, 8, device="cuda"), A, 4, 8)
    with pytest.raises(ValueError):
        loader.orthogonalize(torch.zeros_like(A), A, 4, 8, steps=0)
    with pytest.raises(ValueError, match="holds"):
        loader.orthogonalize(torch.zeros_like(A), A, 4, 8, 2)
    torch.cuda.synchronize()


def test_the_example_runs():
    """One training step and one decode step through the operators together."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, os.path.join(root, "examples", "expert_layer.py"), "--tokens", "300",
                           "--experts", "5", "--hidden", "256", "--inner", "384"], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout + done.stderr
    before, after = (float(x) for x in done.stdout.split("mean square of the output: ")[1].split("\n")[0].split(" -> "))
    assert after < before


def test_operands_on_another_device_than_the_current_one(loader, monkeypatch):
    A, B, C = (torch.zeros(s, dtype=BF16, device="cuda") for s in ((4, 8), (16, 8), (4, 16)))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="the current one is 1"):
        loader.linear(C, A, B, 4, 16, 8)
    with pytest.raises(ValueError, match="the current one is 1"):
        loader.linear_backward(torch.zeros_like(A), None, None, C, A, B, 4, 16, 8)
    with pytest.raises(ValueError, match="the current one is 1"):
        loader.orthogonalize(C, C, 4, 16)


@pytest.mark.parametrize("rows", [0, 1, 100, 3840, 3841, 3904], ids=_id)
def test_one_group_of_fewer_rows_than_the_call(loader, rows):
    """The gradient of a single group's weight, whose tiles are cut along the rows: those that its offsets
    leave out are not read."""
    M, N, K = 3904, 512, 512
    assert loader.product_select("gradient_b", M, N, K, 1, 3).cut_tail == 1
    for layout, before, add in ((R.col_major, 0, False), (R.row_major, (M - rows) // 2, True)):
        _, offsets = offsets_of([rows], before)
        at = slice(before, before + rows)
        A, B, dC = rnd((M, K), BF16, 1), weights((K, N), layout, BF16, 2, 1), rnd((M, N), BF16, 3)
        for t in (A, dC):
            t[:at.start] = math.nan
            t[at.stop:] = math.nan
        dA = torch.full((M, K), -7.0, dtype=F32, device="cuda")
        dB, dbias = rnd(B.shape, F32, 5), rnd((1, N), F32, 6)
        old = (dB[0].clone(), dbias[0].clone())
        loader.grouped_backward(dA, dB, dbias, dC, A, B, offsets, M, N, K, layout, accumulate=add)
        assert (dA[:at.start] == -7).all() and (dA[at.stop:] == -7).all()
        check_backward(dA[at] if rows else None, dB[0], dbias[0], dC[at], None, A[at], B[0], layout, R.activation.none, F32,
                       f"{rows} rows {layout.name}", old if add else None)


@pytest.mark.parametrize("size", [((1 << 25) + 1000, 8), (3, (1 << 22) + 64), (5, (1 << 22) + 65)], ids=_id)
def test_backward_of_more_runs_and_columns_than_the_grid_has(loader, size):
    """Rows past 2^25 (more than a million runs) and more than 65535 blocks of 64 columns."""
    M, N = size
    dC, Z = torch.zeros((M, N), dtype=F16, device="cuda"), torch.zeros((M, N), dtype=F16, device="cuda")
    rows = [r for r in (0, 1, 31, 32, 4095, (1 << 25) - 1, 1 << 25, (1 << 25) + 31, M - 33, M - 1) if 0 <= r < M]
    for i, r in enumerate(rows):
        dC[r], Z[r] = rnd((N,), F16, i), rnd((N,), F16, 100 + i)
    B = weights((4, N), R.col_major, F16, 2)
    dA, dbias = (torch.full(s, math.nan, dtype=F16, device="cuda") for s in ((M, 4), (N,)))
    loader.linear_backward(dA, None, dbias, dC, None, B, M, N, 4, preact=Z, activation=R.activation.silu)
    at = sorted(set(rows))
    check_backward(dA[at], None, dbias, dC[at], Z[at], None, B, R.col_major, R.activation.silu, F16, f"{size}")
    others = torch.ones(M, dtype=torch.bool, device="cuda")
    others[at] = False
    assert (dA[others] == 0).all()


@pytest.mark.parametrize("shape", [(4, 1000, 520), (1, 1024, 2048), (8, 640, 1024), (1, 2304, 2304)], ids=_id)
def test_large_updates_repeat_bit_for_bit(loader, shape):
    """Sizes whose symmetric products run on tiles that are written twice, mirrored."""
    batch, M, N = shape
    G = rnd(shape, F32, 4)
    seen = []
    for _ in range(6):
        O = torch.empty(G.shape, dtype=F16, device="cuda")
        loader.orthogonalize(O, G, M, N, batch)
        seen.append(O)
    assert all(torch.equal(seen[0], other) for other in seen[1:])


def test_more_updates_than_the_scratch_buffer_holds(loader):
    batch, M, N = 31, 72, 1 << 20  # 18.9 GB of state
    G = torch.empty((batch, M, N), dtype=BF16, device="cuda")
    for i in range(batch):
        G[i] = rnd((M, N), BF16, i)
    O = torch.full(G.shape, math.nan, dtype=BF16, device="cuda")
    loader.orthogonalize(O, G, M, N, batch)
    for i in (0, 14, 15, 16, 30):
        want = steps64(G[i:i + 1])[0]
        off = (O[i].double() - want).norm() / want.norm()
        assert off <= STEPS_TOLERANCE[BF16], (i, off)
    loader.workspace_release()


@pytest.mark.parametrize("shape", [(3, 40, 56), (2, 96, 160), (1, 300, 201), (1, 640, 1024)], ids=_id)
@pytest.mark.parametrize("given", [F32, BF16], ids=_id)
def test_updates_of_any_scale(loader, shape, given):
    """The square of an element may leave fp32 where the element does not: a power of two that all of G is
    multiplied by changes no bit of the update."""
    batch, M, N = shape
    G = rnd(shape, F32, 1).to(given)
    G = torch.where(G.abs() < 2.0 ** -10, torch.zeros_like(G), G)  # (nothing turns subnormal below)
    want = torch.empty(shape, dtype=F16, device="cuda")
    loader.orthogonalize(want, G, M, N, batch, epsilon=0.0)
    off = (want.double() - steps64(G, epsilon=0.0)).norm() / want.double().norm()
    assert off <= STEPS_TOLERANCE[F16], off
    for power in (-110, -75, 70, 120):
        O = torch.full(shape, math.nan, dtype=F16, device="cuda")
        loader.orthogonalize(O, G * 2.0 ** power, M, N, batch, epsilon=0.0)
        assert torch.equal(O, want), power


# Updates whose products run on each kernel form, with odd and even numbers of tile rows (128: 5, 9, 18; 192: 5, 22;
# 256: 4, 5), odd sides, tall and wide, alone and in a batch.
STEPS_COVERED = [(1, 8, 8), (1, 8, 300), (32, 33, 262), (2, 65, 130), (3, 70, 900), (32, 8, 520), (64, 65, 65), (64, 900, 65),
                 (1, 1024, 2048), (4, 1000, 520), (16, 1001, 520), (4, 1100, 1101), (1, 2304, 2304), (16, 900, 900), (1, 4096, 4096),
                 (16, 1024, 1024), (16, 1275, 1280), (8, 768, 2304), (1, 1536, 4096), (1, 3000, 1100), (1, 4090, 1530)]


def check_update(O, G, what):
    """By norm, and element by element.  Where the norm of the error is within its bound, its root mean square is;
    an element's error is a sum of many roundings, which pass eight times that in fewer than one of 10^14."""
    want = steps64(G)
    tol = STEPS_TOLERANCE[O.dtype]
    for i in range(G.shape[0]):
        err = O[i].double() - want[i]
        size = want[i].norm() / math.sqrt(want[i].numel())
        off = err.norm() / want[i].norm()
        assert off <= tol, (what, i, off)
        worst = (err.abs() - UNIT[O.dtype] * want[i].abs()).max() / size
        assert worst <= 8 * tol, (what, i, worst, int((err.abs() - UNIT[O.dtype] * want[i].abs()).argmax()))


@pytest.mark.parametrize("shape", STEPS_COVERED, ids=_id)
@pytest.mark.parametrize("spectrum", ["noise", "few strong directions"])
def test_updates_on_every_form(loader, shape, spectrum):
    batch, M, N = shape
    G = rnd(shape, F32, 1)
    if spectrum != "noise":
        rank = max(1, min(M, N) // 32)
        G = 0.1 * G + torch.matmul(rnd((batch, M, rank), F32, 2), rnd((batch, rank, N), F32, 3))
    for given, out in ((F32, BF16), (BF16, F16)):
        O = torch.full(shape, math.nan, dtype=out, device="cuda")
        loader.orthogonalize(O, G.to(given), M, N, batch)
        check_update(O, G.to(given), f"{shape} {given} {out}")


def test_the_updates_above_cover_the_forms(loader):
    seen = {}
    for batch, M, N in STEPS_COVERED:
        for product in ("steps_s", "steps_q", "steps_x", "steps_last"):
            for types in (0, 2):
                seen.setdefault(product, set()).add(loader.product_select(product, M, N, 0, batch, types).form)
    assert seen["steps_s"] >= {2, 3, 5, 9, 11, 12, 14} and seen["steps_q"] >= {2, 3, 5, 9, 11, 12, 14}, seen
    assert seen["steps_x"] >= {2, 3, 4, 9, 10, 11, 14} and seen["steps_last"] >= {2, 3, 4, 9, 10, 11, 14}, seen


ACCUMULATED = [  # (M, N, K, groups, layout of B, types): gradients of weights
    (40, 100, 77, 0, 1, 2), (300, 64, 64, 0, 1, 2), (4096, 520, 999, 0, 1, 3), (2048, 520, 512, 0, 1, 2), (3904, 512, 512, 1, 1, 3),
    (4096, 4096, 512, 0, 0, 0), (777, 14336, 512, 0, 1, 1), (8192, 1024, 1024, 0, 0, 1), (1024, 4096, 4096, 0, 0, 3),
    (4096, 5120, 5120, 0, 1, 2), (8192, 4352, 4608, 0, 1, 3), (2000, 2048, 4096, 4, 1, 1), (2048, 2048, 2048, 16, 1, 2),
    (2048, 1024, 1000, 37, 0, 2), (3000, 2048, 1024, 11, 1, 3), (999, 1001, 999, 24, 1, 0),
]


@pytest.mark.parametrize("case", range(len(ACCUMULATED)))
def test_accumulated_gradients_on_every_form(loader, case):
    """dB and dbias added to what is there, at the sizes of an accumulating training step: on each kernel form,
    on tiles that are cut along the rows, on groups that are dealt to teams of workgroups."""
    M, N, K, groups, layout, types = ACCUMULATED[case]
    ab, out = PAIRS[types]
    layout = R.m_layout(layout)
    counts = routing(groups, M, case) if groups else [M]
    if groups > 2:
        counts[1] += counts[2]  # (a group without rows keeps what it has)
        counts[2] = 0
    ends, offsets = offsets_of(counts)
    act = ACTS[case % 4]
    A, dC, Z = rnd((M, K), ab, 1), rnd((M, N), ab, 3), rnd((M, N), ab, 4, 2.0)
    shape = (N, K) if layout == R.col_major else (K, N)
    lead = (groups,) if groups else ()
    dB, dbias = rnd(lead + shape, out, 5), rnd(lead + (N,), out, 6)
    old = (dB.clone(), dbias.clone())
    for twice in range(2):
        if groups:
            loader.grouped_backward(None, dB, dbias, dC, A, None, offsets, M, N, K, layout, preact=Z, activation=act,
                                    accumulate=True)
        else:
            loader.linear_backward(None, dB, dbias, dC, A, None, M, N, K, layout, preact=Z, activation=act, accumulate=True)
        for e in range(len(counts)):
            at, what = slice(ends[e], ends[e + 1]), f"{ACCUMULATED[case]} group {e}, call {twice}"
            mine = (lambda t: t[e]) if groups else (lambda t: t)
            shape_only = torch.zeros(shape, dtype=ab, device="cuda")
            check_backward(None, mine(dB), mine(dbias), dC[at], Z[at], A[at], shape_only, layout, act, out, what,
                           (mine(old[0]), mine(old[1])))
            if counts[e] == 0:
                assert torch.equal(mine(dB), mine(old[0])) and torch.equal(mine(dbias), mine(old[1])), what
        old = (dB.clone(), dbias.clone())


def test_the_accumulated_sizes_cover_the_forms(loader):
    plans = [loader.product_select("gradient_b", M, N, K, groups, types, R.m_layout(layout))
             for M, N, K, groups, layout, types in ACCUMULATED]
    assert {p.form for p in plans} >= {1, 2, 3, 4, 6} and {p.form for p in plans if p.cut_tail} >= {2, 3, 4, 6}, plans


def steps_bound(G, steps, coefficients, out, epsilon=1e-7):
    """What f16 operands may leave of an update, to first order, in the Frobenius norm: every operand is off by
    2^-11 of itself, and a step passes on what came before times the largest slope of its polynomial."""
    a, b, c = coefficients
    u, X = 2.0 ** -11, G.double()
    X = X / (X.norm() + epsilon)
    X = X.t().contiguous() if X.shape[0] > X.shape[1] else X
    norm2 = lambda t: torch.linalg.matrix_norm(t, 2).item()  # noqa: E731
    normf = lambda t: t.norm().item()  # noqa: E731
    E = 0.0
    for _ in range(steps):
        S = X @ X.t()
        Q = b * S + c * (S @ S)
        x2, s2 = norm2(X), norm2(S)
        dS = 2 * u * x2 * normf(X) + u * normf(S)
        dQ = abs(b) * dS + abs(c) * (2 * s2 * dS + 2 * u * s2 * normf(S)) + u * normf(Q)
        E = E * (abs(a) + 3 * abs(b) * x2 ** 2 + 5 * abs(c) * x2 ** 4) + dQ * x2 + u * norm2(Q) * normf(X)
        X = a * X + Q @ X
    return 1.1 * E / normf(X) + UNIT[out]


@pytest.mark.parametrize("shape", [(64, 256), (256, 64), (64, 257), (65, 256), (300, 200), (520, 1001)], ids=_id)
@pytest.mark.parametrize("steps, coefficients", [(2, (3.0, -1.0, 0.0)), (1, (4.0, -2.0, 0.0)), (2, (2.0, 1.0, 1.0))], ids=_id)
def test_updates_whose_singular_values_grow(loader, shape, steps, coefficients):
    """Coefficients whose iterates reach 2 (and back), 2 and several hundred, on both sides of the size from which
    operands are rounded to f16."""
    M, N = shape
    G = 0.02 * rnd((M, N), F32, 1) / math.sqrt(M + N) + torch.outer(rnd((M,), F32, 2), rnd((N,), F32, 3)) / math.sqrt(M * N)
    O = torch.full((M, N), math.nan, dtype=BF16, device="cuda")
    loader.orthogonalize(O, G, M, N, steps=steps, coefficients=coefficients)
    want = steps64(G[None], steps, coefficients)[0]
    off = ((O.double() - want).norm() / want.norm()).item()
    assert off <= steps_bound(G, steps, coefficients, BF16), off
