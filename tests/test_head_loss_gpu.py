"""A projection onto a vocabulary with its loss on the GPU, against the definitions in 64 bits.

Bounds, element by element.  A logit is a sum of K products in fp32: off by (K + 8) 2^-23 of the sum of their absolute values,
`dz`.  The statistics add up to N exponentials in parts: each off by its argument's error and a few 2^-24, their sum by a
rounding for each of the additions that a value goes through (16 in a thread, 8 across a workgroup, the parts of a row).  The
gradient of a logit, rounded to A's type before it is multiplied (u of itself; f16 has a floor of 2^-25 / 2^13 of the largest), comes
out as sums of N and of M products.
"""
import math

import pytest
import torch

import rocm_wmma_gemm_amd as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
LEAST = {F16: 2.0 ** -25, BF16: 2.0 ** -133, F32: 2.0 ** -149}
SUM, E32 = 2.0 ** -23, 2.0 ** -24
PAIRS = [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]  # (A and B, gradients)


@pytest.fixture(scope="module")
def loader():
    return R.Loader()


def _id(v):
    return str(v).replace("torch.", "")


def rnd(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=F32) * scale).to(dtype)


def odd_start(t):
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    over = (got.double() - want).abs() - tol
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3g} over its bound at {int(over.argmax())}"


def problem(M, N, K, dtype, layout, seed):
    a, w = rnd((M, K), dtype, seed), rnd((N, K), dtype, seed + 1, 2.0 / math.sqrt(max(K, 1)))
    return a, w, (w if layout == R.col_major else w.t().contiguous())


def targets_of(M, N, seed, dtype=torch.int64):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = torch.randint(0, max(N, 1), (M,), device="cuda", generator=g)
    t[::5] = -100
    if M > 3:
        t[3] = N  # outside as well
    return t.to(dtype)


def logits64(a, w, t=1.0):
    """z / t and its bound."""
    return a.double() @ w.double().t() / t, (a.shape[1] + 8) * SUM * (a.double().abs() @ w.double().abs().t()) / t


def check_loss(loss, lse, x, dx, q, log_q, real, t, picked=None):
    """q, log_q: M x N."""
    want_lse = torch.logsumexp(x, 1)
    # every value goes through 16 + 8 additions and those of the row's parts, and through as many joins
    rounds = 64 + x.shape[1] / 1024
    d_lse = dx.max(1)[0] + rounds * E32 + 4 * E32 * x.abs().max(1)[0] + 2 * E32 * want_lse.abs()
    within(lse, want_lse, d_lse, "lse")
    terms = q * (log_q - x + want_lse[:, None])
    want = t * t * terms.sum(1)
    size = (q * (log_q.abs() + x.abs() + want_lse.abs()[:, None])).sum(1)
    tol = t * t * ((q * dx).sum(1) + d_lse + (16 + 12 + 8) * E32 * size + (16 * E32) * (terms.abs()).sum(1) * 4) * 1.01
    within(loss[real], want[real], tol[real], "loss")
    assert (loss[~real] == 0).all()


def check_gradients(dA, dB, a, w, layout, x, dx, q, real, dloss, t, before=None):
    dtype, out = a.dtype, (dA if dA is not None else dB).dtype
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - lse[:, None])
    g = (t * dloss.double() * real.double())[:, None]
    dz = g * (p - q)
    # p: the logit's error, the lse's, the exponential's argument and its own
    rel = dx + dx.max(1)[0][:, None] + (80 + x.shape[1] / 1024 + 8 * (x.abs() + lse.abs()[:, None])) * E32
    err = g.abs() * (p * rel + (p + q) * 40 * E32) * 1.01
    # what f16 holds ends at 2^-25 of a largest value of 2^13
    floor = g.abs().max().item() * 2.0 ** -38 if dtype is F16 and g.numel() else 0.0
    err = err + UNIT[dtype] * (dz.abs() + err) + floor
    err = torch.where(real[:, None], err, torch.zeros_like(err))
    W, A = w.double(), a.double()
    if dA is not None:
        want = dz @ W
        size = (dz.abs() + err) @ W.abs()
        tol = err @ W.abs() + (x.shape[1] + 16) * SUM * size
        within(dA, want, tol + UNIT[out] * (want.abs() + tol) + LEAST[out], "dA")
    if dB is not None:
        want = dz.t() @ A
        size = (dz.abs() + err).t() @ A.abs()
        tol = err.t() @ A.abs() + (a.shape[0] + 16) * SUM * size
        got = dB if layout == R.col_major else dB.t()
        if before is not None:
            add = (before if layout == R.col_major else before.t()).double()
            want, tol = want + add, tol + 2 * E32 * (want.abs() + add.abs())
        within(got, want, tol + UNIT[out] * (want.abs() + tol) + LEAST[out], "dB")


def one_hot(targets, N):
    real = (targets >= 0) & (targets < N)
    q = torch.zeros((targets.numel(), N), dtype=torch.float64, device="cuda")
    q[real, targets[real].long()] = 1.0
    return q, real


SIZES = [(1, 1, 1), (1, 7, 9), (1, 5000, 64), (2, 1000, 40), (5, 300, 17), (17, 4097, 96), (33, 2056, 264), (64, 12289, 72),
         (100, 520, 513), (129, 1111, 128), (256, 2048, 256), (300, 777, 77), (511, 5003, 192), (640, 8200, 136), (1300, 640, 320)]


@pytest.mark.parametrize("types", PAIRS, ids=_id)
@pytest.mark.parametrize("size", SIZES, ids=_id)
def test_cross_entropy_and_its_gradients(loader, size, types):
    M, N, K = size
    ab, out = types
    for layout, index in ((R.col_major, torch.int64), (R.row_major, torch.int32)):
        a, w, B = problem(M, N, K, ab, layout, 1)
        targets = targets_of(M, N, 2, index)
        q, real = one_hot(targets, N)
        x, dx = logits64(a, w)
        loss, lse = (torch.full((M,), math.nan, device="cuda") for _ in range(2))
        loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
        check_loss(loss, lse, x, dx, q, torch.zeros_like(q), real, 1.0)
        dloss = rnd((M,), F32, 5)
        dA, dB = torch.full((M, K), math.nan, dtype=out, device="cuda"), torch.full(B.shape, math.nan, dtype=out, device="cuda")
        loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K, layout)
        check_gradients(dA, dB, a, w, layout, x, dx, q, real, dloss, 1.0)


def lists_of(M, N, k, seed, dtype=torch.int64):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    entries = torch.randint(0, N, (M, k), device="cuda", generator=g)
    if M > 2:
        entries[1, k // 2:] = -1  # a short list
        entries[2] = -1  # an empty one
        entries[0, k - 1] = entries[0, 0]  # one listed twice
        entries[M - 1, 0] = N  # outside
    return entries.to(dtype), torch.randn((M, k), device="cuda", generator=g) * 2


def shares(entries, teacher, N, t):
    there = (entries >= 0) & (entries < N)
    given = torch.where(there, teacher.double() / t, -math.inf)
    real = there.any(1)
    share = torch.softmax(torch.where(real[:, None], given, 0.0), 1) * there
    q = torch.zeros((entries.shape[0], N), dtype=torch.float64, device="cuda")
    q.scatter_add_(1, entries.clamp(0, N - 1).long(), share)
    return share, q, real


def check_distillation(loss, lse, picked, x, dx, entries, teacher, t):
    M, N = x.shape
    share, q, real = shares(entries, teacher, N, t)
    want_lse = torch.logsumexp(x, 1)
    rounds = 64 + N / 1024
    d_lse = dx.max(1)[0] + rounds * E32 + 4 * E32 * x.abs().max(1)[0] + 2 * E32 * want_lse.abs()
    within(lse, want_lse, d_lse, "lse")
    at = entries.clamp(0, N - 1).long()
    there = (entries >= 0) & (entries < N)
    x_at, dx_at = (torch.where(there, v.gather(1, at), 0.0) for v in (x, dx))
    within(picked, x_at * t, dx_at * t, "picked")
    log_q = torch.where(share > 0, torch.log(share.clamp_min(1e-300)), 0.0)
    terms = share * (log_q - x_at + want_lse[:, None])
    # an exponential of the teacher: its argument's error (24 at most here) and its own; their sum over 4 rounds and 6 steps
    d_share = share * (2 * 24 + 24) * E32
    size = log_q.abs() + x_at.abs() + want_lse.abs()[:, None]
    tol = t * t * (share * (dx_at + d_lse[:, None] + 80 * E32 + 8 * E32 * size) + d_share * size + 12 * E32 * terms.abs()).sum(1) * 1.02
    within(loss[real], (t * t * terms.sum(1))[real], tol[real], "loss")
    assert (loss[~real] == 0).all()
    return q, real


@pytest.mark.parametrize("types", PAIRS, ids=_id)
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (1, 300, 16, 5), (3, 4099, 40, 256), (40, 1000, 77, 64), (130, 2056, 96, 17),
                                  (300, 5003, 200, 32), (600, 640, 128, 65)], ids=_id)
def test_distillation_and_its_gradients(loader, size, types):
    M, N, K, k = size
    ab, out = types
    for layout, index, t in ((R.col_major, torch.int32, 1.0), (R.row_major, torch.int64, 2.5)):
        a, w, B = problem(M, N, K, ab, layout, 1)
        entries, teacher = lists_of(M, N, k, 2, index)
        x, dx = logits64(a, w, t)
        loss, lse = (torch.full((M,), math.nan, device="cuda") for _ in range(2))
        picked = torch.full((M, k), math.nan, device="cuda")
        loader.linear_distillation(loss, lse, picked, a, B, entries, teacher, M, N, K, layout, temperature=t)
        q, real = check_distillation(loss, lse, picked, x, dx, entries, teacher, t)
        dloss = rnd((M,), F32, 5)
        dA, dB = torch.full((M, K), math.nan, dtype=out, device="cuda"), torch.full(B.shape, math.nan, dtype=out, device="cuda")
        loader.linear_distillation_backward(dA, dB, dloss, lse, picked, a, B, entries, teacher, M, N, K, layout, temperature=t)
        # (a share's own error is within the 40 roundings that (p + q) is given)
        check_gradients(dA, dB, a, w, layout, x, dx, q, real, dloss, t)
        alone = torch.empty_like(dB)
        loader.linear_distillation_backward(None, alone, dloss, lse, picked, a, B, entries, teacher, M, N, K, layout, temperature=t)
        assert torch.equal(alone, dB)


@pytest.mark.parametrize("ab", [F16, BF16], ids=_id)
def test_many_pieces_of_the_vocabulary(loader, ab):
    """More rows than a whole vocabulary's logits fit a piece for; weights either way up, with rows that start anywhere."""
    M, K = 20000, 64
    for N, layout in ((5000, R.col_major), (5000, R.row_major), (4999, R.row_major)):
        a, w, B = problem(M, N, K, ab, layout, 1)
        targets = targets_of(M, N, 2)
        q, real = one_hot(targets, N)
        x, dx = logits64(a, w)
        loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
        check_loss(loss, lse, x, dx, q, torch.zeros_like(q), real, 1.0)
        dloss = rnd((M,), F32, 5) / M
        dA, dB = torch.empty((M, K), dtype=ab, device="cuda"), torch.empty(B.shape, dtype=ab, device="cuda")
        loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K, layout)
        check_gradients(dA, dB, a, w, layout, x, dx, q, real, dloss, 1.0)
        del q, x, dx


@pytest.mark.parametrize("types", PAIRS, ids=_id)
@pytest.mark.parametrize("size", [(1, 16384, 64), (3, 20000, 72), (33, 17001, 136), (64, 40000, 40), (40, 4099, 1030), (65, 20000, 72),
                                  (2, 70000, 9)], ids=_id)
def test_gradients_of_few_rows(loader, size, types):
    """Outer products, and sums over a vocabulary that goes in segments, a whole number of them or not."""
    M, N, K = size
    ab, out = types
    for layout in (R.col_major, R.row_major):
        a, w, B = problem(M, N, K, ab, layout, 1)
        targets, dloss = targets_of(M, N, 2), rnd((M,), F32, 5)
        targets[-1] = N - 1
        q, real = one_hot(targets, N)
        x, dx = logits64(a, w)
        loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
        check_loss(loss, lse, x, dx, q, torch.zeros_like(q), real, 1.0)
        for accumulate in (False, True):
            flat = rnd((B.numel() + 64,), out, 6)
            kept = flat.clone()
            dA, dB = torch.full((M, K), math.nan, dtype=out, device="cuda"), flat[32:32 + B.numel()].view(B.shape)
            loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K, layout, accumulate=accumulate)
            before = kept[32:32 + B.numel()].view(B.shape) if accumulate else None
            check_gradients(dA, dB, a, w, layout, x, dx, q, real, dloss, 1.0, before)
            assert torch.equal(flat[:32], kept[:32]) and torch.equal(flat[32 + B.numel():], kept[32 + B.numel():])


def test_few_rows_and_many_columns_that_start_anywhere(loader):
    """Weights stored K x N whose rows start on odd elements, few rows, many columns."""
    M, N, K = 255, 132001, 24
    for ab in (F16, BF16):
        a, w, B = problem(M, N, K, ab, R.row_major, 1)
        targets, dloss = targets_of(M, N, 2), rnd((M,), F32, 5)
        targets[0] = N - 1
        q, real = one_hot(targets, N)
        x, dx = logits64(a, w)
        loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, R.row_major)
        check_loss(loss, lse, x, dx, q, torch.zeros_like(q), real, 1.0)
        dA, dB = torch.empty((M, K), dtype=F32, device="cuda"), torch.empty(B.shape, dtype=ab, device="cuda")
        loader.linear_cross_entropy_backward(dA, None, dloss, lse, a, B, targets, M, N, K, R.row_major)
        check_gradients(dA, None, a, w, R.row_major, x, dx, q, real, dloss, 1.0)
        loader.linear_cross_entropy_backward(None, dB, dloss, lse, a, B, targets, M, N, K, R.row_major)
        check_gradients(None, dB, a, w, R.row_major, x, dx, q, real, dloss, 1.0)


@pytest.mark.parametrize("types", PAIRS, ids=_id)
def test_gradients_that_are_added_to_and_wanted_alone(loader, types):
    ab, out = types
    for (M, N, K), layout in (((70, 1000, 96), R.col_major), ((300, 1003, 72), R.row_major), ((257, 520, 77), R.col_major)):
        a, w, B = problem(M, N, K, ab, layout, 1)
        targets = targets_of(M, N, 2)
        q, real = one_hot(targets, N)
        x, dx = logits64(a, w)
        loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
        dloss, before = rnd((M,), F32, 5), rnd(B.shape, out, 6)
        dB, dA = before.clone(), torch.empty((M, K), dtype=out, device="cuda")
        loader.linear_cross_entropy_backward(None, dB, dloss, lse, a, B, targets, M, N, K, layout, accumulate=True)
        check_gradients(None, dB, a, w, layout, x, dx, q, real, dloss, 1.0, before)
        loader.linear_cross_entropy_backward(dA, None, dloss, lse, a, B, targets, M, N, K, layout)
        check_gradients(dA, None, a, w, layout, x, dx, q, real, dloss, 1.0)


@pytest.mark.parametrize("types", PAIRS, ids=_id)
@pytest.mark.parametrize("odd", [0, 1])
def test_weight_gradients_whose_rows_start_anywhere(loader, types, odd):
    """Rows of odd lengths, several tiles of them: every element is right, also where it is added to, and nothing around
    the gradient is written."""
    ab, out = types
    for (M, N, K), layout in (((700, 1501, 301), R.row_major), ((513, 300, 1031), R.col_major), ((300, 5003, 130), R.row_major),
                              ((400, 2305, 259), R.col_major), ((260, 513, 255), R.row_major)):
        a, w, B = problem(M, N, K, ab, layout, 1)
        targets, dloss = targets_of(M, N, 2), rnd((M,), F32, 5)
        q, real = one_hot(targets, N)
        x, dx = logits64(a, w)
        loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
        for accumulate in (False, True):
            flat = rnd((B.numel() + 2048 + odd,), out, 6)
            kept = flat.clone()
            dB = flat[1024 + odd:1024 + odd + B.numel()].view(B.shape)
            loader.linear_cross_entropy_backward(None, dB, dloss, lse, a, B, targets, M, N, K, layout, accumulate=accumulate)
            before = kept[1024 + odd:1024 + odd + B.numel()].view(B.shape) if accumulate else None
            check_gradients(None, dB, a, w, layout, x, dx, q, real, dloss, 1.0, before)
            assert torch.equal(flat[:1024 + odd], kept[:1024 + odd])
            assert torch.equal(flat[1024 + odd + B.numel():], kept[1024 + odd + B.numel():])


@pytest.mark.parametrize("which", range(4))
def test_operands_that_start_anywhere(loader, which):
    for (M, N, K), layout in (((40, 520, 72), R.col_major), ((300, 520, 72), R.row_major), ((300, 1000, 136), R.col_major)):
        t = list(problem(M, N, K, BF16, layout, 1)[i] for i in (0, 2)) + [torch.empty((M, K), dtype=BF16, device="cuda")]
        w = t[1] if layout == R.col_major else t[1].t()
        t.append(torch.empty_like(t[1]))
        t[which] = odd_start(t[which])
        a, B, dA, dB = t
        targets = targets_of(M, N, 2)
        q, real = one_hot(targets, N)
        x, dx = logits64(a, w)
        loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
        check_loss(loss, lse, x, dx, q, torch.zeros_like(q), real, 1.0)
        dloss = rnd((M,), F32, 5)
        loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K, layout)
        check_gradients(dA, dB, a, w, layout, x, dx, q, real, dloss, 1.0)


def test_what_lies_behind_the_operands_is_not_read_into_the_results(loader):
    """Numbers that would show right behind A, B and, for weights stored K x N, behind every block of columns."""
    for (M, N, K), layout in (((300, 1000, 72), R.row_major), ((300, 1000, 72), R.col_major), ((20, 1000, 72), R.row_major),
                              ((20000, 5000, 72), R.row_major)):
        a, w, B = problem(M, N, K, BF16, layout, 1)

        def fenced(t):
            flat = torch.full((t.numel() + 4096,), math.nan, dtype=t.dtype, device="cuda")
            flat[:t.numel()] = t.flatten()
            return flat[:t.numel()].view(t.shape)

        targets, dloss = targets_of(M, N, 2), rnd((M,), F32, 5)
        results = []
        for A_, B_ in ((a, B), (fenced(a), fenced(B))):
            loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
            dA, dB = torch.empty((M, K), dtype=BF16, device="cuda"), torch.empty_like(B)
            loader.linear_cross_entropy(loss, lse, A_, B_, targets, M, N, K, layout)
            loader.linear_cross_entropy_backward(dA, dB, dloss, lse, A_, B_, targets, M, N, K, layout)
            results.append((loss, lse, dA, dB))
        assert all(torch.isfinite(t.float()).all() and torch.equal(t, u) for t, u in zip(*results))


def test_extreme_logits_and_small_losses(loader):
    """Logits of thousands, a row that is sure of its target, a loss's gradient far below what f16 holds."""
    M, N, K = 64, 600, 64
    for ab in (F16, BF16):
        a, w, B = problem(M, N, K, ab, R.col_major, 1)
        targets = torch.arange(M, device="cuda")
        a[:32] = (w[targets[:32]].float() * torch.linspace(0.1, 60, 32, device="cuda")[:, None]).to(ab)
        a[32:40] *= 300
        q, real = one_hot(targets, N)
        x, dx = logits64(a, w)
        loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
        loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K)
        check_loss(loss, lse, x, dx, q, torch.zeros_like(q), real, 1.0)
        for size in (1e-9, 1.0, 1e6):
            dloss = rnd((M,), F32, 5) * size
            dA, dB = torch.empty((M, K), dtype=F32, device="cuda"), torch.empty(B.shape, dtype=F32, device="cuda")
            loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K)
            check_gradients(dA, dB, a, w, R.col_major, x, dx, q, real, dloss, 1.0)


def test_gradient_of_the_loss_against_differences(loader):
    """A step along a random direction of the states, in 64 bits, against the gradient."""
    M, N, K, k, t = 5, 200, 32, 6, 2.0
    a, w, B = problem(M, N, K, BF16, R.col_major, 1)
    entries, teacher = lists_of(M, N, k, 2)
    loss, lse, picked = torch.empty(M, device="cuda"), torch.empty(M, device="cuda"), torch.empty((M, k), device="cuda")
    loader.linear_distillation(loss, lse, picked, a, B, entries, teacher, M, N, K, temperature=t)
    dA, dB = torch.empty((M, K), device="cuda"), torch.empty((N, K), device="cuda")
    loader.linear_distillation_backward(dA, dB, torch.ones(M, device="cuda"), lse, picked, a, B, entries, teacher, M, N, K, temperature=t)
    share, q, real = shares(entries, teacher, N, t)

    def total(states, weights):
        log_p = torch.log_softmax(states @ weights.t() / t, 1)
        return (t * t * (torch.xlogy(share, share).sum(1) - (q * log_p).sum(1)) * real).sum()

    for seed in range(3):
        va, vw, step = rnd((M, K), F32, 20 + seed).double(), rnd((N, K), F32, 30 + seed).double(), 1e-5
        by_a = (total(a.double() + step * va, w.double()) - total(a.double() - step * va, w.double())) / (2 * step)
        by_w = (total(a.double(), w.double() + step * vw) - total(a.double(), w.double() - step * vw)) / (2 * step)
        for got, want, size in (((dA.double() * va).sum(), by_a, (dA.double() * va).abs().sum()),
                                ((dB.double() * vw).sum(), by_w, (dB.double() * vw).abs().sum())):
            # every term of the gradient is off by dz's rounding, 2^-8 of what it is made of (up to twice itself here)
            assert (got - want).abs() < 4 * 2.0 ** -8 * size + 1e-6


def test_losses_of_nothing(loader):
    f32 = lambda *s: torch.full(s, math.nan, device="cuda")  # noqa: E731
    b16 = lambda *s: torch.full(s, math.nan, dtype=BF16, device="cuda")  # noqa: E731
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64, device="cuda")  # noqa: E731
    loader.linear_cross_entropy(f32(0), f32(0), b16(0, 8), b16(16, 8), i64(0), 0, 16, 8)
    dB = b16(16, 8)
    loader.linear_cross_entropy_backward(b16(0, 8), dB, f32(0), f32(0), b16(0, 8), b16(16, 8), i64(0), 0, 16, 8)
    assert (dB == 0).all()
    dB = torch.ones((16, 8), dtype=F16, device="cuda")
    loader.linear_cross_entropy_backward(None, dB, f32(0), f32(0), dB[:0], dB, i64(0), 0, 16, 8, accumulate=True)
    assert (dB == 1).all()
    # states of no length: every logit is 0
    loss, lse = f32(3), f32(3)
    loader.linear_cross_entropy(loss, lse, b16(3, 0), b16(16, 0), i64(3), 3, 16, 0)
    assert ((loss - math.log(16)).abs() < 1e-5).all() and ((lse - math.log(16)).abs() < 1e-5).all()
    # no vocabulary: every row is left out
    loss, lse, dA = f32(3), f32(3), b16(3, 8)
    loader.linear_cross_entropy(loss, lse, torch.ones_like(dA), b16(0, 8), i64(3), 3, 0, 8)
    assert (loss == 0).all() and (lse == -math.inf).all()
    loader.linear_cross_entropy_backward(dA, None, torch.ones(3, device="cuda"), lse, torch.ones_like(dA), b16(0, 8), i64(3), 3, 0, 8)
    assert (dA == 0).all()
    # nobody has a target: no gradient, whatever dloss says
    M, N, K = 40, 300, 64
    a, w, B = problem(M, N, K, BF16, R.col_major, 1)
    none, dA, dB = i64(M) - 100, b16(M, K), b16(N, K)
    loss, lse = f32(M), f32(M)
    loader.linear_cross_entropy(loss, lse, a, B, none, M, N, K)
    loader.linear_cross_entropy_backward(dA, dB, f32(M), lse, a, B, none, M, N, K)
    assert (loss == 0).all() and (dA == 0).all() and (dB == 0).all()


def test_losses_on_a_side_stream_and_in_a_graph(loader):
    """A step of the head recorded once and replayed with new states and targets, against the eager step."""
    M, N, K, k = 300, 3000, 72, 9
    for ab in (F16, BF16):
        a, w, B = problem(M, N, K, ab, R.col_major, 1)
        targets, dloss = targets_of(M, N, 2), rnd((M,), F32, 5)
        entries, teacher = lists_of(M, N, k, 2)
        out = [torch.empty(s, dtype=d, device="cuda") for s, d in (((M,), F32), ((M,), F32), ((M, K), ab), ((N, K), ab), ((M,), F32),
                                                                   ((M,), F32), ((M, k), F32), ((M, K), ab), ((N, K), ab))]

        def both(stream=None):
            loader.linear_cross_entropy(out[0], out[1], a, B, targets, M, N, K, stream=stream)
            loader.linear_cross_entropy_backward(out[2], out[3], dloss, out[1], a, B, targets, M, N, K, stream=stream)
            loader.linear_distillation(out[4], out[5], out[6], a, B, entries, teacher, M, N, K, stream=stream)
            loader.linear_distillation_backward(out[7], out[8], dloss, out[5], out[6], a, B, entries, teacher, M, N, K, stream=stream)

        both()
        torch.cuda.synchronize()
        want = [t.clone() for t in out]
        side = torch.cuda.Stream()
        for t in out:
            t.zero_()
        side.wait_stream(torch.cuda.current_stream())
        both(side)
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, out))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            both()
        for seed in (11, 12, 13):
            a.copy_(rnd((M, K), ab, seed)), targets.copy_(targets_of(M, N, seed))
            both()
            torch.cuda.synchronize()
            want = [t.clone() for t in out]
            for t in out:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want, out))


def test_losses_refuse(loader):
    M, N, K = 4, 16, 8
    a, w, B = problem(M, N, K, BF16, R.col_major, 1)
    loss, lse, t = torch.empty(M, device="cuda"), torch.empty(M, device="cuda"), torch.zeros(M, dtype=torch.int64, device="cuda")
    entries, teacher = t.view(M, 1), torch.zeros((M, 1), device="cuda")
    with pytest.raises(TypeError):
        loader.linear_cross_entropy(loss, lse, a.float(), B.float(), t, M, N, K)
    with pytest.raises(TypeError):
        loader.linear_cross_entropy(loss, lse, a, B.half(), t, M, N, K)
    with pytest.raises(TypeError):
        loader.linear_cross_entropy(loss, lse, a, B, t.to(torch.int16), M, N, K)
    with pytest.raises(TypeError):
        loader.linear_cross_entropy(loss.half(), lse, a, B, t, M, N, K)
    with pytest.raises(ValueError):
        loader.linear_cross_entropy(loss, lse, a, B, t, M + 1, N, K)
    with pytest.raises(ValueError):
        loader.linear_cross_entropy_backward(None, None, loss, lse, a, B, t, M, N, K)
    with pytest.raises(TypeError):
        loader.linear_cross_entropy_backward(a.half(), None, loss, lse, a, B, t, M, N, K)
    with pytest.raises(ValueError):
        loader.linear_distillation(loss, lse, loss, a, B, t, teacher, M, N, K)  # entries without rows
    with pytest.raises(ValueError):
        loader.linear_distillation(loss, lse, loss, a, B, torch.zeros((M, 257), dtype=torch.int32, device="cuda"), teacher, M, N, K)
    for temperature in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(R.GemmLibraryError):
            loader.linear_distillation(loss, lse, loss, a, B, entries, teacher, M, N, K, temperature=temperature)


def slopes64(x, dx, lse, d_lse, q, real, dloss, dtype):
    """The gradient of some columns of logits and its bound, as in check_gradients, from the lse of whole rows (up to 2^20
    columns) and the largest of their logits' bounds."""
    p = torch.exp(x - lse[:, None])
    g = (dloss.double() * real.double())[:, None]
    dz = g * (p - q)
    rel = dx + d_lse[:, None] + (80 + 1024 + 8 * (x.abs() + lse.abs()[:, None])) * E32
    err = g.abs() * (p * rel + (p + q) * 40 * E32) * 1.01
    err = err + UNIT[dtype] * (dz.abs() + err)
    return dz, torch.where(real[:, None], err, torch.zeros_like(err))


@pytest.mark.parametrize("size", [(9, 540001, R.col_major), (300, 540000, R.col_major), (9, 540000, R.row_major),
                                  (300, 540001, R.row_major)], ids=_id)
def test_weights_past_32_bits(loader, size):
    """More than 2^31 weights, 4.4 GB, on few rows and on tiles; their gradient at the ends and on both sides of 2^31 elements."""
    (M, N, layout), K, ab = size, 4096, BF16
    assert N * K > 1 << 31
    a = rnd((M, K), ab, 1)
    B = torch.empty((N, K) if layout == R.col_major else (K, N), dtype=ab, device="cuda")
    w = B if layout == R.col_major else B.t()
    x, dx = (torch.empty((M, N), dtype=torch.float64, device="cuda") for _ in range(2))
    for v0 in range(0, N, 65536):
        w[v0:v0 + 65536] = rnd((min(65536, N - v0), K), ab, v0 + 2, 2.0 / math.sqrt(K))
        x[:, v0:v0 + 65536], dx[:, v0:v0 + 65536] = logits64(a, w[v0:v0 + 65536])
    targets = targets_of(M, N, 2)
    targets[1], targets[2] = N - 1, (1 << 31) // K
    q, real = one_hot(targets, N)
    loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
    check_loss(loss, lse, x, dx, q, torch.zeros_like(q), real, 1.0)
    dloss = rnd((M,), F32, 5)
    dA, dB = torch.full((M, K), math.nan, dtype=ab, device="cuda"), torch.full(B.shape, math.nan, dtype=ab, device="cuda")
    loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K, layout)
    lse64, A = torch.logsumexp(x, 1), a.double()
    want, size64, tol = (torch.zeros((M, K), dtype=torch.float64, device="cuda") for _ in range(3))
    got_b = dB if layout == R.col_major else dB.t()
    for v0 in range(0, N, 65536):
        at = slice(v0, min(v0 + 65536, N))
        dz, err = slopes64(x[:, at], dx[:, at], lse64, dx.max(1)[0], q[:, at], real, dloss, ab)
        W = w[at].double()
        want += dz @ W
        tol += err @ W.abs()
        size64 += (dz.abs() + err) @ W.abs()
        want_b = dz.t() @ A
        tol_b = err.t() @ A.abs() + (M + 16) * SUM * ((dz.abs() + err).t() @ A.abs())
        within(got_b[at], want_b, tol_b + UNIT[ab] * (want_b.abs() + tol_b) + LEAST[ab], f"dB from {v0} on")
    tol += (N + 16) * SUM * size64
    within(dA, want, tol + UNIT[ab] * (want.abs() + tol) + LEAST[ab], "dA")


def test_logits_past_32_bits(loader):
    """More than 2^32 logits: rows that go together for their statistics, and pieces of their gradient."""
    M, N, K, ab = 70001, 66000, 64, F16
    assert M * N > 1 << 32
    a, w, B = problem(M, N, K, ab, R.col_major, 1)
    targets = targets_of(M, N, 2)
    targets[-1] = N - 1
    dloss = torch.where(rnd((M,), F32, 5) > 0, 1.0, -0.5)  # (of one size, so that f16's least number counts for nothing)
    loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K)
    dA, dB = torch.full((M, K), math.nan, device="cuda"), torch.full((N, K), math.nan, device="cuda")
    loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K)
    want_b, tol_b, size_b = (torch.zeros((N, K), dtype=torch.float64, device="cuda") for _ in range(3))
    W = w.double()
    for row in range(0, M, 4096):
        at = slice(row, min(row + 4096, M))
        x, dx = logits64(a[at], w)
        q, real = one_hot(targets[at], N)
        check_loss(loss[at], lse[at], x, dx, q, torch.zeros_like(q), real, 1.0)
        dz, err = slopes64(x, dx, torch.logsumexp(x, 1), dx.max(1)[0], q, real, dloss[at], ab)
        err = err + 2.0 ** -38 * real[:, None]
        want, A = dz @ W, a[at].double()
        tol = err @ W.abs() + (N + 16) * SUM * ((dz.abs() + err) @ W.abs())
        within(dA[at], want, tol + UNIT[F32] * (want.abs() + tol) + LEAST[F32], f"dA from {row} on")
        want_b += dz.t() @ A
        tol_b += err.t() @ A.abs()
        size_b += (dz.abs() + err).t() @ A.abs()
    tol_b += (M + 16) * SUM * size_b
    within(dB, want_b, tol_b + UNIT[F32] * (want_b.abs() + tol_b) + LEAST[F32], "dB")


@pytest.mark.parametrize("layout", [R.col_major, R.row_major], ids=_id)
@pytest.mark.parametrize("size", [(3, 2100001, 40), (100, 2200000, 24)], ids=_id)
def test_vocabularies_of_more_than_two_million(loader, size, layout):
    """Rows of 2^21 logits and more, which are too long for the tiles' offsets."""
    (M, N, K), ab = size, BF16
    a, w, B = problem(M, N, K, ab, layout, 1)
    targets, dloss = targets_of(M, N, 2), rnd((M,), F32, 5)
    targets[-1] = N - 1
    q, real = one_hot(targets, N)
    x, dx = logits64(a, w)
    loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
    check_loss(loss, lse, x, dx, q, torch.zeros_like(q), real, 1.0)
    dA, dB = torch.full((M, K), math.nan, dtype=ab, device="cuda"), torch.full(B.shape, math.nan, dtype=ab, device="cuda")
    loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K, layout)
    check_gradients(dA, dB, a, w, layout, x, dx, q, real, dloss, 1.0)


@pytest.mark.parametrize("ab", [F16, BF16], ids=_id)
@pytest.mark.parametrize("size", [(40, 700, 64), (300, 1000, 72), (1500, 520, 64), (16385, 264, 40)], ids=_id)
def test_whatever_dloss_says_of_rows_that_are_left_out(loader, size, ab):
    """Large, infinite and unset values there change no bit of the gradients."""
    (M, N, K), k = size, 5
    a, w, B = problem(M, N, K, ab, R.col_major, 1)
    dloss = rnd((M,), F32, 5, 1e-4)
    targets = targets_of(M, N, 2)
    entries, teacher = lists_of(M, N, k, 3)
    entries[5::3] = -1
    teacher[7::9] = -math.inf  # (a list without a share)
    loss, lse, picked = torch.empty(M, device="cuda"), torch.empty(M, device="cuda"), torch.empty((M, k), device="cuda")
    out = {}
    for kind in ("target", "list"):
        out_of = ~one_hot(targets, N)[1] if kind == "target" else ~((entries >= 0) & (entries < N) & (teacher > -math.inf)).any(1)
        assert out_of.any() and not out_of.all()
        for said in (0.0, 1.0, 1e8, 3e38, math.inf, math.nan):
            d = torch.where(out_of, torch.full_like(dloss, said), dloss)
            dA, dB = torch.full((M, K), math.nan, dtype=ab, device="cuda"), torch.full((N, K), math.nan, dtype=ab, device="cuda")
            if kind == "target":
                loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K)
                loader.linear_cross_entropy_backward(dA, dB, d, lse, a, B, targets, M, N, K)
            else:
                loader.linear_distillation(loss, lse, picked, a, B, entries, teacher, M, N, K)
                loader.linear_distillation_backward(dA, dB, d, lse, picked, a, B, entries, teacher, M, N, K)
            assert (dA[out_of] == 0).all() and dA.abs().max() > 0
            if said == 0.0:
                out[kind] = dA, dB
            assert torch.equal(dA, out[kind][0]) and torch.equal(dB, out[kind][1]), (kind, said)


@pytest.mark.parametrize("layout", [R.col_major, R.row_major], ids=_id)
def test_gradients_of_a_million_long_rows(loader, layout):
    """2^20 rows of 4096 elements: dA in fp32 would fill the scratch buffer, so the rows go in blocks."""
    M, N, K, ab = 1 << 20, 264, 4096, BF16
    w = rnd((N, K), ab, 2, 2.0 / math.sqrt(K))
    B = w if layout == R.col_major else w.t().contiguous()
    a = torch.empty((M, K), dtype=ab, device="cuda")
    for row in range(0, M, 1 << 16):
        a[row:row + (1 << 16)] = rnd((1 << 16, K), ab, row + 3)
    targets, dloss = targets_of(M, N, 2), rnd((M,), F32, 5)
    loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
    before = rnd(B.shape, F32, 6)
    dA, dB = torch.full((M, K), math.nan, dtype=ab, device="cuda"), torch.full(B.shape, math.nan, dtype=ab, device="cuda")
    alone, added = torch.full_like(dA, math.nan), before.clone()
    loader.linear_cross_entropy_backward(dA, dB, dloss, lse, a, B, targets, M, N, K, layout)
    loader.linear_cross_entropy_backward(alone, None, dloss, lse, a, B, targets, M, N, K, layout)
    assert torch.equal(alone, dA)
    del alone
    loader.linear_cross_entropy_backward(None, added, dloss, lse, a, B, targets, M, N, K, layout, accumulate=True)
    W = w.double()
    want_b, tol_b, size_b = (torch.zeros((N, K), dtype=torch.float64, device="cuda") for _ in range(3))
    for row in range(0, M, 1 << 15):
        at = slice(row, row + (1 << 15))
        x, dx = logits64(a[at], w)
        q, real = one_hot(targets[at], N)
        dz, err = slopes64(x, dx, torch.logsumexp(x, 1), dx.max(1)[0], q, real, dloss[at], ab)
        want, A = dz @ W, a[at].double()
        tol = err @ W.abs() + (N + 16) * SUM * ((dz.abs() + err) @ W.abs())
        within(dA[at], want, tol + UNIT[ab] * (want.abs() + tol) + LEAST[ab], f"dA from {row} on")
        want_b += dz.t() @ A
        tol_b += err.t() @ A.abs()
        size_b += (dz.abs() + err).t() @ A.abs()
    tol_b += (M + 16) * SUM * size_b
    got = (dB, added) if layout == R.col_major else (dB.t(), added.t())
    within(got[0], want_b, tol_b + UNIT[ab] * (want_b.abs() + tol_b) + LEAST[ab], "dB")
    more = (before if layout == R.col_major else before.t()).double()
    within(got[1], want_b + more, tol_b + UNIT[F32] * (want_b.abs() + tol_b) + 2 * E32 * (want_b.abs() + more.abs()) + LEAST[F32], "dB added to")


def test_a_row_that_is_sure_of_its_target_has_no_negative_loss(loader):
    """-log p is 0 or more.  Where the vocabulary is one entry, or all others are far below, the largest logit is the target's: the
    kernels that pick it from the logits they add up (few rows, logits that are written) leave exactly 0, tiles whose target is
    added up on its own are at most the two sums' difference above."""
    for ab in (F16, BF16):
        for M, N, K, layout in ((64, 1, 96, R.col_major), (40, 600, 64, R.row_major), (64, 600, 264, R.col_major),
                                (2000, 1, 520, R.col_major), (2000, 777, 264, R.col_major), (1000, 1000, 136, R.row_major)):
            a, w, B = problem(M, N, K, ab, layout, 1)
            targets = torch.randint(N, (M,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
            a = (w[targets].float() * torch.linspace(25, 90, M, device="cuda")[:, None]).to(ab)
            x, dx = logits64(a, w)
            others = x.scatter(1, targets[:, None], -math.inf).max(1)[0]
            sure = x.gather(1, targets[:, None])[:, 0] - others > 40 + 2 * dx.max(1)[0]  # (e^-40: nothing in fp32)
            assert sure.sum() > M // 2
            loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
            loader.linear_cross_entropy(loss, lse, a, B, targets, M, N, K, layout)
            assert (loss >= 0).all(), (M, N, K, loss.min().item())
            if M <= 64:
                assert (loss[sure] == 0).all(), (M, N, K, loss[sure].max().item())
            else:
                assert (loss[sure] <= 2 * dx.max(1)[0][sure]).all()
            # a list of the one entry is the same distance
            picked = torch.empty((M, 1), device="cuda")
            loader.linear_distillation(loss, lse, picked, a, B, targets[:, None].contiguous(), torch.zeros((M, 1), device="cuda"), M, N, K, layout)
            assert (loss >= 0).all() and (M > 64 and layout == R.col_major or (loss[sure] == 0).all())


def test_gradients_of_lists_in_blocks_of_rows(loader):
    """The states' gradient of 2^20 rows with lists, which goes in two blocks, has the bits of two calls of half of the rows."""
    M, N, K, k, t = 1 << 20, 72, 4096, 3, 2.0
    w = rnd((N, K), BF16, 2, 2.0 / math.sqrt(K))
    a = torch.empty((M, K), dtype=BF16, device="cuda")
    for row in range(0, M, 1 << 16):
        a[row:row + (1 << 16)] = rnd((1 << 16, K), BF16, row + 3)
    entries, teacher = lists_of(M, N, k, 4)
    dloss = rnd((M,), F32, 5)
    loss, lse, picked = torch.empty(M, device="cuda"), torch.empty(M, device="cuda"), torch.empty((M, k), device="cuda")
    for index in (torch.int64, torch.int32):
        listed = entries.to(index)
        loader.linear_distillation(loss, lse, picked, a, w, listed, teacher, M, N, K, temperature=t)
        dA, halves = torch.full((M, K), math.nan, dtype=BF16, device="cuda"), torch.full((M, K), math.nan, dtype=BF16, device="cuda")
        loader.linear_distillation_backward(dA, None, dloss, lse, picked, a, w, listed, teacher, M, N, K, temperature=t)
        for row in (0, M // 2):
            at = slice(row, row + M // 2)
            loader.linear_distillation_backward(halves[at], None, dloss[at], lse[at], picked[at], a[at], w, listed[at], teacher[at], M // 2, N, K,
                                                temperature=t)
        assert torch.isfinite(dA[::4099].float()).all() and torch.equal(dA, halves)
