"""The losses of a projection without a GPU: what the C entry points refuse before they touch the device, and what calls
would launch."""
import ctypes

import pytest

import rocm_wmma_gemm_amd as R
from test_operators_host import recorded  # noqa: F401  (a fixture)

ARGUMENT, SCRATCH, LIMIT, OK = -2, -3, -5, 0


@pytest.fixture(scope="module")
def library():
    return R.Loader(arch="gfx950")._lib


def test_losses_refuse(library):
    p, nan, inf = ctypes.c_void_p(1 << 20), float("nan"), float("inf")
    loss = lambda *a: library.rocm_wmma_gemm_linear_cross_entropy(*a, None)  # noqa: E731
    assert loss(2, p, p, p, p, p, 0, 4, 16, 8, 1) == ARGUMENT  # fp32 operands
    assert loss(0, None, p, p, p, p, 0, 4, 16, 8, 1) == ARGUMENT
    assert loss(0, p, None, p, p, p, 0, 4, 16, 8, 1) == ARGUMENT
    assert loss(0, p, p, None, p, p, 0, 4, 16, 8, 1) == ARGUMENT
    assert loss(0, p, p, p, None, p, 0, 4, 16, 8, 1) == ARGUMENT
    assert loss(0, p, p, p, p, None, 0, 4, 16, 8, 1) == ARGUMENT
    assert loss(0, p, p, p, p, p, 2, 4, 16, 8, 1) == ARGUMENT  # index width
    assert loss(0, p, p, p, p, p, 0, 4, 16, 8, 2) == ARGUMENT  # layout
    assert loss(0, p, p, p, p, p, 0, (1 << 20) + 1, 16, 8, 1) == LIMIT
    assert loss(0, p, p, p, p, p, 0, 4, 1 << 31, 8, 1) == LIMIT
    assert loss(0, p, p, p, p, p, 0, 4, 16, (1 << 31) - 255, 1) == LIMIT
    assert loss(0, None, None, None, None, None, 0, 0, 16, 8, 1) == OK
    back = lambda *a: library.rocm_wmma_gemm_linear_cross_entropy_backward(*a, None)  # noqa: E731
    assert back(4, p, p, p, p, p, p, p, 0, 4, 16, 8, 1, 0) == ARGUMENT
    assert back(0, p, p, p, p, p, p, p, 0, 4, 16, 8, 1, 2) == ARGUMENT
    assert back(0, p, p, None, p, p, p, p, 0, 4, 16, 8, 1, 0) == ARGUMENT
    assert back(0, p, p, p, None, p, p, p, 0, 4, 16, 8, 1, 0) == ARGUMENT
    assert back(0, p, p, p, p, p, None, p, 0, 4, 16, 8, 1, 0) == ARGUMENT
    assert back(0, None, None, p, p, p, p, p, 0, 4, 16, 8, 1, 0) == OK  # nothing wanted
    far = lambda *a: library.rocm_wmma_gemm_linear_distillation(*a, None)  # noqa: E731
    for temperature in (0.0, -1.0, nan, inf, 1e-45):
        assert far(0, p, p, p, p, p, p, 0, p, 4, 16, 8, 2, temperature, 1) == ARGUMENT
    assert far(0, p, p, None, p, p, p, 0, p, 4, 16, 8, 2, 1.0, 1) == ARGUMENT
    assert far(0, p, p, p, p, p, p, 0, None, 4, 16, 8, 2, 1.0, 1) == ARGUMENT
    assert far(0, p, p, p, p, p, p, 0, p, 4, 16, 8, 0, 1.0, 1) == ARGUMENT
    assert far(0, p, p, p, p, p, p, 0, p, 4, 16, 8, 257, 1.0, 1) == LIMIT
    gone = lambda *a: library.rocm_wmma_gemm_linear_distillation_backward(*a, None)  # noqa: E731
    assert gone(0, p, p, p, p, None, p, p, p, 0, p, 4, 16, 8, 2, 1.0, 1, 0) == ARGUMENT
    assert gone(5, p, p, p, p, p, p, p, p, 0, p, 4, 16, 8, 2, 1.0, 1, 0) == ARGUMENT


def calls_of(kind, m, n, k, layout, entries=8):
    """Both directions of both losses."""
    pair = {0: 0, 1: 2}[kind]
    return [["linear_cross_entropy", [kind, "p", "p", "p", "p", "p", 1, m, n, k, layout, None]],
            ["linear_cross_entropy_backward", [pair, "p", "p", "p", "p", "p", "p", "p", 1, m, n, k, layout, 0, None]],
            ["linear_distillation", [kind, "p", "p", "p", "p", "p", "p", 0, "p", m, n, k, entries, 2.0, layout, None]],
            ["linear_distillation_backward",
             [pair + 1, "p", None, "p", "p", "p", "p", "p", "p", 0, "p", m, n, k, entries, 2.0, layout, 1, None]],
            ["linear_distillation_backward",
             [pair + 1, None, "p", "p", "p", "p", "p", "p", "p", 0, "p", m, n, k, entries, 2.0, layout, 1, None]]]


def test_every_launch_of_a_loss_fits_the_grid(recorded):  # noqa: F811
    most = (1 << 31) - 256
    calls = []
    for m, n, k in ((1, 1, 1), (1, most, 8), (3, 1 << 27, 3), (1 << 20, 5000, 8), (1 << 20, 3, 1 << 12), (1 << 20, 40000, 16), (7, 8, 1 << 24),
                    (4096, 131072, 4096), (1, 1, most), (300, 1001, 77), (0, 16, 8), (5, 0, 8), (5, 16, 0)):
        for kind, layout in ((0, 0), (0, 1), (1, 0), (1, 1)):
            calls += calls_of(kind, m, n, k, layout)
    for call, (status, launches) in zip(calls, recorded(*calls)):
        # (-3: more scratch memory than there may be; nothing is launched then)
        assert status == 0 or status == SCRATCH and not launches, (call, status, launches[:3])
        assert not any(failed for *_, failed in launches), (call, launches)


def test_nothing_of_a_loss_follows_a_launch_that_failed(recorded):  # noqa: F811
    for kind in (0, 1):
        for call in calls_of(kind, 20000, 3001, 77, 0):
            (status, whole), = recorded(call)
            assert status == 0 and len(whole) >= 5
            for n in range(0, len(whole), 3):
                (status, launches), = recorded(["fail", n], call)
                assert status == -4 and len(launches) == n + 1, (call[0], n)


def test_the_logits_of_a_large_vocabulary_are_not_kept(recorded):  # noqa: F811
    """2^19 rows over 2^17 entries (137 GB of logits in 16 bits) go in pieces that the scratch buffer holds."""
    for call in calls_of(1, 1 << 19, 1 << 17, 64, 1):
        (status, launches), = recorded(call)
        assert status == 0 and len(launches) > 100
