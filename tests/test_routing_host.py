"""Routing without a GPU: what the C entry points refuse before they touch the device, and what calls would launch."""
import ctypes
import os
import subprocess
import sys

import pytest

import rocm_wmma_gemm_amd as R
from rocm_wmma_gemm_amd import loader as module
from test_operators_host import recorded  # noqa: F401  (a fixture)

ARGUMENT, LIMIT, OK = -2, -5, 0
MOST = (1 << 31) - 256


@pytest.fixture(scope="module")
def library():
    return R.Loader(arch="gfx950")._lib


def routing(score=0, groups=1, kept=1, best=2, renormalize=1, scale=1.0):
    return ctypes.byref(module._RoutingC(score, None, None, groups, kept, best, renormalize, scale))


def test_route_refuses(library):
    p = ctypes.c_void_p(1 << 20)
    route = lambda *a: library.rocm_wmma_gemm_route(*a, None)  # noqa: E731
    assert route(0, p, p, p, None, 4, 8, 2) == ARGUMENT
    assert route(3, p, p, p, routing(), 4, 8, 2) == ARGUMENT  # type
    assert route(0, None, p, p, routing(), 4, 8, 2) == ARGUMENT
    assert route(0, p, None, p, routing(), 4, 8, 2) == ARGUMENT
    assert route(0, p, p, None, routing(), 4, 8, 2) == ARGUMENT
    for bad in (dict(score=2), dict(groups=0), dict(groups=3), dict(groups=2, kept=3), dict(groups=2, kept=0), dict(best=0),
                dict(best=3), dict(renormalize=2), dict(scale=float("inf")), dict(scale=float("nan")), dict(groups=8, kept=1)):
        assert route(0, p, p, p, routing(**bad), 4, 8, 2) == ARGUMENT, bad
    assert route(0, p, p, p, routing(), 4, 8, 9) == ARGUMENT  # more choices than experts
    assert route(0, p, p, p, routing(), 4, 0, 1) == ARGUMENT  # none to choose from
    assert route(0, p, p, p, routing(), 4, 513, 2) == LIMIT
    assert route(0, p, p, p, routing(), 4, 512, 33) == LIMIT
    assert route(0, p, p, p, routing(groups=17), 4, 34, 2) == LIMIT
    assert route(0, p, p, p, routing(), 1 << 30, 8, 2) == LIMIT  # 2^31 choices
    assert route(0, None, None, None, routing(), 0, 8, 2) == OK
    assert route(0, None, None, None, routing(), 4, 8, 0) == OK
    back = lambda *a: library.rocm_wmma_gemm_route_backward(*a, None)  # noqa: E731
    assert back(0, None, p, p, p, 4, 8, 2, 0, 1, 1.0) == ARGUMENT
    assert back(0, p, None, p, p, 4, 8, 2, 0, 1, 1.0) == ARGUMENT
    assert back(0, p, p, p, p, 4, 8, 2, 2, 1, 1.0) == ARGUMENT
    assert back(0, p, p, p, p, 4, 8, 2, 0, 1, float("nan")) == ARGUMENT
    assert back(0, p, p, p, p, 4, 513, 2, 0, 1, 1.0) == LIMIT
    assert back(0, None, None, None, None, 0, 8, 2, 0, 1, 1.0) == OK


def test_dispatch_and_combine_refuse(library):
    p = ctypes.c_void_p(1 << 20)
    dispatch = lambda *a: library.rocm_wmma_gemm_dispatch(*a, None)  # noqa: E731
    assert dispatch(3, p, p, p, p, p, 8, 4, 16, 2) == ARGUMENT
    assert dispatch(0, p, None, p, p, p, 8, 4, 16, 2) == ARGUMENT
    assert dispatch(0, p, p, None, p, p, 8, 4, 16, 2) == ARGUMENT
    assert dispatch(0, p, p, p, None, p, 8, 4, 16, 2) == ARGUMENT
    assert dispatch(0, p, p, p, p, None, 8, 4, 16, 2) == ARGUMENT
    assert dispatch(0, p, p, p, p, p, 513, 4, 16, 2) == LIMIT
    assert dispatch(0, p, p, p, p, p, 8, 4, 16, 33) == LIMIT
    assert dispatch(0, p, p, p, p, p, 8, 1 << 30, 16, 2) == LIMIT
    combine = lambda *a: library.rocm_wmma_gemm_combine(*a, None)  # noqa: E731
    assert combine(0, 1, p, p, p, p, None, 4, 16, 2) == ARGUMENT  # f16 rows, bf16 sum
    assert combine(2, 0, p, p, p, p, None, 4, 16, 2) == ARGUMENT
    assert combine(0, 0, None, p, p, p, None, 4, 16, 2) == ARGUMENT
    assert combine(0, 0, p, None, p, p, None, 4, 16, 2) == ARGUMENT
    assert combine(0, 0, p, p, None, p, None, 4, 16, 2) == ARGUMENT
    assert combine(0, 0, p, p, p, p, None, 4, 16, 33) == LIMIT
    assert combine(0, 0, None, None, None, None, None, 0, 16, 2) == OK
    back = lambda *a: library.rocm_wmma_gemm_combine_backward(*a, None)  # noqa: E731
    assert back(0, 1, p, p, p, p, p, p, 4, 16, 2) == ARGUMENT
    assert back(0, 0, p, p, None, p, p, p, 4, 16, 2) == ARGUMENT
    assert back(0, 0, p, p, p, None, p, p, 4, 16, 2) == ARGUMENT  # the weights' gradient reads the rows
    assert back(0, 0, p, p, p, p, None, p, 4, 16, 2) == ARGUMENT
    assert back(0, 0, None, None, p, p, p, p, 4, 16, 2) == OK  # nothing wanted
    assert back(0, 0, p, p, p, p, p, p, 1 << 30, 16, 2) == LIMIT


def test_every_launch_of_routing_fits_the_grid(recorded):  # noqa: F811
    calls = []
    for m, n, k in ((1, 1, 1), (MOST, 1, 1), (MOST // 32, 8, 32), (MOST // 2, 4096, 2), (3, MOST, 8), (5, MOST - 1, 2), (1 << 20, 64, 8)):
        for kind in (0, 2):
            calls.append(["dispatch", [kind, "p", "p", "p", "p", "p", 512, m, n, k, None]])
            calls.append(["combine", [kind, 2, "p", "p", "p", "p", "p", m, n, k, None]])
            calls.append(["combine_backward", [kind, kind, "p", "p", "p", "p", "p", "p", m, n, k, None]])
        calls.append(["route_backward", [0, "p", "p", "p", "p", m, 512, k, 0, 1, 1.0, None]])
    for call, (status, launches) in zip(calls, recorded(*calls)):
        assert status == 0 and launches, (call, status, launches)
        assert not any(failed for *_, failed in launches), (call, launches)


def test_nothing_of_a_dispatch_follows_a_launch_that_failed(recorded):  # noqa: F811
    # few choices, a table of counts that every workgroup adds up, one that is added up by a launch of its own
    for m, e, steps in ((1000, 64, 1), (5000, 64, 2), (70000, 512, 3)):
        call = ["dispatch", [1, "p", "p", "p", "p", "p", e, m, 64, 4, None]]
        (status, whole), = recorded(call)
        assert status == 0 and len(whole) == steps
        for n in range(steps):
            (status, launches), = recorded(["fail", n], call)
            assert status == -4 and len(launches) == n + 1


ROUTES = """
import ctypes, sys
recorder = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path[:0] = sys.argv[2:]
import rocm_wmma_gemm_amd as R
from recorded_launches import Launch
from rocm_wmma_gemm_amd import loader
library, p = R.Loader(arch="gfx950")._lib, ctypes.c_void_p(1 << 20)
for m, e, k, groups in ((1, 1, 1, 1), ((1 << 31) - 256, 512, 1, 16), (5, 504, 32, 9), (1 << 26, 512, 31, 1)):
    how = loader._RoutingC(1, None, None, groups, groups, 2, 1, 1.0)
    assert library.rocm_wmma_gemm_route(2, p, p, p, ctypes.byref(how), m, e, k, None) == 0
    seen = (Launch * 16)()
    assert recorder.recorder_take(seen, 16) == 1 and not seen[0].failed, (m, list(seen[0].grid))
print("all fit")
"""


def test_every_launch_of_route_fits_the_grid(tmp_path):
    here = os.path.dirname(os.path.abspath(__file__))
    so = tmp_path / "recorder.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(here, "hip_recorder.cpp"), "-o", str(so)], check=True)
    r = subprocess.run([sys.executable, "-c", ROUTES, str(so), os.path.dirname(here), here], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "all fit" in r.stdout, r.stdout + r.stderr
