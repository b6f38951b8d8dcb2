"""The losses of a projection without a GPU: what the C entry points refuse before they touch the device, and what calls
would launch."""
import ctypes
import os
import re
import subprocess

import pytest

import rocm_wmma_gemm_amd as R
from test_host import ROOT, _mfma_loops
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
    for temperature in (0.0, -1.0, nan, inf, 1e-45, 4.2e-39):
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
            assert status == 0 and len(whole) >= 4  # (two copies, the product, the join)
            for n in range(0, len(whole), 3):
                (status, launches), = recorded(["fail", n], call)
                assert status == -4 and len(launches) == n + 1, (call[0], n)


def test_the_logits_of_a_large_vocabulary_are_not_kept(recorded):  # noqa: F811
    """2^19 rows over 2^17 entries (137 GB of logits in 16 bits) go in pieces that the scratch buffer holds: the loss in
    33 blocks of rows (256 MB of statistics, 8 bytes for 64 columns, hold 16376 rows) of three launches each, the
    gradient in at least as many pieces of columns as 512 MB hold 1024 of them, 128, of three."""
    for call in calls_of(1, 1 << 19, 1 << 17, 64, 1):
        (status, launches), = recorded(call)
        assert status == 0 and len(launches) >= (128 * 2 if "backward" in call[0] else 3 * 33)


def test_tiled_products_behind_a_loss_keep_accumulators_in_place(tmp_path):
    """As for the layers' (test_operators_host.py): no accumulator copies and no spills in the MFMA loops, and behind every MFMA
    that a path leaves the loop from two s_nop 15 before anything names an accumulator."""
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    asm = tmp_path / "loss_isa.s"
    subprocess.run([hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I" + os.path.join(ROOT, "rocm_wmma_gemm_amd", "csrc"), "-S", "--cuda-device-only", "-o", str(asm),
                    os.path.join(ROOT, "tests", "loss_isa.hip")], check=True, capture_output=True, timeout=900)
    text = asm.read_text()
    loops = {}
    for f, body in _mfma_loops(text):
        if "tiled_product" in f and (f not in loops or len(body) < len(loops[f])):
            loops[f] = body
    assert len(loops) == 12
    for func, body in loops.items():
        whole = text[text.index(func + ":"):]
        whole = whole[:whole.index(".Lfunc_end")]
        expected = 32 if "Li128ELi128E" in func else 64 if "Li128ELi256E" in func else 128
        assert sum("v_mfma_f32_16x16x32" in b for b in body) == whole.count("v_mfma_f32_16x16x32") == expected, func
        assert not [b for b in body if re.search(r"v_accvgpr_|scratch_", b)] and "scratch_" not in whole, func
        lines = whole.split("\n")
        label_at = {m.group(1): n for n, line in enumerate(lines) if (m := re.match(r"^(\.LBB\w+):", line))}
        seen, checked, todo = set(), 0, [(n + 1, 0) for n, line in enumerate(lines) if "v_mfma" in line]
        while todo:
            n, nops = todo.pop()
            while n < len(lines) and (n, nops) not in seen:
                seen.add((n, nops))
                line = lines[n]
                if "v_mfma" in line or "s_endpgm" in line:
                    break
                nops += "s_nop 15" in line
                if nops >= 2:
                    checked += 1
                    break
                assert not re.search(r"[ ,]a\[?\d", line), f"{func}: {line.strip()} too early after the MFMAs"
                m = re.match(r"^\s+s_(c?)branch\w*\s+(\.LBB\w+)", line)
                if m:
                    todo.append((label_at[m.group(2)], nops))
                    if not m.group(1):
                        break
                n += 1
        assert checked >= 1, func


def test_only_copies_of_operands_are_more_than_the_scratch_buffer_holds(recorded):  # noqa: F811
    """Sizes up to the documented ones are launched, a gradient of 2^20 rows of 4096 and more elements in blocks of rows.  Only operands
    whose rows do not start on 16 bytes, and whose copies take more than 16 GiB, are refused, before anything is launched."""
    most = (1 << 31) - 256
    for m, n, k in ((1, 1, 1), (300, 1001, 77), (4096, 131072, 4096), (1, most, 8), (3, 1 << 27, 3), (1 << 20, 5000, 8), (1 << 20, 40000, 16),
                    (1 << 20, 264, 4096), (1 << 20, 32000, 4096), (1 << 19, 32000, 8192), (1 << 20, 128, 8192), (1 << 20, 1000, 4095),
                    (1 << 16, 131072, 16384), (2, 8, most), (64, 1000, 1 << 26), (1, 1, most), (1 << 20, 128, 8201), (1 << 19, 72, 16385)):
        calls, large = [], []
        for kind, layout in ((0, 0), (1, 1)):
            calls += calls_of(kind, m, n, k, layout)
            padded = lambda rows, length: rows * ((length + 7) // 8) * 16 if length % 8 else 0  # noqa: E731
            copied = padded(m, k) + (padded(k, n) if layout == 0 else padded(n, k))
            # (a gradient of the states alone goes in blocks of rows: half of the states' copies at a time, or less)
            alone = padded(m // 4, k) + (padded(k, n) if layout == 0 else padded(n, k))
            large += [copied > 1 << 34] * 3 + [alone > 1 << 34] + [copied > 1 << 34]
        for call, refused, (status, launches) in zip(calls, large, recorded(*calls)):
            assert (status, bool(launches)) == ((SCRATCH, False) if refused else (OK, True)), (call, status, len(launches))
            assert not any(failed for *_, failed in launches), (call, launches)


def test_nothing_of_a_gradient_in_blocks_follows_a_launch_that_failed(recorded):  # noqa: F811
    for call in calls_of(1, 1 << 20, 264, 4096, 1)[1::2]:
        (status, whole), = recorded(call)
        assert status == OK and len(whole) >= 14  # (of every block: the unit, records, logits, dA's product, its rounding; more of lists)
        for n in range(0, len(whole), 5):
            (status, launches), = recorded(["fail", n], call)
            assert status == -4 and len(launches) == n + 1, (call[0], n)
