"""The layer products without a GPU: what the compiler made of the hand-placed loop, and what the
C entry points refuse before they touch the device."""
import ctypes
import json
import os
import re
import subprocess
import sys

import pytest

import rocm_wmma_gemm_amd as R
from test_host import ROOT, _mfma_loops

INSTANTIATED = 17


def test_tiled_products_keep_accumulators_in_place(tmp_path):
    """The MFMAs are inline assembly, so the compiler does not know when their results become
    readable: the loop must hold no accumulator copies and no spills, and behind it nothing may
    name an accumulator before the explicit wait states."""
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    asm = tmp_path / "product_isa.s"
    cmd = [hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature",
           "-Xclang", "-packed-fp32-ops", "-I" + os.path.join(ROOT, "rocm_wmma_gemm_amd", "csrc"),
           "-S", "--cuda-device-only", "-o", str(asm), os.path.join(ROOT, "tests", "product_isa.hip")]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    text = asm.read_text()
    loops = {}
    for f, body in _mfma_loops(text):
        if "tiled_product" in f and (f not in loops or len(body) < len(loops[f])):
            loops[f] = body
    assert len(loops) == INSTANTIATED
    for func, body in loops.items():
        whole = text[text.index(func + ":"):]
        whole = whole[:whole.index(".Lfunc_end")]
        expected = 32 if "Li128ELi128E" in func else 64 if "Li128ELi256E" in func else 72 if "Li192E" in func else 128
        assert sum("v_mfma_f32_16x16x32" in b for b in body) == whole.count("v_mfma_f32_16x16x32") == expected, func
        bad = [b for b in body if re.search(r"v_accvgpr_|scratch_", b)]
        assert not bad, f"{func}: accumulator traffic or spills inside the MFMA loop: {bad[:3]}"
        assert "scratch_" not in whole, f"{func}: spills"
        lines = whole.split("\n")
        label_at = {m.group(1): n for n, line in enumerate(lines) if (m := re.match(r"^(\.LBB\w+):", line))}
        seen, checked = set(), 0
        todo = [(n + 1, 0) for n, line in enumerate(lines) if "v_mfma" in line]
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


@pytest.fixture(scope="module")
def library():
    return R.Loader(arch="gfx950")


def test_entry_points_refuse_before_they_touch_the_device(library):
    """Arguments out of range, missing operands and sizes beyond the limits are status codes, asked
    of the C functions themselves, without a device."""
    L, one = library._lib, ctypes.c_void_p(16)
    epilogue = lambda act: ctypes.byref(loader_module()._EpilogueC(None, None, None, act))  # noqa: E731
    ERR_ARGUMENT, ERR_LIMIT, OK = -2, -5, 0
    linear = lambda *a: L.rocm_wmma_gemm_linear(*a, None)  # noqa: E731
    assert linear(4, one, one, one, 8, 8, 8, 1, None) == ERR_ARGUMENT  # type pair
    assert linear(0, one, one, one, 8, 8, 8, 2, None) == ERR_ARGUMENT  # layout
    assert linear(0, one, one, one, 8, 8, 8, 1, epilogue(4)) == ERR_ARGUMENT  # activation
    assert linear(0, one, one, one, 1 << 31, 8, 8, 1, None) == ERR_LIMIT
    assert linear(0, one, one, one, 8, 8, (1 << 31) - 255, 1, None) == ERR_LIMIT  # (its tiles' end leaves an int)
    assert linear(0, None, one, one, 8, 8, 8, 1, None) == ERR_ARGUMENT
    assert linear(0, one, one, None, 8, 8, 8, 1, None) == ERR_ARGUMENT
    assert linear(0, None, None, None, 0, 8, 8, 1, None) == OK  # nothing to do
    grouped = lambda *a: L.rocm_wmma_gemm_grouped(*a, None)  # noqa: E731
    assert grouped(0, one, one, one, None, 4, 8, 8, 8, 1, None) == ERR_ARGUMENT  # no offsets
    assert grouped(0, one, one, one, one, 513, 8, 8, 8, 1, None) == ERR_LIMIT
    assert grouped(0, one, one, one, None, 0, 8, 8, 8, 1, None) == OK
    backward = lambda *a: L.rocm_wmma_gemm_linear_backward(*a, None)  # noqa: E731
    assert backward(0, one, None, None, None, one, one, None, 8, 8, 8, 1, 0, 0) == ERR_ARGUMENT  # no dC
    assert backward(0, one, None, None, one, one, None, None, 8, 8, 8, 1, 0, 0) == ERR_ARGUMENT  # dA without B
    assert backward(0, None, one, None, one, None, one, None, 8, 8, 8, 1, 0, 0) == ERR_ARGUMENT  # dB without A
    assert backward(0, one, None, None, one, one, one, None, 8, 8, 8, 1, 2, 0) == ERR_ARGUMENT  # no preact
    assert backward(0, one, None, None, one, one, one, None, 8, 8, 8, 1, 7, 0) == ERR_ARGUMENT
    steps = (ctypes.c_float * 3)(1.5, -0.5, 0.0)
    orth = lambda *a: L.rocm_wmma_gemm_orthogonalize(*a, None)  # noqa: E731
    assert orth(3, 0, one, one, 8, 8, 1, 5, steps, 1e-7) == ERR_ARGUMENT  # G's type
    assert orth(0, 2, one, one, 8, 8, 1, 5, steps, 1e-7) == ERR_ARGUMENT  # O's type
    assert orth(0, 0, one, one, 8, 8, 1, 0, steps, 1e-7) == ERR_ARGUMENT  # no step
    assert orth(0, 0, one, one, 8, 8, 1, 5, None, 1e-7) == ERR_ARGUMENT
    assert orth(0, 0, None, one, 8, 8, 1, 5, steps, 1e-7) == ERR_ARGUMENT
    assert orth(0, 0, one, one, (1 << 20) + 1, 8, 1, 5, steps, 1e-7) == ERR_LIMIT
    assert orth(0, 0, None, None, 0, 8, 1, 5, steps, 1e-7) == OK


def loader_module():
    from rocm_wmma_gemm_amd import loader

    return loader


def test_product_plans(library):
    """What the estimate picks follows the sizes: few rows stream a weight, many take large tiles,
    a long K with few tiles is cut, and rows that do not start on 16 bytes are copied or staged."""
    pick = library.product_select
    assert pick("forward", 1, 4096, 4096).block_m <= 32
    large = pick("forward", 8192, 8192, 4096)
    assert (large.block_m, large.block_n, large.copies, large.cut_tail) == (256, 256, 0, 0)
    assert pick("forward", 2048, 1024, 16384).cut_tail == 1
    assert pick("forward", 16, 8192, 8192).once == 1 and pick("forward", 16, 4096, 4096).once == 0
    assert pick("forward", 2048, 4096, 4001).copies == 3  # K-contiguous rows of 4001: A and B
    assert pick("forward", 2048, 4096, 4001, layout_b=R.row_major).copies == 1
    assert pick("gradient_b", 2048, 4001, 4096, layout_b=R.row_major).copies == 0  # dZ is written padded
    assert pick("forward", 1, 520, 999, groups=64).form in (0, 1)
    with pytest.raises(R.GemmLibraryError):
        pick("forward", 0, 8, 8)
    with pytest.raises(R.GemmLibraryError):
        pick("forward", 8, 8, 8, groups=513)


@pytest.fixture(scope="module")
def product_checks(tmp_path_factory):
    out = tmp_path_factory.mktemp("products") / "product_checks"
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "rocm_wmma_gemm_amd", "csrc"),
                    os.path.join(ROOT, "tests", "product_checks.cpp"), "-o", str(out)], check=True)
    return str(out)


def test_every_slice_of_a_cut_tile_lies_in_its_sum(product_checks):
    r = subprocess.run([product_checks, "cuts"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


def test_every_tile_of_a_symmetric_product_is_written_once(product_checks):
    r = subprocess.run([product_checks, "triangle"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.fixture(scope="module")
def recorded(tmp_path_factory):
    """What calls would launch: a function of [entry point, arguments] pairs (recorded_launches.py)."""
    so = tmp_path_factory.mktemp("recorder") / "recorder.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(ROOT, "tests", "hip_recorder.cpp"), "-o",
                    str(so)], check=True)

    def ask(*calls):
        r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "recorded_launches.py"), str(so), json.dumps(calls)],
                           capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout + r.stderr
        return json.loads(r.stdout.strip().split("\n")[-1])

    return ask


MOST = (1 << 31) - 256  # the largest extent that the entry points take


def test_every_launch_fits_the_grid(recorded):
    """Sizes up to the documented limits launch what HIP takes: fewer than 2^32 threads along x, at most 65535
    workgroups along y."""
    calls = []
    for m, n, k in ((1, 1, 1), (1 << 29, 8, 8), (MOST, 8, 8), (MOST, 4, 8), (3, MOST, 8), (3, MOST - 1, 1), (8, 8, MOST),
                    (1 << 24, 64, 64), (MOST, 1, 1)):
        calls.append(["linear", [2, "p", "p", "p", m, n, k, 1, None, None]])
        calls.append(["linear", [0, "p", "p", "p", m, n, k, 0, None, None]])
        calls.append(["grouped", [2, "p", "p", "p", "p", 512, m, n, k, 1, None, None]])
    for m, n, k in ((1 << 24, 8, 8), (1 << 29, 8, 8), (MOST, 8, 8), (3, 5 << 20, 8), (3, 1 << 28, 8)):
        for act in (0, 2):
            for wanted in (("p", None, None), (None, "p", None), (None, None, "p"), ("p", "p", "p")):
                calls.append(["linear_backward", [3, *wanted, "p", "p", "p", "p", m, n, k, 1, act, 0, None]])
                calls.append(["grouped_backward", [3, *wanted, "p", "p", "p", "p", "p", 4, m, n, k, 0, act, 1, None]])
    for m, n, batch in ((1, 1, 65535), (64, 256, 65535), (100, 70, 65535), (1 << 20, 8, 3), (1 << 20, 65, 1), (65, 1 << 20, 1)):
        calls.append(["orthogonalize", [2, 1, "p", "p", m, n, batch, 5, "s", 1e-7, None]])
    for call, (status, launches) in zip(calls, recorded(*calls)):
        # (-3: more scratch memory than there may be; nothing is launched then)
        assert status == 0 and launches or status == -3 and not launches, (call, status, launches)
        assert not any(failed for *_, failed in launches), (call, launches)


def test_nothing_follows_a_launch_that_failed(recorded):
    """A kernel that reads what a rejected one was to write is not launched: the results stay as they were."""
    for call in (["linear_backward", [2, "p", "p", "p", "p", "p", "p", "p", 300, 512, 256, 1, 2, 0, None]],
                 ["grouped_backward", [2, "p", "p", "p", "p", "p", "p", "p", "p", 4, 300, 512, 256, 1, 2, 1, None]],
                 ["linear", [2, "p", "p", "p", 2048, 4096, 4001, 1, None, None]],  # copies of A and B first
                 ["orthogonalize", [2, 1, "p", "p", 300, 200, 2, 2, "s", 1e-7, None]]):
        (status, whole), = recorded(call)
        assert status == 0 and len(whole) >= 2
        for n in range(len(whole)):
            (status, launches), = recorded(["fail", n], call)
            assert status == -4 and len(launches) == n + 1, (call, n, launches)


def test_a_large_batch_of_updates_goes_in_parts(recorded):
    """More matrices than the scratch buffer may hold (16 GiB) go in parts of one size, each the launches of a
    batch; one matrix past it is refused."""
    one = lambda batch, m=4096, n=8192: ["orthogonalize", [2, 1, "p", "p", m, n, batch, 2, "s", 1e-7, None]]  # noqa: E731
    (rc, alone), (rc64, all64), (rc65, all65), (refused, none) = recorded(one(32), one(64), one(65), one(1, 1 << 18, 1 << 14))
    assert (rc, rc64, rc65) == (0, 0, 0)
    assert len(all64) == 2 * len(alone) and len(all65) == 2 * len(alone)
    assert [x[1] for x in all64[:2]] == [32, 32] and [x[1] for x in all65[:1] + all65[len(alone):len(alone) + 1]] == [33, 32]
    assert (refused, none) == (-3, [])


def test_plans_of_an_update(library):
    """The products of an update's steps are described like a layer's; small matrices stay in one workgroup."""
    pick = lambda part, m, n, batch: library.product_select(part, m, n, 0, batch)  # noqa: E731
    for part in ("steps_s", "steps_q", "steps_x", "steps_last"):
        assert pick(part, 64, 256, 7).form == 14 and pick(part, 256, 64, 1).form == 14
        assert pick(part, 64, 257, 1).form != 14
        assert pick(part, 300, 200, 2) == pick(part, 200, 300, 2)  # a tall matrix is transposed
        for m, n, batch in ((0, 8, 1), (8, 0, 1), (8, 8, 0), ((1 << 20) + 1, 8, 1), (8, 8, 65536)):
            with pytest.raises(R.GemmLibraryError):
                pick(part, m, n, batch)
    large = pick("steps_s", 4096, 4096, 1)
    assert (large.block_m, large.block_n) == (192, 192) and pick("steps_x", 4096, 4096, 1).block_m == 256


def test_the_bias_alone_needs_no_dz(recorded):
    """dbias without dA and dB is answered where dZ itself (34 GB here) would pass the scratch buffer."""
    bias_only = lambda n, act: ["linear_backward", [2, None, None, "p", "p", None, None, "p", 1 << 28, n, 8, 1, act, 0, None]]  # noqa: E731
    for status, launches in recorded(bias_only(64, 2), bias_only(63, 0)):
        assert status == 0 and len(launches) >= 2, (status, launches)
