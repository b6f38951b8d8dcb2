"""The layer products without a GPU: what the compiler made of the hand-placed loop, and what the
C entry points refuse before they touch the device."""
import ctypes
import os
import re
import subprocess

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
