"""Python mirror of ``rocm_wmma_gemm::loader``.

Reference interface: rocm_wmma_gemm/include/rocm_wmma_gemm/kernel_loader.hpp:51-182
 - library name ``librocm_wmma_gemm_<arch>.so`` with ``<arch>`` taken from device 0's
   architecture string cut at the first ':' (:74-91);
 - search order: the configured library directory first, then the dynamic linker's
   own path (:93-102);
 - the four ``rocm_wmma_gemm_<Ctype>_<ABtype>`` symbols are resolved eagerly and a
   missing library or symbol raises (:104-113) -- here ``GemmLibraryError``;
 - ``gemm`` takes (C, A, B, M, N, K[, batch_count], stream) with the layouts in
   C, A, B order and passes the ADDRESS of the stream handle (:138-154).

There is no CPU fallback: if the library cannot be loaded every call fails.
"""
from __future__ import annotations

import ctypes
import enum
import os
import subprocess
from dataclasses import dataclass

_HERE = os.path.dirname(os.path.abspath(__file__))
_DEFAULT_LIB_DIR = os.path.join(_HERE, "lib")

ENTRY_SUFFIXES = ("f16_f16", "f32_f16", "bf16_bf16", "f32_bf16")

# status codes and the fixed scratch size of include/rocm_wmma_gemm_c.h
OK, ERR_VARIANT, ERR_ARGUMENT, ERR_SCRATCH, ERR_RUNTIME, ERR_LIMIT = 0, -1, -2, -3, -4, -5
NOALLOC_SCRATCH_BYTES = 64 << 20


class GemmLibraryError(RuntimeError):
    """Library or symbol could not be loaded (the C++ loader throws std::runtime_error)."""


class m_layout(enum.IntEnum):
    row_major = 0
    col_major = 1


row_major = m_layout.row_major
col_major = m_layout.col_major


class activation(enum.IntEnum):
    """What a linear layer applies to its sums (the codes of include/rocm_wmma_gemm_c.h)."""

    none = 0
    relu = 1
    silu = 2  # x / (1 + e^-x)
    gelu = 3  # the tanh form


class score(enum.IntEnum):
    """What a router makes of its logits (the codes of include/rocm_wmma_gemm_c.h)."""

    softmax = 0
    sigmoid = 1


def _score(code):
    return code if type(code) is score else score(code)


class _RoutingC(ctypes.Structure):
    _fields_ = [("score", ctypes.c_int), ("bias", ctypes.c_void_p), ("mask", ctypes.c_void_p)] + [
        (n, ctypes.c_int) for n in ("groups", "kept_groups", "group_best", "renormalize")] + [("scale", ctypes.c_float)]


class _EpilogueC(ctypes.Structure):
    _fields_ = [("bias", ctypes.c_void_p), ("residual", ctypes.c_void_p), ("preact", ctypes.c_void_p),
                ("activation", ctypes.c_int)]


class _ProductPlanC(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("form", "block_m", "block_n", "cut_tail", "k_slices", "once", "copies")]


@dataclass(frozen=True)
class ProductPlan:
    """How a layer's product would run (the fields of rocm_wmma_gemm_product_plan)."""

    form: int
    block_m: int
    block_n: int
    cut_tail: int
    k_slices: int
    once: int
    copies: int


MAX_GROUPS = 512
MAX_EXPERTS, MAX_CHOICES, MAX_EXPERT_GROUPS, MAX_ENTRIES = 512, 32, 16, 256


class _VariantInfoC(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in (
        "block_m", "block_n", "block_k", "warps_m", "warps_n", "warp_tile_m", "warp_tile_n",
        "pipeline", "lds_bytes", "threads")]


@dataclass(frozen=True)
class VariantInfo:
    index: int
    block_m: int
    block_n: int
    block_k: int
    warps_m: int
    warps_n: int
    warp_tile_m: int
    warp_tile_n: int
    pipeline: int
    lds_bytes: int
    threads: int


def library_dir() -> str:
    """Directory searched first (the C++ loader's ROCM_WMMA_GEMM_LIB_DIR define)."""
    return os.environ.get("ROCM_WMMA_GEMM_LIB_DIR", _DEFAULT_LIB_DIR)


def library_path(arch: str = "gfx950") -> str:
    return os.path.join(library_dir(), f"librocm_wmma_gemm_{arch}.so")


def build_library(jobs: int = 8, force: bool = False) -> str:
    """Compile the HIP library in-tree (cross-compiles without a GPU)."""
    cmd = ["make", "-C", os.path.join(_HERE, "csrc"), f"-j{jobs}", "all"]
    if force:
        cmd.insert(1, "-B")
    subprocess.run(cmd, check=True, stdout=subprocess.DEVNULL)
    return os.path.join(_DEFAULT_LIB_DIR, "librocm_wmma_gemm_gfx950.so")


def source_stamp() -> str:
    """Sixteen hex digits over everything a kernel launch of the library depends on: the
    kernel and host sources under csrc/ (the generated table left out) and the tuned
    tables.  A counter summary under profiles/ records the stamp of the tree it was measured
    on, so that a reader (and bench.py) can tell whether it still describes this library."""
    import glob
    import hashlib

    files = []
    for pattern in ("csrc/*.hip", "csrc/*.hpp", "csrc/*.cpp", "csrc/*.def", "csrc/kernel/*.hpp",
                    "config/gemm_config_gfx950_*.json", "config/model_gfx950.json"):
        files += glob.glob(os.path.join(_HERE, pattern))
    h = hashlib.sha256()
    for path in sorted(f for f in files if not f.endswith("config_generated.hpp")):
        h.update(os.path.relpath(path, _HERE).encode())
        with open(path, "rb") as f:
            h.update(f.read())
    return h.hexdigest()[:16]


def detect_arch() -> str:
    import torch

    if not torch.cuda.is_available():
        raise GemmLibraryError("rocm_wmma_gemm::loader: hipGetDeviceProperties failed (no GPU)")
    name = torch.cuda.get_device_properties(0).gcnArchName
    return name.split(":", 1)[0]


_TORCH = None


def _torch():
    """torch, imported with the first tensor that is passed (a statement in every call costs more than this)."""
    global _TORCH
    if _TORCH is None:
        import torch

        _TORCH = torch
    return _TORCH


_SLOTS = {}


def _type_slot(c_dtype, ab_dtype) -> int:
    slot = _SLOTS.get((c_dtype, ab_dtype))
    if slot is None:
        import torch

        _SLOTS.update({(torch.float16, torch.float16): 0, (torch.float32, torch.float16): 1,
                       (torch.bfloat16, torch.bfloat16): 2, (torch.float32, torch.bfloat16): 3})
        slot = _SLOTS.get((c_dtype, ab_dtype))
        if slot is None:
            raise TypeError(f"Unsupported type pair for rocm_wmma_gemm loader: C={c_dtype}, A/B={ab_dtype}")
    return slot


class Loader:
    """Opens the per-architecture library and forwards gemm calls through its C ABI."""

    _ENTRY_ARGS = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t,
                   ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int, ctypes.c_int,
                   ctypes.c_int, ctypes.c_void_p]

    def __init__(self, arch: str | None = None, lib_dir: str | None = None):
        self.arch = arch if arch is not None else detect_arch()
        name = f"librocm_wmma_gemm_{self.arch}.so"
        first = os.path.join(lib_dir if lib_dir is not None else library_dir(), name)
        errors = []
        self._lib = None
        for candidate in (first, name):
            try:
                self._lib = ctypes.CDLL(candidate, mode=os.RTLD_NOW | os.RTLD_LOCAL)
                self.path = candidate
                break
            except OSError as e:
                errors.append(str(e))
        if self._lib is None:
            raise GemmLibraryError(f"rocm_wmma_gemm::loader: could not open {name}: " + "; ".join(errors))
        self._entries = []
        for suffix in ENTRY_SUFFIXES:
            sym = "rocm_wmma_gemm_" + suffix
            try:
                fn = getattr(self._lib, sym)
            except AttributeError as e:
                raise GemmLibraryError(f"rocm_wmma_gemm::loader: symbol not found: {sym} ({e})")
            fn.restype = None
            fn.argtypes = self._ENTRY_ARGS
            self._entries.append(fn)
        self._bind_extras()

    # ------------------------------------------------------------------ extras
    def _bind_extras(self):
        L = self._lib
        self._has_extras = hasattr(L, "rocm_wmma_gemm_run_variant")
        if not self._has_extras:
            return
        L.rocm_wmma_gemm_arch.restype = ctypes.c_char_p
        L.rocm_wmma_gemm_arch.argtypes = []
        L.rocm_wmma_gemm_variant_count.restype = ctypes.c_int
        L.rocm_wmma_gemm_variant_count.argtypes = []
        L.rocm_wmma_gemm_variant_info_get.restype = ctypes.c_int
        L.rocm_wmma_gemm_variant_info_get.argtypes = [ctypes.c_int, ctypes.POINTER(_VariantInfoC)]
        L.rocm_wmma_gemm_select.restype = ctypes.c_int
        L.rocm_wmma_gemm_select.argtypes = [ctypes.c_size_t] * 3 + [ctypes.c_int] * 4 + [
            ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int)]
        L.rocm_wmma_gemm_select_batched.restype = ctypes.c_int
        L.rocm_wmma_gemm_select_batched.argtypes = [ctypes.c_size_t] * 4 + [ctypes.c_int] * 4 + [
            ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int)]
        L.rocm_wmma_gemm_run_variant.restype = ctypes.c_int
        L.rocm_wmma_gemm_run_variant.argtypes = [ctypes.c_int] * 4 + self._ENTRY_ARGS
        if hasattr(L, "rocm_wmma_gemm_run_variant_ex"):
            L.rocm_wmma_gemm_run_variant_ex.restype = ctypes.c_int
            L.rocm_wmma_gemm_run_variant_ex.argtypes = [ctypes.c_int] * 5 + self._ENTRY_ARGS
            L.rocm_wmma_gemm_select_ex.restype = ctypes.c_int
            L.rocm_wmma_gemm_select_ex.argtypes = [ctypes.c_size_t] * 4 + [ctypes.c_int] * 4 + [
                ctypes.POINTER(ctypes.c_int)] * 3
        if hasattr(L, "rocm_wmma_gemm_workspace_release"):
            L.rocm_wmma_gemm_workspace_release.restype = ctypes.c_int
            L.rocm_wmma_gemm_workspace_release.argtypes = []
        if hasattr(L, "rocm_wmma_gemm_noalloc"):
            L.rocm_wmma_gemm_noalloc.restype = ctypes.c_int
            L.rocm_wmma_gemm_noalloc.argtypes = [ctypes.c_int] + self._ENTRY_ARGS
        if hasattr(L, "rocm_wmma_gemm_linear"):
            p, z, i = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int
            for name, args in (
                    ("linear", [i, p, p, p, z, z, z, i, p, p]),
                    ("linear_backward", [i] + [p] * 7 + [z] * 3 + [i] * 3 + [p]),
                    ("grouped", [i, p, p, p, p, z, z, z, z, i, p, p]),
                    ("grouped_backward", [i] + [p] * 8 + [z] * 4 + [i] * 3 + [p]),
                    ("product_select", [i, i, z, z, z, z, i, i, p]),
                    ("orthogonalize", [i, i, p, p, z, z, z, i, p, ctypes.c_float, p]),
                    ("route", [i, p, p, p, p, z, z, z, p]),
                    ("route_backward", [i, p, p, p, p, z, z, z, i, i, ctypes.c_float, p]),
                    ("dispatch", [i] + [p] * 5 + [z] * 4 + [p]),
                    ("combine", [i, i] + [p] * 5 + [z] * 3 + [p]),
                    ("combine_backward", [i, i] + [p] * 6 + [z] * 3 + [p]),
                    ("linear_cross_entropy", [i] + [p] * 5 + [i, z, z, z, i, p]),
                    ("linear_cross_entropy_backward", [i] + [p] * 7 + [i, z, z, z, i, i, p]),
                    ("linear_distillation", [i] + [p] * 6 + [i, p, z, z, z, z, ctypes.c_float, i, p]),
                    ("linear_distillation_backward", [i] + [p] * 8 + [i, p, z, z, z, z, ctypes.c_float, i, i, p])):
                fn = getattr(L, "rocm_wmma_gemm_" + name)
                fn.restype = ctypes.c_int
                fn.argtypes = args

    def library_arch(self) -> str:
        return self._lib.rocm_wmma_gemm_arch().decode()

    def variants(self) -> list[VariantInfo]:
        out = []
        for i in range(self._lib.rocm_wmma_gemm_variant_count()):
            c = _VariantInfoC()
            if self._lib.rocm_wmma_gemm_variant_info_get(i, ctypes.byref(c)) != 0:
                raise GemmLibraryError(f"variant {i} not described by the library")
            out.append(VariantInfo(i, *[getattr(c, n) for n, _ in _VariantInfoC._fields_]))
        return out

    def select(self, M: int, N: int, K: int, type_idx: int, layout_c: int, layout_a: int,
               layout_b: int, batch_count: int = 1) -> tuple[int, int, int]:
        """(variant, swizzle, split_k) the dispatcher picks for this problem (for a strided
        batch of batch_count such problems)."""
        swz, sk = ctypes.c_int(0), ctypes.c_int(0)
        v = self._lib.rocm_wmma_gemm_select_batched(
            M, N, K, batch_count, type_idx, int(layout_c), int(layout_a), int(layout_b),
            ctypes.byref(swz), ctypes.byref(sk))
        return v, swz.value, sk.value

    # ------------------------------------------------------------------ gemm
    @staticmethod
    def _stream_handle(stream) -> int:
        import torch

        if stream is None:
            stream = torch.cuda.current_stream()
        return int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)

    @staticmethod
    def _check(C, A, B, M, N, K, batch):
        for name, t, need in (("A", A, M * K * batch), ("B", B, K * N * batch), ("C", C, M * N * batch)):
            if not t.is_cuda:
                raise ValueError(f"{name} must be a device tensor")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be densely packed")
            if t.numel() < need:
                raise ValueError(f"{name} holds {t.numel()} elements, the problem needs {need}")
        if A.dtype != B.dtype:
            raise TypeError("A and B must share an element type")
        # the library's own limits: beyond them its C++ side throws, which a caller that
        # came in through ctypes could not catch
        for name, v in (("M", M), ("N", N), ("K", K)):
            if v < 0 or v > 0x7FFFFFFF:
                raise ValueError(f"{name} = {v} does not fit in 31 bits")
        if batch < 0:
            raise ValueError("batch_count must not be negative")

    def gemm(self, C, A, B, M: int, N: int, K: int, layout_c=row_major, layout_a=row_major,
             layout_b=row_major, batch_count: int = 1, stream=None) -> None:
        """C = A * B, enqueued on ``stream`` (default: torch's current stream).

        C, A, B are device tensors used as flat packed storage in the stated layouts."""
        self._check(C, A, B, M, N, K, batch_count)
        slot = _type_slot(C.dtype, A.dtype)
        handle = ctypes.c_void_p(self._stream_handle(stream))
        self._entries[slot](C.data_ptr(), A.data_ptr(), B.data_ptr(), M, N, K, batch_count,
                            int(layout_c), int(layout_a), int(layout_b), ctypes.byref(handle))

    def gemm_raw(self, slot: int, c_ptr: int, a_ptr: int, b_ptr: int, M: int, N: int, K: int,
                 batch_count: int, layout_c: int, layout_a: int, layout_b: int,
                 stream_handle: int) -> None:
        """Direct C-ABI call with raw device addresses (no checks)."""
        handle = ctypes.c_void_p(stream_handle)
        self._entries[slot](c_ptr, a_ptr, b_ptr, M, N, K, batch_count, layout_c, layout_a,
                            layout_b, ctypes.byref(handle))

    def workspace_release(self) -> int:
        """Frees the current device's library-owned scratch buffer (0), unless a captured
        graph may hold its address (1)."""
        return self._lib.rocm_wmma_gemm_workspace_release()

    def gemm_noalloc(self, C, A, B, M: int, N: int, K: int, layout_c=row_major,
                     layout_a=row_major, layout_b=row_major, batch_count: int = 1,
                     stream=None) -> int:
        """gemm() through the entry point that allocates nothing: scratch memory comes from
        a fixed per-GPU array of NOALLOC_SCRATCH_BYTES.  Returns the library's status code
        (0 = enqueued, ERR_SCRATCH = the call needs more scratch memory than that)."""
        self._check(C, A, B, M, N, K, batch_count)
        slot = _type_slot(C.dtype, A.dtype)
        handle = ctypes.c_void_p(self._stream_handle(stream))
        return self._lib.rocm_wmma_gemm_noalloc(
            slot, C.data_ptr(), A.data_ptr(), B.data_ptr(), M, N, K, batch_count,
            int(layout_c), int(layout_a), int(layout_b), ctypes.byref(handle))

    def select_ex(self, M: int, N: int, K: int, type_idx: int, layout_c: int, layout_a: int,
                  layout_b: int, batch_count: int = 1) -> tuple[int, int, int, int]:
        """(variant, swizzle, split_k, touch_ahead) the dispatcher picks for this problem."""
        swz, sk, touch = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
        v = self._lib.rocm_wmma_gemm_select_ex(
            M, N, K, batch_count, type_idx, int(layout_c), int(layout_a), int(layout_b),
            ctypes.byref(swz), ctypes.byref(sk), ctypes.byref(touch))
        return v, swz.value, sk.value, touch.value

    def run_variant(self, variant: int, swizzle: int, split_k: int, C, A, B, M: int, N: int,
                    K: int, layout_c=row_major, layout_a=row_major, layout_b=row_major,
                    batch_count: int = 1, stream=None, touch_ahead: int = 0) -> int:
        """Same as gemm() with the tile variant, swizzle, split-K form and line touches forced
        (tuner hook)."""
        self._check(C, A, B, M, N, K, batch_count)
        slot = _type_slot(C.dtype, A.dtype)
        handle = ctypes.c_void_p(self._stream_handle(stream))
        return self._lib.rocm_wmma_gemm_run_variant_ex(
            slot, variant, swizzle, split_k, touch_ahead, C.data_ptr(), A.data_ptr(), B.data_ptr(),
            M, N, K, batch_count, int(layout_c), int(layout_a), int(layout_b), ctypes.byref(handle))

    # ------------------------------------------------------------------ layer products
    _STATUS = {ERR_VARIANT: "no kernel for this problem", ERR_ARGUMENT: "an argument is out of range or missing",
               ERR_SCRATCH: "no scratch memory (too much asked for, or the stream is capturing: size the "
                            "library's buffer with one eager call first)",
               ERR_RUNTIME: "the HIP runtime reported an error", ERR_LIMIT: "a size is beyond the library's limits"}

    def _done(self, name, status):
        if status != OK:
            raise GemmLibraryError(f"rocm_wmma_gemm_{name}: {self._STATUS.get(status, status)}")

    # (A decode step is many small calls, each a few microseconds on the GPU: what is checked here is
    # asked of each tensor once, in the cheapest form.)
    @staticmethod
    def _held(name, t, need, dtype, device):
        """Address of a packed tensor on `device` that holds `need` elements of `dtype`."""
        if t.dtype is dtype and t.get_device() == device and t.is_contiguous() and t.numel() >= need:
            return t.data_ptr()
        if t.get_device() != device:
            raise ValueError(f"{name} must be a device tensor" if not t.is_cuda else
                             f"{name} is on device {t.get_device()}, the other operands on {device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be densely packed")
        if t.dtype is not dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        raise ValueError(f"{name} holds {t.numel()} elements, the problem needs {need}")

    @staticmethod
    def _stream_on(stream, device):
        """Handle of `stream`, or of torch's current one on `device` (whose stream object takes 3 us
        to make, a third of a small call)."""
        if stream is None:
            torch = _torch()
            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
            return raw(device) if raw is not None else int(torch.cuda.current_stream(device).cuda_stream)
        return Loader._stream_handle(stream)

    @staticmethod
    def _device_of(name, t):
        torch = _torch()
        device = t.get_device()
        if device < 0:
            raise ValueError(f"{name} must be a device tensor")
        if device != torch.cuda.current_device():  # (whose scratch buffer and streams the library uses)
            raise ValueError(f"{name} is on device {device}, the current one is {torch.cuda.current_device()}")
        return device

    @staticmethod
    def _sizes(*sizes):
        all_bits = 0
        for v in sizes:
            all_bits |= v  # (negative if one is, past 31 bits if one is)
        if 0 <= all_bits <= 0x7FFFFFFF:
            return
        for v in sizes:
            if v < 0 or v > 0x7FFFFFFF:
                raise ValueError(f"a size of {v} does not fit in 31 bits")

    def _groups(self, offsets, device):
        import torch

        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must hold groups + 1 row offsets")
        groups = offsets.numel() - 1
        if groups > MAX_GROUPS:
            raise ValueError(f"{groups} groups: at most {MAX_GROUPS} in one call")
        return self._held("offsets", offsets, groups + 1, torch.int32, device), groups

    def _forward(self, fn, name, C, A, B, offsets, M, N, K, layout_b, bias, residual, preact, act, stream):
        self._sizes(M, N, K)
        out, ab = C.dtype, A.dtype
        slot = _type_slot(out, ab)
        act = act if type(act) is activation else activation(act)
        layout_b = layout_b if type(layout_b) is m_layout else m_layout(layout_b)
        held, device = self._held, self._device_of("C", C)
        groups, where = 1, ()
        if offsets is not None:
            where = self._groups(offsets, device)
            groups = where[1]
        e = _EpilogueC(None if bias is None else held("bias", bias, groups * N, ab, device),
                       None if residual is None else held("residual", residual, M * N, out, device),
                       None if preact is None else held("preact", preact, M * N, ab, device), act)
        status = fn(slot, held("C", C, M * N, out, device), held("A", A, M * K, ab, device),
                    held("B", B, groups * K * N, ab, device), *where, M, N, K, layout_b, ctypes.byref(e),
                    ctypes.byref(ctypes.c_void_p(self._stream_on(stream, device))))
        if status != OK:
            self._done(name, status)

    def _backward(self, fn, name, dA, dB, dbias, dC, A, B, offsets, M, N, K, layout_b, preact, act, accumulate, stream):
        self._sizes(M, N, K)
        wanted = [t for t in (dA, dB, dbias) if t is not None]
        if not wanted:
            raise ValueError("none of dA, dB and dbias is wanted")
        out, ab = wanted[0].dtype, dC.dtype
        if any(t.dtype is not out for t in wanted):
            raise TypeError("dA, dB and dbias must share an element type")
        slot = _type_slot(out, ab)
        act = act if type(act) is activation else activation(act)
        layout_b = layout_b if type(layout_b) is m_layout else m_layout(layout_b)
        if act is activation.none:
            preact = None
        elif preact is None:
            raise ValueError(f"the gradient of {act.name} needs preact")
        if dB is not None and A is None or dA is not None and B is None:
            raise ValueError("dA needs B, and dB needs A")
        held, device = self._held, self._device_of("dC", dC)
        groups, where = 1, ()
        if offsets is not None:
            where = self._groups(offsets, device)
            groups = where[1]
        args = [None if t is None else held(what, t, need, dtype, device)
                for what, t, need, dtype in (("dA", dA, M * K, out), ("dB", dB, groups * K * N, out),
                                             ("dbias", dbias, groups * N, out), ("dC", dC, M * N, ab),
                                             ("A", A, M * K, ab), ("B", B, groups * K * N, ab),
                                             ("preact", preact, M * N, ab))]
        status = fn(slot, *args, *where, M, N, K, layout_b, act, 1 if accumulate else 0,
                    ctypes.byref(ctypes.c_void_p(self._stream_on(stream, device))))
        if status != OK:
            self._done(name, status)

    def linear(self, C, A, B, M: int, N: int, K: int, layout_b=col_major, bias=None, residual=None, preact=None,
               activation=activation.none, stream=None) -> None:
        """C = activation(A B + bias) + residual on ``stream`` (default: torch's current stream).

        A (M x K) and C (M x N) are row-major; B (K x N) is column-major (weights stored N x K)
        or row-major.  bias: N values of A's type; residual: M x N of C's type, may be C itself;
        preact: M x N of A's type, receives A B + bias for the backward pass."""
        self._forward(self._lib.rocm_wmma_gemm_linear, "linear", C, A, B, None, M, N, K, layout_b, bias, residual, preact, activation, stream)

    def linear_backward(self, dA, dB, dbias, dC, A, B, M: int, N: int, K: int, layout_b=col_major, preact=None,
                        activation=activation.none, accumulate: bool = False, stream=None) -> None:
        """The gradients of linear() from dC (M x N, A's type): dA = dZ B^T, dB = A^T dZ in B's
        layout and dbias = the sum of dZ's rows, with dZ = dC activation'(preact).  A result that
        is None is not computed.  accumulate: dB and dbias are added to."""
        self._backward(self._lib.rocm_wmma_gemm_linear_backward, "linear_backward", dA, dB, dbias, dC, A, B, None, M, N, K, layout_b, preact, activation,
                       accumulate, stream)

    def grouped(self, C, A, B, offsets, M: int, N: int, K: int, layout_b=col_major, bias=None, residual=None,
                preact=None, activation=activation.none, stream=None) -> None:
        """linear() for groups of rows with a weight (and bias) each: rows offsets[e] ..
        offsets[e+1] - 1 of A and C belong to weight e of B (groups x K x N).  offsets: groups + 1
        int32 on the device; they are read there, never by the host.  Rows outside the groups are
        not touched."""
        self._forward(self._lib.rocm_wmma_gemm_grouped, "grouped", C, A, B, offsets, M, N, K, layout_b, bias, residual, preact, activation, stream)

    def grouped_backward(self, dA, dB, dbias, dC, A, B, offsets, M: int, N: int, K: int, layout_b=col_major,
                         preact=None, activation=activation.none, accumulate: bool = False, stream=None) -> None:
        """The gradients of grouped(); an empty group's are zero (unchanged with accumulate)."""
        self._backward(self._lib.rocm_wmma_gemm_grouped_backward, "grouped_backward", dA, dB, dbias, dC, A, B, offsets, M, N, K, layout_b, preact, activation,
                       accumulate, stream)

    _PRODUCTS = ("forward", "gradient_a", "gradient_b", "steps_s", "steps_q", "steps_x", "steps_last")

    def product_select(self, product: str, M: int, N: int, K: int, groups: int = 0, type_idx: int = 2,
                       layout_b=col_major, activation=activation.none) -> ProductPlan:
        """Which kernel ``product`` ("forward", "gradient_a" or "gradient_b") of linear() (groups = 0)
        or grouped() runs on, and how; operands that start on 16 bytes assumed.  Or a product of
        orthogonalize() for ``groups`` M x N matrices: "steps_s" (X X^T), "steps_q" (b S + c S^2), "steps_x"
        (a X + Q X) or "steps_last" (the last step's; type_idx one whose A has the type of O)."""
        c = _ProductPlanC()
        self._done("product_select", self._lib.rocm_wmma_gemm_product_select(
            self._PRODUCTS.index(product), type_idx, M, N, K, groups, int(layout_b),
            int(activation), ctypes.byref(c)))
        return ProductPlan(*[getattr(c, n) for n, _ in _ProductPlanC._fields_])

    def orthogonalize(self, O, G, M: int, N: int, batch_count: int = 1, steps: int = 5,
                      coefficients=(3.4445, -4.7750, 2.0315), epsilon: float = 1e-7, stream=None) -> None:
        """O = G / (|G| + epsilon) after ``steps`` Newton-Schulz steps x -> a x + b x^3 + c x^5 on
        its singular values, for a batch of row-major M x N matrices: an update with singular
        values near 1.  G: f16, bf16 or f32; O: f16 or bf16.  Matrices past 64 x 256 are multiplied with f16
        operands: coefficients may not let the singular values s of an iterate grow past |b| s^2 + |c| s^4 or
        2 s sqrt(min(M, N)) of 65504 (with the default they stay below 1.3); smaller ones are worked on in fp32."""
        import torch

        self._sizes(M, N, batch_count)
        codes = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
        if G.dtype not in codes or codes.get(O.dtype, 2) == 2:
            raise TypeError(f"Unsupported type pair for orthogonalize: O={O.dtype}, G={G.dtype}")
        if steps < 1 or len(coefficients) != 3:
            raise ValueError("at least one step, and three coefficients")
        device = self._device_of("O", O)
        o = self._held("O", O, batch_count * M * N, O.dtype, device)
        g = self._held("G", G, batch_count * M * N, G.dtype, device)
        handle = ctypes.c_void_p(self._stream_on(stream, device))
        self._done("orthogonalize", self._lib.rocm_wmma_gemm_orthogonalize(
            codes[G.dtype], codes[O.dtype], o, g, M, N, batch_count, steps, (ctypes.c_float * 3)(*coefficients),
            epsilon, ctypes.byref(handle)))

    # ------------------------------------------------------------------ from a router to the experts and back
    _ELEMENTS = {}

    @classmethod
    def _element(cls, name, t):
        """Code of a tensor's element type."""
        code = cls._ELEMENTS.get(t.dtype)
        if code is None:
            import torch

            cls._ELEMENTS.update({torch.float16: 0, torch.bfloat16: 1, torch.float32: 2})
            code = cls._ELEMENTS.get(t.dtype)
            if code is None:
                raise TypeError(f"{name} must be f16, bf16 or f32, got {t.dtype}")
        return code

    @staticmethod
    def _plain_types():
        torch = _TORCH or _torch()
        return torch.int32, torch.float32

    def _handle_on(self, stream, device):
        return ctypes.byref(ctypes.c_void_p(self._stream_on(stream, device)))

    def route(self, chosen, weights, logits, M: int, E: int, k: int, score=score.softmax, bias=None, mask=None,
              groups: int = 1, kept_groups: int | None = None, group_best: int = 2, renormalize: bool = True,
              scale: float = 1.0, stream=None) -> None:
        """The k experts of every token, the best first, and their weights, from a router's logits (M x E: f16, bf16
        or f32).  chosen: M x k int32; weights: M x k f32.

        score: softmax over the experts, or sigmoid.  bias (E, f32) is added to the scores for the choice alone; the experts
        of the largest sums are chosen, of the largest logits where there is no bias; of equal ones the lower.  groups: the
        experts form so many groups of neighbours, of which those ``kept_groups`` (all) take part whose
        ``group_best`` (1 or 2) best biased scores sum to most.  renormalize: a token's weights are divided by their sum; then
        multiplied by ``scale``.  mask (M, bool or uint8): tokens where it is 0 go nowhere: experts -1, weights 0."""
        self._sizes(M, E, k)
        int32, f32 = self._plain_types()
        held, device = self._held, self._device_of("logits", logits)
        r = _RoutingC(_score(score), None if bias is None else held("bias", bias, E, f32, device),
                      None if mask is None else held("mask", mask, M, _torch().uint8 if mask.dtype is not _torch().bool
                                                     else _torch().bool, device), groups,
                      groups if kept_groups is None else kept_groups, group_best, 1 if renormalize else 0, scale)
        self._done("route", self._lib.rocm_wmma_gemm_route(
            self._element("logits", logits), held("chosen", chosen, M * k, int32, device),
            held("weights", weights, M * k, f32, device), held("logits", logits, M * E, logits.dtype, device),
            ctypes.byref(r), M, E, k, self._handle_on(stream, device)))

    def route_backward(self, dlogits, dweights, chosen, logits, M: int, E: int, k: int, score=score.softmax,
                       renormalize: bool = True, scale: float = 1.0, stream=None) -> None:
        """The gradient of route()'s weights by the logits: dlogits (M x E, the logits' type) from dweights (M x k, f32)
        and the experts that were chosen.  The choice itself has no gradient, nor has the bias."""
        self._sizes(M, E, k)
        int32, f32 = self._plain_types()
        held, device = self._held, self._device_of("dlogits", dlogits)
        self._done("route_backward", self._lib.rocm_wmma_gemm_route_backward(
            self._element("logits", logits), held("dlogits", dlogits, M * E, logits.dtype, device),
            held("dweights", dweights, M * k, f32, device), held("chosen", chosen, M * k, int32, device),
            held("logits", logits, M * E, logits.dtype, device), M, E, k, _score(score), 1 if renormalize else 0, scale,
            self._handle_on(stream, device)))

    def dispatch(self, rows, offsets, places, X, chosen, M: int, N: int, k: int, stream=None) -> None:
        """Sorts the choices of M tokens by expert, in their order within one.  offsets (E + 1 int32): where every expert's
        rows start, as grouped() reads them; places (M x k int32): the row of every choice, -1 for a choice outside 0 .. E - 1;
        rows (M k x N): the tokens' rows of X (M x N: f16, bf16 or f32) in that order.  rows None: the offsets and
        places alone.  Rows from offsets[E] on are left as they were.  The gradient of X is
        combine() of rows' without weights."""
        self._sizes(M, N, k)
        int32, _ = self._plain_types()
        held, device = self._held, self._device_of("offsets", offsets)
        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must hold experts + 1 row offsets")
        E = offsets.numel() - 1
        code, to, x = 2, None, None
        if rows is not None:
            if X is None:
                raise ValueError("rows needs X")
            code, to = self._element("X", X), held("rows", rows, M * k * N, X.dtype, device)
            x = held("X", X, M * N, X.dtype, device)
        self._done("dispatch", self._lib.rocm_wmma_gemm_dispatch(
            code, to, held("offsets", offsets, E + 1, int32, device), held("places", places, M * k, int32, device), x,
            held("chosen", chosen, M * k, int32, device), E, M, N, k, self._handle_on(stream, device)))

    def combine(self, C, rows, places, M: int, N: int, k: int, weights=None, residual=None, stream=None) -> None:
        """C (M x N) = the sum over a token's k choices of weights (M x k, f32; None: 1) times the row of ``rows`` (M k x N)
        that ``places`` names, plus residual (M x N of C's type; may be C itself).  A place of -1 adds nothing.  C: the type
        of rows, or f32; summed in f32, rounded once."""
        self._sizes(M, N, k)
        int32, f32 = self._plain_types()
        held, device = self._held, self._device_of("C", C)
        out = self._element("C", C)
        self._done("combine", self._lib.rocm_wmma_gemm_combine(
            self._element("rows", rows), out, held("C", C, M * N, C.dtype, device),
            held("rows", rows, M * k * N, rows.dtype, device), held("places", places, M * k, int32, device),
            None if weights is None else held("weights", weights, M * k, f32, device),
            None if residual is None else held("residual", residual, M * N, C.dtype, device), M, N, k,
            self._handle_on(stream, device)))

    def combine_backward(self, drows, dweights, dC, rows, places, M: int, N: int, k: int, weights=None,
                         stream=None) -> None:
        """The gradients of combine() from dC (M x N, C's type): drows (M k x N, the type of rows) = weight times dC's row,
        for the rows that ``places`` names, each once (others are left as they were); dweights (M x k, f32) = the product of
        dC's row with the choice's.  A result that is None is not computed.  (The gradient of the residual is dC.)"""
        self._sizes(M, N, k)
        if drows is None and dweights is None:
            raise ValueError("none of drows and dweights is wanted")
        if dweights is not None and rows is None:
            raise ValueError("dweights needs rows")
        int32, f32 = self._plain_types()
        held, device = self._held, self._device_of("dC", dC)
        kind = rows if rows is not None else drows
        self._done("combine_backward", self._lib.rocm_wmma_gemm_combine_backward(
            self._element("rows", kind), self._element("dC", dC),
            None if drows is None else held("drows", drows, M * k * N, kind.dtype, device),
            None if dweights is None else held("dweights", dweights, M * k, f32, device),
            held("dC", dC, M * N, dC.dtype, device),
            None if rows is None else held("rows", rows, M * k * N, kind.dtype, device),
            held("places", places, M * k, int32, device),
            None if weights is None else held("weights", weights, M * k, f32, device), M, N, k,
            self._handle_on(stream, device)))

    # ------------------------------------------------------------------ a projection onto a vocabulary and its loss
    def _indices(self, name, t, need, device):
        """(address, 1 for 64 bits) of a tensor of indices."""
        import torch

        if t.dtype is not torch.int64 and t.dtype is not torch.int32:
            raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
        return self._held(name, t, need, t.dtype, device), 1 if t.dtype is torch.int64 else 0

    def _list(self, entries, teacher, M, device):
        if entries.dim() != 2 or entries.shape[0] != M:
            raise ValueError(f"entries must be {M} lists of one length, got {tuple(entries.shape)}")
        k = entries.shape[1]
        if k > MAX_ENTRIES:
            raise ValueError(f"{k} entries a row: at most {MAX_ENTRIES}")
        _, f32 = self._plain_types()
        return (*self._indices("entries", entries, M * k, device), self._held("teacher", teacher, M * k, f32, device), k)

    def _operands(self, A, B, M, N, K, device):
        """Element code and addresses of the states and the weights."""
        code = self._element("A", A)
        if code == 2:
            raise TypeError("A and B must be f16 or bf16")
        return code, self._held("A", A, M * K, A.dtype, device), self._held("B", B, K * N, A.dtype, device)

    def _gradients(self, dA, dB, A, M, N, K, device):
        """Type pair and addresses of the gradients that are wanted."""
        wanted = [t for t in (dA, dB) if t is not None]
        if not wanted:
            raise ValueError("none of dA and dB is wanted")
        out = wanted[0].dtype
        if any(t.dtype is not out for t in wanted):
            raise TypeError("dA and dB must share an element type")
        return (_type_slot(out, A.dtype), None if dA is None else self._held("dA", dA, M * K, out, device),
                None if dB is None else self._held("dB", dB, K * N, out, device))

    def linear_cross_entropy(self, loss, lse, A, B, targets, M: int, N: int, K: int, layout_b=col_major, stream=None) -> None:
        """The cross entropy of every row of the logits A B (A: M x K, B: K x N as in linear(), f16 or bf16) against its
        target, without keeping the logits: loss (M, f32) = log sum_v e^z_v - z_target; 0 for a target outside 0 .. N - 1,
        whose row is left out.  lse (M, f32) receives the logarithms, for the backward pass.  targets: M int32 or int64."""
        self._sizes(M, N, K)
        _, f32 = self._plain_types()
        held, device = self._held, self._device_of("A", A)
        code, a, b = self._operands(A, B, M, N, K, device)
        self._done("linear_cross_entropy", self._lib.rocm_wmma_gemm_linear_cross_entropy(
            code, held("loss", loss, M, f32, device), held("lse", lse, M, f32, device), a, b,
            *self._indices("targets", targets, M, device), M, N, K, m_layout(layout_b), self._handle_on(stream, device)))

    def linear_cross_entropy_backward(self, dA, dB, dloss, lse, A, B, targets, M: int, N: int, K: int, layout_b=col_major,
                                      accumulate: bool = False, stream=None) -> None:
        """The gradients of linear_cross_entropy() from dloss (M, f32) and its lse: dz = dloss (softmax(z) - 1 at the
        target), dA = dz B^T (M x K) and dB = A^T dz in B's layout, of A's type or f32.  A result that is None is not
        computed.  accumulate: dB is added to."""
        self._sizes(M, N, K)
        _, f32 = self._plain_types()
        held, device = self._held, self._device_of("A", A)
        _, a, b = self._operands(A, B, M, N, K, device)
        self._done("linear_cross_entropy_backward", self._lib.rocm_wmma_gemm_linear_cross_entropy_backward(
            *self._gradients(dA, dB, A, M, N, K, device), held("dloss", dloss, M, f32, device), held("lse", lse, M, f32, device),
            a, b, *self._indices("targets", targets, M, device), M, N, K, m_layout(layout_b), 1 if accumulate else 0,
            self._handle_on(stream, device)))

    def linear_distillation(self, loss, lse, picked, A, B, entries, teacher, M: int, N: int, K: int, layout_b=col_major,
                            temperature: float = 1.0, stream=None) -> None:
        """How far every row of the logits A B is from the entries that a teacher lists for it (entries: M x k int32 or int64,
        teacher: M x k f32, its logits): loss (M, f32) = temperature^2 sum_j q_j (log q_j - log p_j) with q the
        softmax of the row's teacher over the temperature and p that of the logits over all N.  An entry outside 0 .. N - 1 is not
        in the list; a row with an empty list is left out, its loss is 0.  lse (M, f32) and picked (M x k, f32: the logits of
        the entries) are for the backward pass."""
        self._sizes(M, N, K)
        _, f32 = self._plain_types()
        held, device = self._held, self._device_of("A", A)
        code, a, b = self._operands(A, B, M, N, K, device)
        at, wide, given, k = self._list(entries, teacher, M, device)
        self._done("linear_distillation", self._lib.rocm_wmma_gemm_linear_distillation(
            code, held("loss", loss, M, f32, device), held("lse", lse, M, f32, device), held("picked", picked, M * k, f32, device),
            a, b, at, wide, given, M, N, K, k, temperature, m_layout(layout_b), self._handle_on(stream, device)))

    def linear_distillation_backward(self, dA, dB, dloss, lse, picked, A, B, entries, teacher, M: int, N: int, K: int,
                                     layout_b=col_major, temperature: float = 1.0, accumulate: bool = False, stream=None) -> None:
        """The gradients of linear_distillation() by the states and the weights, as linear_cross_entropy_backward()'s, from
        its lse and picked.  (The teacher's logits have none.)"""
        self._sizes(M, N, K)
        _, f32 = self._plain_types()
        held, device = self._held, self._device_of("A", A)
        _, a, b = self._operands(A, B, M, N, K, device)
        at, wide, given, k = self._list(entries, teacher, M, device)
        self._done("linear_distillation_backward", self._lib.rocm_wmma_gemm_linear_distillation_backward(
            *self._gradients(dA, dB, A, M, N, K, device), held("dloss", dloss, M, f32, device), held("lse", lse, M, f32, device),
            held("picked", picked, M * k, f32, device), a, b, at, wide, given, M, N, K, k, temperature, m_layout(layout_b),
            1 if accumulate else 0, self._handle_on(stream, device)))
