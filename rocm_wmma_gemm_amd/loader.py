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
                    ("orthogonalize", [i, i, p, p, z, z, z, i, p, ctypes.c_float, p])):
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
        if t.get_device() != device:
            raise ValueError(f"{name} must be a device tensor" if not t.is_cuda else
                             f"{name} is on device {t.get_device()}, the other operands on {device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be densely packed")
        if t.dtype is not dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        if t.numel() < need:
            raise ValueError(f"{name} holds {t.numel()} elements, the problem needs {need}")
        return t.data_ptr()

    @staticmethod
    def _stream_on(stream, device):
        """Handle of `stream`, or of torch's current one on `device` (whose stream object takes 3 us
        to make, a third of a small call)."""
        if stream is None:
            import torch

            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
            return raw(device) if raw is not None else int(torch.cuda.current_stream(device).cuda_stream)
        return Loader._stream_handle(stream)

    @staticmethod
    def _device_of(name, t):
        import torch

        device = t.get_device()
        if device < 0:
            raise ValueError(f"{name} must be a device tensor")
        if device != torch.cuda.current_device():  # (whose scratch buffer and streams the library uses)
            raise ValueError(f"{name} is on device {device}, the current one is {torch.cuda.current_device()}")
        return device

    @staticmethod
    def _sizes(*sizes):
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
