"""What calls of the layer products would launch, asked in a process of its own where the HIP runtime's
calls are stood in for (hip_recorder.cpp): ``python recorded_launches.py <recorder.so> <calls as JSON>``.

A call is [entry point, arguments]; an argument "p" is the address of an operand, "s" coefficients, null a null
pointer.  ["fail", n] lets the n-th launch of the next call fail.  Prints, for every call, its status and
[grid x, y, z, block x, failed] of its launches.
"""
import ctypes
import json
import os
import sys


class Launch(ctypes.Structure):
    _fields_ = [("grid", ctypes.c_uint32 * 3), ("block", ctypes.c_uint32 * 3), ("failed", ctypes.c_int32)]


def main():
    recorder = ctypes.CDLL(sys.argv[1], mode=os.RTLD_NOW | os.RTLD_GLOBAL)
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    import rocm_wmma_gemm_amd as R

    library = R.Loader(arch="gfx950")._lib
    operand, steps = ctypes.c_void_p(1 << 20), (ctypes.c_float * 3)(1.5, -0.5, 0.0)
    answers = []
    for name, args in json.loads(sys.argv[2]):
        if name == "fail":
            recorder.recorder_fail(args)
            continue
        rc = getattr(library, "rocm_wmma_gemm_" + name)(*[operand if a == "p" else steps if a == "s" else a for a in args])
        seen = (Launch * 4096)()
        n = recorder.recorder_take(seen, 4096)
        answers.append([rc, [list(x.grid) + [x.block[0], x.failed] for x in seen[:n]]])
    print(json.dumps(answers))


if __name__ == "__main__":
    main()
