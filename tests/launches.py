"""What the dense operators launch, without a GPU: in a process of its own the HIP
runtime's launch entry points are liblaunches.so's (native/launches.cpp), the
operators are called with addresses that nothing reads, and every launch is
written down.

`in_child("module:function", ...)` runs a function there and returns its result; in
that process `recorded(call)` makes a call and returns its launches."""

from __future__ import annotations

import ctypes as C
import importlib
import json
import subprocess
import sys
from pathlib import Path
from typing import Callable, NamedTuple

from tests.native import build as native_build

ROOT = Path(__file__).resolve().parents[1]


class Launch(NamedTuple):
    kernel: str  # "translation unit:mangled name"
    grid: tuple[int, int, int]
    block: tuple[int, int, int]
    stream: int

    @property
    def threads(self) -> int:
        g, b = self.grid, self.block
        return g[0] * b[0] * g[1] * b[1] * g[2] * b[2]


def in_child(function: str, *args):
    proc = subprocess.run([sys.executable, "-m", "tests.launches", function, json.dumps(args)], cwd=ROOT, capture_output=True, text=True,
                          timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    assert "Traceback" not in proc.stderr, proc.stderr  # an error in a callback is only printed
    return json.loads(proc.stdout.splitlines()[-1])


# ---- in the child ----

_lib = _callback_type = None
dense_kernels: list[str] = []


def _start() -> None:
    """Loads the stand-ins, then the libraries."""
    global _lib, _callback_type
    _lib = C.CDLL(str(native_build.LAUNCHES), mode=C.RTLD_GLOBAL)
    _lib.launches_kernel.restype = C.c_char_p
    _callback_type = C.CFUNCTYPE(None, C.c_char_p, C.POINTER(C.c_uint), C.POINTER(C.c_uint), C.c_void_p)
    from darknet_zig_amd import _lib as package

    package.load()
    first = _lib.launches_kernels()
    assert first > 0, "the libraries do not take liblaunches.so's entry points"
    package.load_dense()
    dense_kernels.extend(_lib.launches_kernel(i).decode() for i in range(first, _lib.launches_kernels()))


def recorded(call: Callable[[], object], after: Callable[[], object] | None = None) -> list[Launch]:
    """The launches of call(); `after` is called behind each."""
    seen: list[Launch] = []

    def take(name, grid, block, stream):
        seen.append(Launch(name.decode(), tuple(grid[:3]), tuple(block[:3]), stream or 0))
        if after is not None:
            after()

    callback = _callback_type(take)
    _lib.launches_to(callback)
    try:
        call()
    finally:
        _lib.launches_to(None)
    return seen


def buf(i: int, shift: int = 0):
    """A buffer of a region of its own, `shift` bytes off its alignment; nothing reads it."""
    from darknet_zig_amd import gpu

    return gpu.Buf((i << 40) + shift, 1 << 37)


if __name__ == "__main__":
    from tests import launches  # the module that the called function imports, not __main__

    launches._start()
    module, name = sys.argv[1].split(":")
    print(json.dumps(getattr(importlib.import_module(module), name)(*json.loads(sys.argv[2]))))
