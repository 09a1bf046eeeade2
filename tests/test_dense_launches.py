"""What the dense operators launch, on the CPU (tests/launches.py): kernels, grids and streams."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from tests import dense_cases as cases
from tests import launches
from tests.launches import buf, in_child, recorded

F32, BF16, LEAKY = 0, 1, 7


def forward(kind, rows, inputs, outputs, shift=0, act=LEAKY):
    from darknet_zig_amd import gpu

    gpu.linearForward(kind, rows, inputs, outputs, act, 0.5, 2.0, 1, 0, buf(1, shift), buf(2, shift), buf(3), buf(4, shift), buf(5, shift),
                      buf(6, shift), buf(7))


def backward(kind, rows, inputs, outputs, shift=0, act=LEAKY):
    from darknet_zig_amd import gpu

    gpu.linearBackward(kind, rows, inputs, outputs, act, 0.5, 2.0, 1, 0, buf(1, shift), buf(2, shift), buf(3, shift), buf(4, shift),
                       buf(5, shift), 0.5, buf(6), buf(7, shift), buf(8, shift), buf(9))


def loss(kind, rows, inputs, classes, least=False, shift=0):
    from darknet_zig_amd import gpu

    ws = gpu.Buf(buf(7).ptr, gpu.linearCrossEntropyForwardWorkspace(kind, rows, inputs, classes)[0 if least else 1] // 4)
    gpu.linearCrossEntropyForward(kind, rows, inputs, classes, buf(1, shift), buf(2, shift), buf(3), buf(4), buf(5), buf(6), ws)


def gradients(kind, rows, inputs, classes, least=False, shift=0, between=False):
    from darknet_zig_amd import gpu

    sizes = gpu.linearCrossEntropyBackwardWorkspace(kind, rows, inputs, classes)
    ws = gpu.Buf(buf(10).ptr, (cases.between(sizes) if between else sizes[0 if least else 1]) // 4)
    gpu.linearCrossEntropyBackward(kind, rows, inputs, classes, buf(1, shift), buf(2, shift), buf(3), buf(4), buf(5), buf(6), 1.0, 0.5, buf(7),
                                   buf(8, shift), buf(9, shift), ws)


CALLS = {"forward": forward, "backward": backward, "loss": loss, "gradients": gradients}


# ---- streams ----

# Ops of several launches each: packing, ranges of K and their join, delta and its sums, pieces of the classes.
SEVERAL = [("forward", BF16, 40, 4097, 100), ("forward", F32, 256, 4096, 4096), ("backward", BF16, 300, 129, 200),
           ("backward", BF16, 8192, 4096, 4096), ("backward", F32, 300, 129, 200), ("loss", BF16, 200, 65, 1000),
           ("loss", F32, 200, 65, 1000, True), ("gradients", BF16, 200, 65, 1000, True), ("gradients", F32, 200, 65, 1000, True),
           ("gradients", BF16, 128, 4096, 1000)]


def streams_of(name, *args):
    """The streams of a call's launches, another host thread setting another stream behind each."""
    from darknet_zig_amd import _lib

    lib = _lib.load()
    lib.dkz_set_stream(0x1000)
    return [x.stream for x in recorded(lambda: CALLS[name](*args), after=lambda: lib.dkz_set_stream(0x2000))]


@pytest.mark.parametrize("call", SEVERAL, ids=str)
def test_an_op_s_launches_are_of_one_stream(call):
    streams = in_child("tests.test_dense_launches:streams_of", *call)
    assert len(streams) > 1 and set(streams) == {0x1000}, streams


# ---- the host's part of a call ----


def host_time(shapes):
    """us of the host in a call of the loss and of its gradients, nothing being launched: the least of many."""
    from time import perf_counter

    from darknet_zig_amd import _lib, gpu

    lib, out = _lib.load_dense(), []
    p = [buf(i).ptr for i in range(12)]
    for kind, rows, inputs, classes, least in shapes:
        need = [f(kind, rows, inputs, classes)[0 if least else 1]
                for f in (gpu.linearCrossEntropyForwardWorkspace, gpu.linearCrossEntropyBackwardWorkspace)]
        ends = []
        for call in (lambda: lib.dkz_linear_cross_entropy_forward(kind, rows, inputs, classes, p[1], p[2], p[3], p[4], p[5], p[6], p[7], need[0]),
                     lambda: lib.dkz_linear_cross_entropy_backward(kind, rows, inputs, classes, p[1], p[2], p[3], p[4], p[6], None, 1.0, 0.0,
                                                                   p[8], p[9], p[10], p[11], need[1])):
            best = 1.0
            for _ in range(30):
                t = perf_counter()
                for _ in range(20):
                    assert call() == 0
                best = min(best, (perf_counter() - t) / 20)
            ends.append(best * 1e6)
        out.append(ends)
    return out


def test_the_gradients_are_planned_as_often_as_they_are_needed():
    """A backward pass is at most three products where a forward pass is one, so its host time is a few times the forward's;
    it was 15 to 30 times that when every call searched for the smallest workspace."""
    shapes = [(kind, *shape, least) for kind in (F32, BF16) for shape in ((1, 432, 8493), (8, 1024, 1000), (128, 4096, 1000))
              for least in (False, True)]
    for shape, (forth, back) in zip(shapes, in_child("tests.test_dense_launches:host_time", shapes)):
        print(shape, round(forth, 1), round(back, 1))
        assert shape[-1] or back < 6 * forth + 4, (shape, forth, back)


# ---- kernels ----


def kernels_of_the_cases():
    """The kernels that the cases launch of those that the library has, and those that none does."""
    from darknet_zig_amd import gpu

    seen = []
    for kind, rows, inputs, outputs, act, shift in cases.FORWARD:
        seen += recorded(lambda: forward(kind, rows, inputs, outputs, shift * (4 if kind == F32 else 2), act))
    for kind, rows, inputs, outputs, act, shift in cases.BACKWARD:
        seen += recorded(lambda: backward(kind, rows, inputs, outputs, shift * (4 if kind == F32 else 2), act))
    for kind, rows, inputs, classes, least, shift in cases.LOSS:
        for f in (loss, gradients):
            seen += recorded(lambda: f(kind, rows, inputs, classes, least, shift * (4 if kind == F32 else 2)))
    for shape in cases.PIECES:
        seen += recorded(lambda: gradients(BF16, *shape, between=True))
    for x, y in ((F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)):  # all of them in the tests of dropout
        seen += recorded(lambda: gpu.seededDropout(100, x, buf(1), None, 0.5, 2.0, 1, 0, y, buf(2)))
    seen += recorded(lambda: gpu.linearCrossEntropyForward(F32, 5, 8, 0, None, None, None, buf(1), buf(2), buf(3), None))
    names = {x.kernel for x in seen}
    return sorted(names), sorted(set(launches.dense_kernels) - names)


def test_the_cases_run_every_kernel():
    """So that no change of the rules leaves one without a GPU test (test_gpu_dense_kernels.py)."""
    seen, missing = in_child("tests.test_dense_launches:kernels_of_the_cases")
    assert not missing, missing
    assert len(seen) > 180


# ---- grids ----

# The most logits that a loss takes (2^38), in products through registers (the inputs' base off a 16-byte boundary, which are not
# copied to the workspace: their rows are whole eights), and tensors of the most rows and columns.
LARGEST = [("loss", BF16, 4096, 8, 1 << 26, False, 2), ("loss", BF16, 4096, 8, 1 << 26), ("loss", BF16, 1 << 26, 8, 4096, False, 2),
           ("loss", F32, 4096, 8, 1 << 26), ("gradients", BF16, 4096, 8, 1 << 26, False, 2), ("gradients", F32, 4096, 8, 1 << 26),
           ("gradients", BF16, 1 << 26, 8, 4096, False, 2), ("gradients", F32, 1 << 26, 8, 4096), ("forward", BF16, 1 << 26, 8, 31, 2),
           ("forward", F32, 1 << 26, 31, 31), ("forward", BF16, 1, 31, 1 << 26, 2), ("backward", BF16, 1 << 26, 31, 31, 2),
           ("backward", F32, 1 << 26, 31, 31), ("backward", BF16, 31, 31, 1 << 26, 2), ("backward", BF16, 31, 1 << 26, 31),
           ("forward", BF16, 46340, 8, 46340, 2), ("backward", BF16, 46340, 8, 46340, 2)]


def grids_of(name, *args):
    seen = recorded(lambda: CALLS[name](*args))
    # Few are looked at: the largest of each kernel.
    most: dict[str, int] = {}
    for x in seen:
        most[x.kernel] = max(most.get(x.kernel, 0), x.threads)
    return most


@pytest.mark.parametrize("call", LARGEST, ids=str)
def test_a_launch_has_fewer_than_2_to_the_32_threads(call):
    most = in_child("tests.test_dense_launches:grids_of", *call)
    assert most and all(0 < threads < 2**32 for threads in most.values()), most


# ---- what the compiler is told ----


def test_asm_names_the_registers_that_it_writes():
    """m0 is no operand: an asm that writes it has to say so, or the compiler may keep a value there."""
    for path in sorted((launches.ROOT / "darknet_zig_amd").rglob("*.h*")):
        for text in re.findall(r"\basm\b[^;]*;", path.read_text()):
            if re.search(r"\bs_\w+ m0,", text):
                assert re.search(r':[^:]*"m0"[^:]*\)\s*;$', text), (path.name, text)


def _scalars(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]|s(\d+)", operand)
    return set() if m is None else {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def test_loads_to_lds_wait_for_the_scalars_of_vector_instructions(tmp_path):
    """A vector memory instruction may read a scalar register that a vector instruction wrote five wait states before, not sooner. The
    compiler sees to that but inside an asm, where the loads to LDS are: in the code that it built none of their scalars comes so late."""
    objdump = Path("/opt/rocm/llvm/bin/llvm-objdump")
    if not objdump.exists():
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(launches.ROOT / "darknet_zig_amd" / "libdkz_dense.so", tmp_path)
    subprocess.run([objdump, "--offloading", lib], capture_output=True, check=True, cwd=tmp_path)
    loads = 0
    for code in sorted(tmp_path.glob("*gfx950")):
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", code], capture_output=True, text=True, check=True).stdout
        before: list[tuple[set[int], int, str]] = []  # the last instructions: scalars that a vector one wrote, wait states, text
        for line in text.splitlines():
            m = re.match(r"\s+([a-z]\w+)(.*?)\s*//", line)
            if not m:
                continue
            op, args = m[1], [x.strip() for x in m[2].split(",")]
            if op == "buffer_load_dwordx4" and "lds" in m[2]:
                loads += 1
                need, waited = _scalars(args[1]), 0
                assert len(need) == 4, line
                for written, states, what in reversed(before):
                    assert waited >= 5 or not written & need, (what, line)
                    waited += states
            written = set().union(*(_scalars(a) for a in args[:2 if "_co_" in op else 1])) if op.startswith("v_") else set()
            before = before[-8:] + [(written, int(args[0], 0) + 1 if op == "s_nop" else 1, line)]
    assert loads > 500, loads
