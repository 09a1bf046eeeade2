"""What a token model's operators launch, on the CPU (tests/launches.py): kernels, grids and streams."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from tests import launches
from tests import lm_cases as cases
from tests.launches import buf, in_child, recorded

F32, BF16, SILU = 0, 1, 14


def forward(kind, rows, inputs, hidden, act=SILU, shift=0, keep=True):
    from darknet_zig_amd import gpu

    shift *= 4 if kind == F32 else 2
    gpu.gatedForward(kind, rows, inputs, hidden, act, buf(1, shift), buf(2, shift), buf(3), buf(4, shift) if keep else None, buf(5, shift), buf(6))


def backward(kind, rows, inputs, hidden, act=SILU, shift=0, want=(1, 1, 1)):
    from darknet_zig_amd import gpu

    shift *= 4 if kind == F32 else 2
    gpu.gatedBackward(kind, rows, inputs, hidden, act, buf(1, shift), buf(2, shift), buf(3, shift), buf(4, shift), buf(5, shift), 0.5,
                      buf(6) if want[0] else None, buf(7, shift) if want[1] else None, buf(8, shift) if want[2] else None, buf(9))


def log_probs(kind, rows, classes, top=5, entropy=True):
    from darknet_zig_amd import gpu

    gpu.tokenLogProbs(kind, rows, classes, classes, buf(1), 1.0, 1, buf(2), top, buf(3), buf(4) if entropy else None, buf(5), buf(6), buf(7), buf(8))


def log_probs_backward(kind, rows, classes, entropy=True, beta=0.0):
    from darknet_zig_amd import gpu

    gpu.tokenLogProbsBackward(kind, rows, classes, classes, buf(1), 1.0, 1, buf(2), buf(3), buf(4), buf(5), buf(6) if entropy else None, beta, buf(7))


def distillation(kind, rows, classes, delta=True):
    from darknet_zig_amd import gpu

    gpu.distillation(kind, rows, classes, classes, buf(1), 1.0, 5, buf(2), buf(3), buf(4), 1.0, buf(5), buf(6) if delta else None, buf(7))


CALLS = {f.__name__: f for f in (forward, backward, log_probs, log_probs_backward, distillation)}


def load():
    """The names of libdkz_lm.so's kernels."""
    from darknet_zig_amd import _lib

    first = launches._lib.launches_kernels()
    _lib.load_lm()
    return [launches._lib.launches_kernel(i).decode() for i in range(first, launches._lib.launches_kernels())]


# ---- kernels ----


def kernels_of_the_cases():
    from darknet_zig_amd import _lib

    all_of_them, seen = load(), []
    for case in cases.FORWARD:
        seen += recorded(lambda: forward(*case))
    for case in cases.BACKWARD:
        seen += recorded(lambda: backward(*case))
    for case, want in cases.BACKWARD_PARTS:
        seen += recorded(lambda: backward(*case, want))
    for kind in (F32, BF16):
        for rows, classes in cases.ROWS:
            for entropy in (False, True):
                for top in (0, 5):
                    seen += recorded(lambda: log_probs(kind, rows, classes, top, entropy))
                for beta in (0.0, 1.0):
                    seen += recorded(lambda: log_probs_backward(kind, rows, classes, entropy, beta))
            for delta in (False, True):
                seen += recorded(lambda: distillation(kind, rows, classes, delta))
    names = {x.kernel for x in seen}
    return sorted(names), sorted(set(all_of_them) - names)


def test_the_cases_run_every_kernel():
    """So that no change of the rules leaves one without a GPU test."""
    seen, missing = in_child("tests.test_lm_launches:kernels_of_the_cases")
    assert not missing, (len(seen), missing)
    assert len(seen) > 60


# ---- streams ----

SEVERAL = [("forward", BF16, 40, 4097, 100), ("forward", F32, 256, 1000, 1003), ("backward", BF16, 300, 129, 101), ("backward", F32, 300, 129, 101),
           ("backward", BF16, 4096, 1024, 1024), ("log_probs", F32, 1, 65536), ("distillation", BF16, 2, 65536)]


def streams_of(name, *args):
    """The streams of a call's launches, another host thread setting another stream behind each."""
    from darknet_zig_amd import _lib

    load()
    lib = _lib.load()
    lib.dkz_set_stream(0x1000)
    return [x.stream for x in recorded(lambda: CALLS[name](*args), after=lambda: lib.dkz_set_stream(0x2000))]


@pytest.mark.parametrize("call", SEVERAL, ids=str)
def test_an_op_s_launches_are_of_one_stream(call):
    streams = in_child("tests.test_lm_launches:streams_of", *call)
    assert len(streams) > 1 and set(streams) == {0x1000}, streams


# ---- grids ----

LARGEST = [("log_probs", BF16, 1 << 26, 3), ("log_probs", F32, 1 << 12, 1 << 26), ("log_probs", F32, 1, 1 << 26), ("log_probs_backward", BF16, 1 << 26, 4096),
           ("log_probs_backward", F32, 1 << 12, 1 << 26), ("distillation", BF16, 1 << 26, 4096), ("distillation", BF16, 1 << 12, 1 << 26),
           ("distillation", F32, 1, 1 << 26), ("forward", BF16, 1 << 26, 8, 15, SILU, 1), ("forward", F32, 1 << 26, 31, 15),
           ("forward", BF16, 1, 31, 1 << 25, SILU, 1), ("backward", BF16, 1 << 26, 31, 15, SILU, 1), ("backward", F32, 1 << 26, 31, 15),
           ("backward", BF16, 31, 31, 1 << 25, SILU, 1), ("forward", BF16, 32768, 8, 32767, SILU, 1), ("backward", BF16, 32768, 8, 32767, SILU, 1)]


def grids_of(name, *args):
    load()
    most: dict[str, int] = {}
    for x in recorded(lambda: CALLS[name](*args)):
        most[x.kernel] = max(most.get(x.kernel, 0), x.threads)
    return most


@pytest.mark.parametrize("call", LARGEST, ids=str)
def test_a_launch_has_fewer_than_2_to_the_32_threads(call):
    most = in_child("tests.test_lm_launches:grids_of", *call)
    assert most and all(0 < threads < 2**32 for threads in most.values()), most


# Many rows of many classes, up to 2^38 logits: what parts of rows add up to.
LARGEST_OF_PARTS = [(name, kind, rows, classes) for name in ("log_probs", "log_probs_backward", "distillation")
                    for kind, rows, classes in [(F32, 1 << 20, 1 << 18), (BF16, 1 << 20, 1 << 18), (F32, 1000000, 65540), (BF16, 1000000, 131080),
                                                (BF16, 511, 1 << 26), (F32, 1 << 14, 1 << 24)]]


@pytest.mark.parametrize("call", [*LARGEST_OF_PARTS, ("distillation", F32, 1 << 20, 1 << 18, False)], ids=str)
def test_many_long_rows_have_fewer_than_2_to_the_32_threads(call):
    most = in_child("tests.test_lm_launches:grids_of", *call)
    assert most and all(0 < threads < 2**32 for threads in most.values()), most


# ---- workspaces ----

CLASSES = [0, 3, 1024, 16400, 32768, 40000, 50001, 65536, 65540, 131080, 262144, 1 << 20, 1 << 26]


def workspaces(kind):
    """What the queries of logits give for 0 to 1100 rows and some more of 2^26 classes at most, by classes and top."""
    from darknet_zig_amd import gpu

    load()
    more = [*range(1101), 2000, 1 << 14, 1 << 20, 1 << 26]
    out = []
    for classes in CLASSES:
        rows = [r for r in more if r * classes <= 1 << 38]
        for top in (0, 5, 64):
            out.append([f"log_probs {classes} {top}", [gpu.tokenLogProbsWorkspace(kind, r, classes, top) for r in rows]])
        out.append([f"distillation {classes}", [gpu.distillationWorkspace(kind, r, classes) for r in rows]])
    return out


@pytest.mark.parametrize("kind", [F32, BF16])
def test_a_workspace_of_logits_does_for_fewer_rows(kind):
    found = in_child("tests.test_lm_launches:workspaces", kind)
    for name, sizes in found:
        assert sizes == sorted(sizes), (name, [(i, a, b) for i, (a, b) in enumerate(zip(sizes, sizes[1:])) if a > b][:5])
    assert sum(sizes[-1] > 0 for _, sizes in found) > 20


def refused_with_the_workspace_of(kind, most, classes):
    """Of 1 .. `most` rows, those whose calls refuse a workspace for `most`."""
    from darknet_zig_amd import gpu

    load()
    refused = []
    words = lambda n: gpu.Buf(buf(9).ptr, n // 4) if n else None
    for top in (0, 5):
        ws = words(gpu.tokenLogProbsWorkspace(kind, most, classes, top))
        for rows in range(1, most + 1):
            try:
                recorded(lambda: gpu.tokenLogProbs(kind, rows, classes, classes, buf(1), 1.0, 0, None, top, None, None, buf(5), buf(6), buf(7), ws))
            except gpu.GpuError:
                refused.append(("log_probs", top, rows))
    ws = words(gpu.distillationWorkspace(kind, most, classes))
    for rows in range(1, most + 1):
        try:
            recorded(lambda: gpu.distillation(kind, rows, classes, classes, buf(1), 1.0, 5, buf(2), buf(3), None, 1.0, buf(5), buf(6), ws))
        except gpu.GpuError:
            refused.append(("distillation", rows))
    return refused


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("most,classes", [(600, 50001), (600, 65536), (300, 131080), (130, 150000)])
def test_a_call_of_fewer_rows_takes_the_workspace(kind, most, classes):
    assert in_child("tests.test_lm_launches:refused_with_the_workspace_of", kind, most, classes) == []


# ---- what the compiler is told ----


def _scalars(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]|s(\d+)", operand)
    return set() if m is None else {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def test_loads_to_lds_wait_for_the_scalars_of_vector_instructions(tmp_path):
    """As in libdkz_dense.so: five wait states between a vector instruction that writes a scalar register and a load to LDS, in an
    asm, that reads it."""
    objdump = Path("/opt/rocm/llvm/bin/llvm-objdump")
    if not objdump.exists():
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(launches.ROOT / "darknet_zig_amd" / "libdkz_lm.so", tmp_path)
    subprocess.run([objdump, "--offloading", lib], capture_output=True, check=True, cwd=tmp_path)
    loads = 0
    for code in sorted(tmp_path.glob("*gfx950")):
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", code], capture_output=True, text=True, check=True).stdout
        before: list[tuple[set[int], int, str]] = []
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
    assert loads > 100, loads
