"""The C ABI of libdkz_dense.so as a boundary: declared == exported == bound, and
what it refuses before any HIP call (no GPU needed)."""

from __future__ import annotations

import ctypes as C
import inspect
import re
import shutil
import subprocess

import pytest

from darknet_zig_amd import _lib, gpu

ROOT = _lib.LIB_PATH.parents[1]
HEADER = ROOT / "include" / "dkz_dense.h"
LIB = _lib.LIB_PATH.parent / _lib.DENSE_LIB_NAME
OK, INVALID = 0, 1
F32, BF16 = gpu.F32, gpu.BF16
LINEAR, RELU = 3, 1


def at(n: int) -> C.c_void_p:
    """A pointer value of its own region; never dereferenced in these calls."""
    return C.c_void_p(n << 32)


X, W, B, A, D, R, Y, Z, WS = (at(i) for i in range(1, 10))
BIG = 1 << 40


def header_symbols() -> list[str]:
    return re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(dkz_\w+)\s*\(", HEADER.read_text(), flags=re.M)


def test_header_exports_and_binding_agree():
    out = subprocess.run(["nm", "-D", "--defined-only", str(LIB)], capture_output=True, text=True, check=True).stdout
    names = sorted(ln.split()[-1] for ln in out.splitlines() if len(ln.split()) >= 3)
    assert names == sorted(header_symbols())
    assert list(_lib.DENSE_SIGNATURES) == header_symbols()


def test_bound_arities_are_the_header_s():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for name, params in re.findall(r"(dkz_\w+)\s*\(([^)]*)\)\s*;", text):
        n = 0 if params.strip() == "void" else len(params.split(","))
        assert len(_lib.DENSE_SIGNATURES[name][1]) == n, name


def test_the_companion_shares_the_library_s_state():
    """It loads the libdkz.so beside it: one stream, one sync-after-launch switch."""
    out = subprocess.run(["readelf", "-d", str(LIB)], capture_output=True, text=True, check=True).stdout
    assert "[libdkz.so]" in out and "$ORIGIN" in out
    _lib.load_dense()
    maps = {ln.split()[-1] for ln in open("/proc/self/maps") if ln.rstrip().endswith("libdkz.so")}
    assert len(maps) == 1


def dropout(L, n=8, xt=F32, x=X, r=None, prob=0.5, yt=F32, y=Y):
    return L.dkz_seeded_dropout(n, xt, x, r, prob, 2.0, 1, 0, yt, y)


@pytest.mark.parametrize("kw,want", [
    (dict(n=-1), INVALID), (dict(n=0, x=None, y=None), OK), (dict(xt=2), INVALID), (dict(yt=-1), INVALID), (dict(x=None), INVALID),
    (dict(y=None), INVALID), (dict(y=X, yt=BF16), INVALID),  # in place between types
    (dict(y=C.c_void_p(X.value + 4)), INVALID),  # overlaps x by all but one element
    (dict(r=C.c_void_p(Y.value + 16)), INVALID),  # the residual overlaps the output
], ids=str)
def test_dropout_refusals(kw, want):
    assert dropout(_lib.load_dense(), **kw) == want


def forward(L, type=BF16, rows=4, inputs=8, outputs=6, act=RELU, x=X, w=W, b=B, r=None, a=None, y=Y, ws=WS, ws_bytes=BIG):
    return L.dkz_linear_forward(type, rows, inputs, outputs, act, 0.0, 1.0, 0, 0, x, w, b, r, a, y, ws, ws_bytes)


@pytest.mark.parametrize("kw,want", [
    (dict(type=2), INVALID), (dict(rows=-1), INVALID), (dict(inputs=-1), INVALID), (dict(outputs=-1), INVALID), (dict(act=14), INVALID),
    (dict(act=-1), INVALID), (dict(rows=0, x=None, w=None, y=None), OK), (dict(outputs=0, x=None, w=None, y=None), OK),
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(y=None), INVALID), (dict(y=X), INVALID), (dict(y=W), INVALID),
    (dict(y=B), INVALID), (dict(a=Y), INVALID), (dict(a=R, r=R), INVALID), (dict(r=C.c_void_p(Y.value + 2)), INVALID), (dict(a=X), INVALID),
    (dict(rows=65536, inputs=8, outputs=32768), INVALID), (dict(rows=1 << 30, inputs=2, outputs=1), INVALID),
    (dict(rows=1, inputs=1, outputs=(1 << 26) + 1), INVALID), (dict(rows=(1 << 26) + 1, inputs=1, outputs=1), INVALID),
    (dict(rows=1, inputs=(1 << 26) + 1, outputs=1), INVALID),
], ids=str)
def test_linear_forward_refusals(kw, want):
    assert forward(_lib.load_dense(), **kw) == want


def test_linear_forward_workspace_is_checked():
    L = _lib.load_dense()
    need = gpu.linearForwardWorkspace(F32, 256, 4096, 4096)
    assert need > 0
    shape = dict(type=F32, rows=256, inputs=4096, outputs=4096)
    assert forward(L, **shape, ws_bytes=need - 1) == INVALID
    assert forward(L, **shape, ws=None, ws_bytes=need) == INVALID
    assert forward(L, **shape, ws=C.c_void_p(WS.value + 8), ws_bytes=need) == INVALID
    assert forward(L, **shape, ws=Y, ws_bytes=need) == INVALID
    assert forward(L, **shape, ws=X, ws_bytes=need) == INVALID
    assert b"dkz_linear_forward" in L.dkz_dense_last_error_context()


def backward(L, type=BF16, rows=4, inputs=8, outputs=6, act=RELU, x=X, w=W, a=A, d=D, r=None, gb=B, gw=Y, gx=Z, ws=WS, ws_bytes=BIG):
    return L.dkz_linear_backward(type, rows, inputs, outputs, act, 0.0, 1.0, 0, 0, x, w, a, d, r, 0.0, gb, gw, gx, ws, ws_bytes)


@pytest.mark.parametrize("kw,want", [
    (dict(type=-1), INVALID), (dict(rows=-1), INVALID), (dict(act=14), INVALID), (dict(a=None), INVALID), (dict(d=None), INVALID),
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(gx=Y), INVALID), (dict(gw=W), INVALID), (dict(gx=X), INVALID), (dict(gb=D), INVALID),
    (dict(gx=D), INVALID), (dict(r=Y), INVALID), (dict(r=C.c_void_p(Z.value + 2)), INVALID), (dict(ws=None), INVALID),
    (dict(ws_bytes=16), INVALID), (dict(ws=C.c_void_p(WS.value + 4)), INVALID), (dict(ws=D), INVALID), (dict(rows=65536, inputs=65536), INVALID),
], ids=str)
def test_linear_backward_refusals(kw, want):
    assert backward(_lib.load_dense(), **kw) == want


def loss(L, type=BF16, rows=4, inputs=8, classes=600, x=X, w=W, b=B, t=A, l=Y, lse=Z, ws=WS, ws_bytes=BIG):
    return L.dkz_linear_cross_entropy_forward(type, rows, inputs, classes, x, w, b, t, l, lse, ws, ws_bytes)


@pytest.mark.parametrize("kw,want", [
    (dict(type=3), INVALID), (dict(rows=-1), INVALID), (dict(classes=-1), INVALID), (dict(rows=0, x=None, w=None, t=None, l=None, lse=None), OK),
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(t=None), INVALID), (dict(l=None), INVALID), (dict(lse=None), INVALID),
    (dict(l=Z), INVALID), (dict(l=A), INVALID), (dict(ws=None), INVALID), (dict(ws_bytes=64), INVALID), (dict(ws=W), INVALID),
    (dict(ws=C.c_void_p(WS.value + 4)), INVALID), (dict(inputs=1 << 16, classes=1 << 16), INVALID),
    (dict(inputs=1, classes=(1 << 26) + 1), INVALID), (dict(rows=1 << 20, inputs=1, classes=1 << 19), INVALID),
], ids=str)
@pytest.mark.parametrize("type", [F32, BF16])
def test_cross_entropy_forward_refusals(kw, want, type):
    assert loss(_lib.load_dense(), **{"type": type, **kw}) == want


def grad(L, type=BF16, rows=4, inputs=8, classes=600, x=X, w=W, b=B, t=A, lse=D, s=None, gb=R, gw=Y, gx=Z, ws=WS, ws_bytes=BIG):
    return L.dkz_linear_cross_entropy_backward(type, rows, inputs, classes, x, w, b, t, lse, s, 1.0, 0.0, gb, gw, gx, ws, ws_bytes)


@pytest.mark.parametrize("kw,want", [
    (dict(type=3), INVALID), (dict(rows=-1), INVALID), (dict(gb=None, gw=None, gx=None, x=None), OK), (dict(x=None), INVALID),
    (dict(w=None), INVALID), (dict(t=None), INVALID), (dict(lse=None), INVALID), (dict(gw=W), INVALID), (dict(gx=X), INVALID),
    (dict(gx=Y), INVALID), (dict(gb=B), INVALID), (dict(gb=D), INVALID), (dict(ws=None), INVALID), (dict(ws_bytes=64), INVALID),
    (dict(ws=X), INVALID), (dict(inputs=1 << 16, classes=1 << 16), INVALID),
], ids=str)
@pytest.mark.parametrize("type", [F32, BF16])
def test_cross_entropy_backward_refusals(kw, want, type):
    assert grad(_lib.load_dense(), **{"type": type, **kw}) == want


@pytest.mark.parametrize("type", [F32, BF16])
@pytest.mark.parametrize("rows,inputs,classes", [(1, 8, 5), (333, 1030, 9001), (4096, 4096, 65536), (8192, 512, 200001)])
def test_cross_entropy_workspaces(type, rows, inputs, classes):
    """The least one holds pieces of the classes, the best one no more than half a gigabyte of logits and its sums."""
    for f in (gpu.linearCrossEntropyForwardWorkspace, gpu.linearCrossEntropyBackwardWorkspace):
        least, best = f(type, rows, inputs, classes)
        assert 0 < least <= best
        assert best < (1 << 30) + 64 * rows * inputs + rows * classes // 4


@pytest.mark.parametrize("type", [F32, BF16])
@pytest.mark.parametrize("rows,inputs,classes", [(1, 1 << 20, 300), (40, 8, 300), (500, 2000, 300), (64, 1 << 18, 1000)])
def test_the_least_workspace_is_the_least(type, rows, inputs, classes):
    """Also where one piece of all classes takes less than several, which add up the input's gradient in fp32."""
    for f in (gpu.linearCrossEntropyForwardWorkspace, gpu.linearCrossEntropyBackwardWorkspace):
        least, best = f(type, rows, inputs, classes)
        assert least <= best
    L = _lib.load_dense()
    args = dict(type=type, rows=rows, inputs=inputs, classes=classes)
    assert grad(L, **args, ws_bytes=least - 256) == INVALID


@pytest.mark.parametrize("call", [
    lambda p: _lib.load_dense().dkz_linear_forward_workspace(2, 1, 1, 1, p),
    lambda p: _lib.load_dense().dkz_linear_forward_workspace(F32, -1, 1, 1, p),
    lambda p: _lib.load_dense().dkz_linear_forward_workspace(F32, 1, 1, 1, None),
    lambda p: _lib.load_dense().dkz_linear_backward_workspace(F32, 65536, 65536, 1, p),
    lambda p: _lib.load_dense().dkz_linear_cross_entropy_forward_workspace(F32, 1, 1, -1, p, p),
    lambda p: _lib.load_dense().dkz_linear_cross_entropy_backward_workspace(F32, 1, 1, 1, p, None),
])
def test_workspace_queries_refuse(call):
    assert call(C.byref(C.c_size_t(0))) == INVALID


# ---- the other hosts' bindings ----

ZIG = ROOT / "darknet_zig_amd" / "zig" / "dkz_dense.zig"
WRAPPERS = ["seededDropout", "linearForwardWorkspace", "linearForward", "linearBackwardWorkspace", "linearBackward",
            "linearCrossEntropyForwardWorkspace", "linearCrossEntropyForward", "linearCrossEntropyBackwardWorkspace",
            "linearCrossEntropyBackward"]


def header_params() -> dict[str, list[tuple[str, str]]]:
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    out = {}
    for name, params in re.findall(r"(dkz_\w+)\s*\(([^)]*)\)\s*;", text):
        ps = [] if params.strip() == "void" else [" ".join(p.split()) for p in params.split(",")]
        out[name] = [re.match(r"(.*?)(\w+)$", p).groups() for p in ps]
    return out


def zig_type(ctype: str) -> str:
    base = ctype.replace("const ", "").replace(" ", "")
    return {"int": "c_int", "float": "f32", "unsignedint": "c_uint", "unsignedlonglong": "c_ulonglong", "size_t": "usize",
            "size_t*": "*usize"}.get(base, "?*anyopaque")


def test_zig_externs_follow_the_header():
    externs = re.findall(r"^pub extern fn (dkz_\w+)\((.*)\) (.+);$", ZIG.read_text(), flags=re.M)
    params = header_params()
    assert [e[0] for e in externs] == list(params) == header_symbols()
    for name, ps, ret in externs:
        got = [tuple(p.split(": ", 1)) for p in ps.split(", ")] if ps else []
        assert got == [(n, zig_type(t)) for t, n in params[name]], name
        assert ret == ("[*:0]const u8" if name.endswith("context") else "Status")


def test_zig_wrappers_pass_every_argument_in_order():
    text = ZIG.read_text()
    params = header_params()
    for name in WRAPPERS:
        m = re.search(r"^pub fn " + name + r"\((.*?)\) [\w.]+ \{\n(.*?)^\}", text, flags=re.M | re.S)
        assert m, name
        body = m.group(2)
        assert body.strip().startswith("if (!gpu.enabled) unreachable;")
        call = re.search(r"must\((dkz_\w+)\((.*)\), \"", body)
        args = re.sub(r"\bci\((\w+)\)", r"\1", call.group(2)).split(", ")
        assert len(args) == len(params[call.group(1)]), name
        for arg, (_, want) in zip(args, params[call.group(1)]):
            bare = re.sub(r"^&need(\.)?|\.ptr$", "", arg)
            assert bare in (want, "", "type_code" if want == "type" else want) or arg == "bytes(workspace)" and want == "workspace_bytes", (
                name, arg, want)


@pytest.mark.parametrize("name", WRAPPERS)
def test_python_and_cpp_wrappers_take_the_same_arguments(name):
    cpp = (ROOT / "darknet_zig_amd" / "host" / "dkz_dense.hpp").read_text()
    m = re.search(r"inline [\w:]+ " + name + r"\((.*?)\) \{", cpp, flags=re.S)
    assert [p.split()[-1] for p in m.group(1).split(",")] == list(inspect.signature(getattr(gpu, name)).parameters)


def test_cpp_mirror_compiles_links_and_refuses(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    src = tmp_path / "dense.cpp"
    src.write_text('''#include <cstdio>
#include "dkz_dense.hpp"
using namespace dkz::gpu;
int main() {
    if (linearForwardWorkspace(DKZ_F32, 256, 4096, 4096) == 0) return 1;
    const Workspaces w = linearCrossEntropyBackwardWorkspace(DKZ_BF16, 64, 128, 5000);
    if (w.least == 0 || w.best < w.least) return 2;
    seededDropout(0, DKZ_F32, Buf{}, Buf{}, 0.5f, 2.0f, 1, 0, DKZ_F32, Buf{});
    try {
        linearForward(DKZ_BF16, 4, 8, 6, 99, 0.0f, 1.0f, 0, 0, Buf{}, Buf{}, Buf{}, Buf{}, Buf{}, Buf{}, Buf{});
        return 3;
    } catch (const Error &e) {
        std::puts(e.what());
        return e.code() == 1 ? 0 : 4;
    }
}
''')
    lib = LIB.parent
    exe = tmp_path / "dense"
    proc = subprocess.run([gxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'include'}", f"-I{lib / 'host'}", str(src), "-o",
                           str(exe), f"-L{lib}", "-ldkz_dense", "-ldkz", f"-Wl,-rpath,{lib}", "-Wl,-rpath-link,/opt/rocm/lib"],
                          capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "dkz_linear_forward" in run.stdout, (run.returncode, run.stdout)
