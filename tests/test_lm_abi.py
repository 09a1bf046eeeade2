"""The C ABI of libdkz_lm.so as a boundary: declared == exported == bound, and what it refuses before any HIP call (no GPU
needed)."""

from __future__ import annotations

import ctypes as C
import inspect
import re
import shutil
import subprocess

import pytest

from darknet_zig_amd import _lib, gpu

from .test_dense_abi import BIG, INVALID, OK, at, zig_type

ROOT = _lib.LIB_PATH.parents[1]
HEADER = ROOT / "include" / "dkz_lm.h"
LIB = _lib.LIB_PATH.parent / _lib.LM_LIB_NAME
F32, BF16 = gpu.F32, gpu.BF16
P = [at(i) for i in range(1, 14)]


def symbols() -> list[str]:
    return re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(dkz_\w+)\s*\(", HEADER.read_text(), flags=re.M)


def header_params() -> dict[str, list[tuple[str, str]]]:
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    out = {}
    for name, params in re.findall(r"(dkz_\w+)\s*\(([^)]*)\)\s*;", text):
        ps = [] if params.strip() == "void" else [" ".join(p.split()) for p in params.split(",")]
        out[name] = [re.match(r"(.*?)(\w+)$", p).groups() for p in ps]
    return out


def test_header_exports_and_binding_agree():
    out = subprocess.run(["nm", "-D", "--defined-only", str(LIB)], capture_output=True, text=True, check=True).stdout
    assert sorted(ln.split()[-1] for ln in out.splitlines() if len(ln.split()) >= 3) == sorted(symbols())
    assert list(_lib.LM_SIGNATURES) == symbols()


def test_bound_types_are_the_header_s():
    of = {"int": C.c_int, "float": C.c_float, "size_t": C.c_size_t, "size_t*": C.POINTER(C.c_size_t)}
    for name, params in header_params().items():
        assert _lib.LM_SIGNATURES[name][1] == [of.get(t.replace(" ", ""), C.c_void_p) for t, _ in params], name


def test_it_shares_the_library_s_state():
    out = subprocess.run(["readelf", "-d", str(LIB)], capture_output=True, text=True, check=True).stdout
    assert "[libdkz.so]" in out and "$ORIGIN" in out
    _lib.load_lm()
    assert len({ln.split()[-1] for ln in open("/proc/self/maps") if ln.rstrip().endswith("libdkz.so")}) == 1


def off(p, n):
    return C.c_void_p(p.value + n)


def forward(L, type=BF16, rows=4, inputs=8, hidden=6, act=14, x=P[0], w=P[1], b=P[2], s=P[3], y=P[4], ws=P[5], n=BIG):
    return L.dkz_gated_forward(type, rows, inputs, hidden, act, x, w, b, s, y, ws, n)


@pytest.mark.parametrize("kw,want", [
    (dict(type=2), INVALID), (dict(rows=-1), INVALID), (dict(inputs=-1), INVALID), (dict(hidden=-1), INVALID), (dict(act=2), INVALID),
    (dict(act=16), INVALID), (dict(act=-1), INVALID), (dict(rows=0, x=None, w=None, y=None), OK), (dict(hidden=0, x=None, w=None, y=None), OK),
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(y=None), INVALID), (dict(y=P[0]), INVALID), (dict(y=P[1]), INVALID),
    (dict(y=P[3]), INVALID), (dict(s=P[0]), INVALID), (dict(s=P[2]), INVALID), (dict(y=off(P[3], 94)), INVALID),
    (dict(w=off(P[4], -8 * 12 * 2 + 2)), INVALID), (dict(rows=1 << 15, hidden=1 << 15), INVALID), (dict(hidden=(1 << 25) + 1, inputs=1, rows=1), INVALID),
    (dict(rows=(1 << 26) + 1, inputs=1, hidden=1), INVALID), (dict(inputs=1 << 16, hidden=1 << 14), INVALID),
], ids=str)
def test_gated_forward_refusals(kw, want):
    assert forward(_lib.load_lm(), **kw) == want


@pytest.mark.parametrize("type", [F32, BF16])
def test_gated_forward_workspace_is_checked(type):
    L = _lib.load_lm()
    shape = dict(type=type, rows=333, inputs=1001, hidden=1503)
    need = gpu.gatedForwardWorkspace(type, 333, 1001, 1503)
    assert need > 0
    for kw in (dict(n=need - 1), dict(ws=None), dict(ws=off(P[5], 8)), dict(ws=P[0]), dict(ws=P[4])):
        assert forward(L, **{**shape, "n": need, **kw}) == INVALID
    assert b"dkz_gated_forward" in L.dkz_lm_last_error_context()


def backward(L, type=BF16, rows=4, inputs=8, hidden=6, act=14, x=P[0], w=P[1], s=P[2], d=P[3], r=None, gb=P[4], gw=P[5], gx=P[6], ws=P[7], n=BIG):
    return L.dkz_gated_backward(type, rows, inputs, hidden, act, x, w, s, d, r, 0.0, gb, gw, gx, ws, n)


@pytest.mark.parametrize("kw,want", [
    (dict(type=-1), INVALID), (dict(rows=-1), INVALID), (dict(act=5), INVALID), (dict(s=None), INVALID), (dict(d=None), INVALID),
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(gx=P[5]), INVALID), (dict(gw=P[1]), INVALID), (dict(gx=P[0]), INVALID),
    (dict(gb=P[2]), INVALID), (dict(gx=P[3]), INVALID), (dict(r=P[5]), INVALID), (dict(r=off(P[6], 2)), INVALID), (dict(ws=None), INVALID),
    (dict(n=16), INVALID), (dict(ws=off(P[7], 4)), INVALID), (dict(ws=P[2]), INVALID), (dict(rows=65536, inputs=65536), INVALID),
    (dict(gb=None, gw=None, gx=None, s=None, d=None, x=None, w=None), OK),
], ids=str)
def test_gated_backward_refusals(kw, want):
    assert backward(_lib.load_lm(), **kw) == want


def log_probs(L, type=BF16, rows=4, classes=100, pitch=104, z=P[0], t=1.0, given=2, tokens=P[1], top=3, lp=P[2], h=P[3], st=P[4], tt=P[5], tl=P[6],
              ws=P[7], n=BIG):
    return L.dkz_token_log_probs(type, rows, classes, pitch, z, t, given, tokens, top, lp, h, st, tt, tl, ws, n)


LOGITS = [
    (dict(type=2), INVALID), (dict(rows=-1), INVALID), (dict(classes=-1), INVALID), (dict(pitch=99), INVALID), (dict(t=0.0), INVALID),
    (dict(t=-1.0), INVALID), (dict(t=float("nan")), INVALID), (dict(t=float("inf")), INVALID), (dict(t=2.0**-65), INVALID), (dict(t=2.0**65), INVALID),
    (dict(z=None), INVALID), (dict(z=off(P[0], 1)), INVALID), (dict(rows=(1 << 26) + 1), INVALID), (dict(pitch=(1 << 26) + 1), INVALID),
    (dict(rows=1 << 20, pitch=(1 << 18) + 1), INVALID),
]


@pytest.mark.parametrize("kw,want", [
    *LOGITS, (dict(given=-1), INVALID), (dict(given=257), INVALID), (dict(top=-1), INVALID), (dict(top=65), INVALID), (dict(tokens=None), INVALID),
    (dict(lp=None), INVALID), (dict(st=None), INVALID), (dict(tt=None), INVALID), (dict(tl=None), INVALID), (dict(lp=P[0]), INVALID),
    (dict(h=P[1]), INVALID), (dict(st=off(P[0], 4 * 104 * 2 - 12)), INVALID), (dict(tl=P[5]), INVALID), (dict(h=off(P[4], 28)), INVALID),
    (dict(rows=0, z=None, tokens=None, lp=None, st=None, tt=None, tl=None), OK), (dict(lp=off(P[2], 4), tl=P[2], h=None), INVALID),
], ids=str)
def test_token_log_probs_refusals(kw, want):
    assert log_probs(_lib.load_lm(), **kw) == want


def test_token_log_probs_workspace_is_checked():
    L = _lib.load_lm()
    need = gpu.tokenLogProbsWorkspace(F32, 1, 65536, 20)
    assert need > 0
    shape = dict(type=F32, rows=1, classes=65536, pitch=65536, top=20)
    for kw in (dict(n=need - 1), dict(ws=None), dict(ws=off(P[7], 8)), dict(ws=P[0]), dict(ws=P[2])):
        assert log_probs(L, **{**shape, "n": need, **kw}) == INVALID


def log_probs_backward(L, type=BF16, rows=4, classes=100, pitch=104, z=P[0], t=1.0, given=2, tokens=P[1], st=P[2], h=P[3], a=P[4], e=P[5], beta=0.0,
                       d=P[6]):
    return L.dkz_token_log_probs_backward(type, rows, classes, pitch, z, t, given, tokens, st, h, a, e, beta, d)


@pytest.mark.parametrize("kw,want", [
    *LOGITS, (dict(given=-1), INVALID), (dict(given=257), INVALID), (dict(tokens=None), INVALID), (dict(st=None), INVALID), (dict(h=None), INVALID),
    (dict(a=None), INVALID), (dict(d=None), INVALID), (dict(d=P[0], beta=1.0), INVALID), (dict(d=off(P[0], 2)), INVALID), (dict(d=off(P[6], 1)), INVALID),
    (dict(d=P[1]), INVALID), (dict(d=P[2]), INVALID), (dict(d=P[5]), INVALID),
    (dict(rows=0, z=None, tokens=None, st=None, h=None, a=None, e=None, d=None), OK),
], ids=str)
def test_token_log_probs_backward_refusals(kw, want):
    assert log_probs_backward(_lib.load_lm(), **kw) == want


def distillation(L, type=BF16, rows=4, classes=100, pitch=104, z=P[0], t=1.0, top=5, tokens=P[1], logits=P[2], scales=P[3], loss=P[4], d=P[5], ws=P[6],
                 n=BIG):
    return L.dkz_distillation(type, rows, classes, pitch, z, t, top, tokens, logits, scales, 1.0, loss, d, ws, n)


@pytest.mark.parametrize("kw,want", [
    *LOGITS, (dict(top=0), INVALID), (dict(top=257), INVALID), (dict(tokens=None), INVALID), (dict(logits=None), INVALID), (dict(loss=None), INVALID),
    (dict(d=off(P[0], 2)), INVALID), (dict(d=off(P[5], 1)), INVALID), (dict(d=P[2]), INVALID), (dict(loss=P[0]), INVALID), (dict(loss=P[3]), INVALID),
    (dict(loss=off(P[5], 8)), INVALID), (dict(rows=0, z=None, tokens=None, logits=None, loss=None, d=None), OK),
], ids=str)
def test_distillation_refusals(kw, want):
    assert distillation(_lib.load_lm(), **kw) == want


def test_distillation_workspace_is_checked():
    L = _lib.load_lm()
    need = gpu.distillationWorkspace(BF16, 2, 65536)
    assert need > 0
    for kw in (dict(n=need - 1), dict(ws=None), dict(ws=off(P[6], 8)), dict(ws=P[0]), dict(ws=P[4])):
        assert distillation(L, **{"rows": 2, "classes": 65536, "pitch": 65536, "n": need, **kw}) == INVALID


@pytest.mark.parametrize("call", [
    lambda L, p: L.dkz_gated_forward_workspace(2, 1, 1, 1, p), lambda L, p: L.dkz_gated_forward_workspace(F32, -1, 1, 1, p),
    lambda L, p: L.dkz_gated_forward_workspace(F32, 1, 1, 1, None), lambda L, p: L.dkz_gated_backward_workspace(F32, 65536, 65536, 1, p),
    lambda L, p: L.dkz_token_log_probs_workspace(F32, 1, 1, 65, p), lambda L, p: L.dkz_token_log_probs_workspace(F32, 1, -1, 1, p),
    lambda L, p: L.dkz_distillation_workspace(2, 1, 1, p), lambda L, p: L.dkz_distillation_workspace(F32, 1, 1, None),
])
def test_workspace_queries_refuse(call):
    assert call(_lib.load_lm(), C.byref(C.c_size_t(0))) == INVALID


def test_a_python_call_raises_with_the_context():
    with pytest.raises(gpu.GpuError) as e:
        gpu.distillation(BF16, 4, 100, 100, gpu.Buf(), 0.0, 5, gpu.Buf(), gpu.Buf(), None, 1.0, gpu.Buf(), None, None)
    assert e.value.code == INVALID and "dkz_distillation" in e.value.context


# ---- the other hosts' bindings ----

ZIG = ROOT / "darknet_zig_amd" / "zig" / "dkz_lm.zig"
WRAPPERS = ["gatedForwardWorkspace", "gatedForward", "gatedBackwardWorkspace", "gatedBackward", "tokenLogProbsWorkspace", "tokenLogProbs",
            "tokenLogProbsBackward", "distillationWorkspace", "distillation"]


def test_zig_externs_follow_the_header():
    externs = re.findall(r"^pub extern fn (dkz_\w+)\((.*)\) (.+);$", ZIG.read_text(), flags=re.M)
    params = header_params()
    assert [e[0] for e in externs] == list(params) == symbols()
    for name, ps, ret in externs:
        got = [tuple(p.split(": ", 1)) for p in ps.split(", ")] if ps else []
        assert got == [(n, zig_type(t)) for t, n in params[name]], name
        assert ret == ("[*:0]const u8" if name.endswith("context") else "Status")


def test_zig_wrappers_pass_every_argument_in_order():
    text, params = ZIG.read_text(), header_params()
    for name in WRAPPERS:
        body = re.search(r"^pub fn " + name + r"\((.*?)\) [\w.]+ \{\n(.*?)^\}", text, flags=re.M | re.S).group(2)
        assert body.strip().startswith("if (!gpu.enabled) unreachable;")
        call = re.search(r"must\((dkz_\w+)\((.*)\), \"", body)
        args = re.sub(r"\bci\((\w+)\)", r"\1", call.group(2)).split(", ")
        assert len(args) == len(params[call.group(1)]), name
        for arg, (_, want) in zip(args, params[call.group(1)]):
            bare = re.sub(r"\.ptr$", "", arg)
            assert bare == want or (bare, want) in (("type_code", "type"), ("&need", "bytes"), ("bytes(workspace)", "workspace_bytes")), (name, arg, want)


@pytest.mark.parametrize("name", WRAPPERS)
def test_python_and_cpp_wrappers_take_the_same_arguments(name):
    cpp = (ROOT / "darknet_zig_amd" / "host" / "dkz_lm.hpp").read_text()
    m = re.search(r"inline [\w:]+ " + name + r"\((.*?)\) \{", cpp, flags=re.S)
    assert [p.split()[-1] for p in m.group(1).split(",")] == list(inspect.signature(getattr(gpu, name)).parameters)


def test_cpp_mirror_compiles_links_and_refuses(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    src = tmp_path / "lm.cpp"
    src.write_text('''#include <cstdio>
#include "dkz_dense.hpp"
#include "dkz_lm.hpp"
using namespace dkz::gpu;
int main() {
    if (gatedForwardWorkspace(DKZ_F32, 256, 4096, 4096) == 0 || gatedBackwardWorkspace(DKZ_BF16, 256, 4096, 4096) == 0) return 1;
    if (tokenLogProbsWorkspace(DKZ_F32, 1, 65536, 20) == 0 || distillationWorkspace(DKZ_F32, 1, 65536) == 0) return 2;
    gatedForward(DKZ_F32, 0, 8, 8, DKZ_SILU, Buf{}, Buf{}, Buf{}, Buf{}, Buf{}, Buf{});
    tokenLogProbs(DKZ_BF16, 0, 8, 8, Buf{}, 1.0f, 0, Buf{}, 0, Buf{}, Buf{}, Buf{}, Buf{}, Buf{}, Buf{});
    tokenLogProbsBackward(DKZ_BF16, 0, 8, 8, Buf{}, 1.0f, 0, Buf{}, Buf{}, Buf{}, Buf{}, Buf{}, 0.0f, Buf{});
    distillation(DKZ_BF16, 0, 8, 8, Buf{}, 1.0f, 1, Buf{}, Buf{}, Buf{}, 1.0f, Buf{}, Buf{}, Buf{});
    try {
        gatedBackward(DKZ_BF16, 4, 8, 6, 99, Buf{}, Buf{}, Buf{}, Buf{}, Buf{}, 0.0f, Buf{}, Buf{}, Buf{}, Buf{});
        return 3;
    } catch (const Error &e) {
        std::puts(e.what());
        return e.code() == 1 ? 0 : 4;
    }
}
''')
    lib, exe = LIB.parent, tmp_path / "lm"
    proc = subprocess.run([gxx, "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'include'}", f"-I{lib / 'host'}", str(src), "-o", str(exe),
                           f"-L{lib}", "-ldkz_lm", "-ldkz_dense", "-ldkz", f"-Wl,-rpath,{lib}", "-Wl,-rpath-link,/opt/rocm/lib"],
                          capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "dkz_gated_backward" in run.stdout, (run.returncode, run.stdout)
