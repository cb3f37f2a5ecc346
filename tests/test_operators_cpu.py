"""Refusals of the epilogue, routing and experts entry points, before any
device is touched, and the plain parts of their Python side. No GPU."""
import ctypes

import numpy as np
import pytest
import torch

vp = ctypes.c_void_p
FAKE = vp(0x1000)  # never dereferenced: checks fail first
NULL, SHAPE, GROUP, ALIGN, VARIANT = -1, -2, -3, -4, -9


@pytest.fixture(scope="module")
def m():
    import sm_120__gemm_b200 as mod
    mod.load()
    return mod


@pytest.fixture(scope="module")
def lib(m):
    return m.load()


def epi(m, **kw):
    e = m.Epilogue()
    for k, v in kw.items():
        setattr(e, k, v)
    return ctypes.byref(e)


def gemm(lib, e, a=FAKE, tiles=FAKE, scales=FAKE, c=FAKE, M=4, N=128, K=128, g=64, ws=None):
    return lib.i4g_gemm_epilogue(a, tiles, scales, c, M, N, K, g, e, ws, 0, None)


def test_epilogue_refusals(m, lib):
    ok = epi(m)
    assert gemm(lib, ok, M=-1) == SHAPE
    assert gemm(lib, ok, N=100) == SHAPE
    assert gemm(lib, ok, K=96, g=32) == SHAPE
    assert gemm(lib, ok, g=96) == GROUP
    assert gemm(lib, ok, K=192, g=128) == GROUP
    for k in ("a", "tiles", "scales", "c"):
        assert gemm(lib, ok, **{k: None}) == NULL
    assert gemm(lib, ok, M=0, a=None, c=None) == 0  # an empty batch is no work
    assert gemm(lib, epi(m, activation=5)) == VARIANT
    assert gemm(lib, epi(m, activation=-1)) == VARIANT
    assert gemm(lib, epi(m, gated=2)) == VARIANT
    assert gemm(lib, epi(m, fp32_out=-1)) == VARIANT
    assert gemm(lib, epi(m, residual=0x1000, ld_residual=127)) == SHAPE
    assert gemm(lib, epi(m, residual=0x1000, ld_residual=63, gated=1)) == SHAPE
    assert gemm(lib, epi(m, residual=0x1001, ld_residual=128)) == ALIGN
    assert gemm(lib, epi(m, bias=0x1001)) == ALIGN
    assert gemm(lib, ok, a=vp(0x1008)) == ALIGN
    assert gemm(lib, ok, c=vp(0x1001)) == ALIGN
    assert gemm(lib, epi(m, fp32_out=1), c=vp(0x1002)) == ALIGN
    assert gemm(lib, ok, ws=vp(0x1010)) == ALIGN
    n = ctypes.c_size_t()
    assert lib.i4g_gemm_epilogue_workspace_size(4, 128, 128, None) == NULL
    assert lib.i4g_gemm_epilogue_workspace_size(4, 100, 128, ctypes.byref(n)) == SHAPE
    assert lib.i4g_gemm_epilogue_workspace_size(0, 128, 128, ctypes.byref(n)) == 0
    assert n.value == 0


def experts(lib, e=None, a=FAKE, a_rows=8, offsets=FAKE, rows=FAKE, div=2, pairs=16, E=4, N=128,
            K=128, g=64, c=FAKE, ws=None):
    return lib.i4g_experts_gemm(a, a_rows, FAKE, FAKE, c, offsets, rows, div, pairs, E, N, K, g, e,
                                ws, 0, None)


def test_experts_refusals(m, lib):
    assert experts(lib, E=0) == SHAPE
    assert experts(lib, E=513) == SHAPE
    assert experts(lib, pairs=-1) == SHAPE
    assert experts(lib, N=64) == SHAPE
    assert experts(lib, K=32, g=32) == SHAPE
    assert experts(lib, g=48) == GROUP
    assert experts(lib, offsets=None) == NULL
    assert experts(lib, a=None) == NULL
    assert experts(lib, c=None) == NULL
    assert experts(lib, div=0) == SHAPE
    assert experts(lib, a_rows=0) == SHAPE
    assert experts(lib, rows=None, a_rows=15) == SHAPE  # sorted rows: one per pair
    assert experts(lib, offsets=vp(0x1002)) == ALIGN
    assert experts(lib, rows=vp(0x1001)) == ALIGN
    assert experts(lib, epi(m, residual=0x1000, ld_residual=128)) == VARIANT
    assert experts(lib, epi(m, activation=9)) == VARIANT
    assert experts(lib, ws=vp(0x1020)) == ALIGN
    assert experts(lib, pairs=1 << 30, N=1 << 20) == SHAPE
    assert experts(lib, pairs=0, a=None, c=None, offsets=None) == 0


def test_experts_parts_refusals(m, lib):
    def call(kept=None, scratch=None, E=4):
        return lib.i4g_experts_gemm_parts(FAKE, 8, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 16, E, 128, 128,
                                          64, None, kept, 0, scratch, 0, None)
    assert call(E=0) == SHAPE
    assert call(kept=vp(0x1080)) == ALIGN
    assert call(scratch=vp(0x1010)) == ALIGN
    kept, scratch = ctypes.c_size_t(), ctypes.c_size_t()
    parts = lib.i4g_experts_workspace_parts
    assert parts(16, 4, 128, 128, None, ctypes.byref(scratch)) == NULL
    assert parts(16, 4, 128, 128, ctypes.byref(kept), None) == NULL
    assert parts(16, 0, 128, 128, ctypes.byref(kept), ctypes.byref(scratch)) == SHAPE
    assert parts(0, 4, 128, 128, ctypes.byref(kept), ctypes.byref(scratch)) == 0
    assert kept.value == scratch.value == 0


def route(m, lib, T=4, E=16, k=2, logits=FAKE, ld=16, out=FAKE, bias=None, offsets=FAKE, **opt):
    o = m.RouteOptions(0, 1, 1, 0, 1, 1.0)
    for name, v in opt.items():
        setattr(o, name, v)
    return lib.i4g_route(logits, 1, ld, bias, T, E, k, ctypes.byref(o), out, out, offsets, out,
                         out, None, 0, None)


def test_route_refusals(m, lib):
    assert route(m, lib, T=-1) == SHAPE
    assert route(m, lib, E=0, ld=0) == SHAPE
    assert route(m, lib, E=513, ld=513) == SHAPE
    assert route(m, lib, k=0) == SHAPE
    assert route(m, lib, k=17) == SHAPE
    assert route(m, lib, E=64, ld=64, k=33) == SHAPE
    assert route(m, lib, T=1 << 30, k=2) == SHAPE
    assert route(m, lib, ld=15) == SHAPE
    assert route(m, lib, logits=None) == NULL
    assert route(m, lib, out=None) == NULL
    assert route(m, lib, offsets=None, T=0) == NULL
    assert route(m, lib, scoring=2) == VARIANT
    assert route(m, lib, group_score=-1) == VARIANT
    assert route(m, lib, n_group=0) == SHAPE
    assert route(m, lib, n_group=3) == SHAPE       # 16 experts in 3 groups
    assert route(m, lib, E=33 * 2, ld=66, n_group=33) == SHAPE
    assert route(m, lib, n_group=4, topk_group=5) == SHAPE
    assert route(m, lib, n_group=8, topk_group=1, k=3) == SHAPE  # groups of two
    assert route(m, lib, logits=vp(0x1002)) == ALIGN
    assert route(m, lib, bias=vp(0x1002)) == ALIGN
    assert lib.i4g_route(FAKE, 1, 16, None, 4, 16, 2, None, FAKE, FAKE, FAKE, FAKE, FAKE, None, 0,
                         None) == NULL


def test_combine_refusals(lib):
    def call(y=FAKE, rows=8, slots=FAKE, w=FAKE, res=None, out=FAKE, T=4, k=2, N=64):
        return lib.i4g_experts_combine(y, rows, slots, w, res, out, T, k, N, None)
    assert call(T=-1) == SHAPE
    assert call(N=12) == SHAPE
    assert call(N=0) == SHAPE
    assert call(k=0) == SHAPE
    assert call(rows=-1) == SHAPE
    assert call(y=None) == NULL
    assert call(slots=None) == NULL
    assert call(w=None) == NULL
    assert call(out=None) == NULL
    assert call(y=vp(0x1008)) == ALIGN
    assert call(res=vp(0x1002)) == ALIGN
    assert call(out=vp(0x1004)) == ALIGN
    assert call(T=0, y=None, slots=None, w=None, out=None) == 0


def test_python_refuses_cpu_tensors_and_unknown_names(m):
    lin = m.QuantizedLinear(torch.zeros(64 * 64, dtype=torch.uint8),
                            torch.zeros(128, dtype=torch.float16), 64, 128, 64)
    a = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(TypeError):
        lin(a, activation="silu")
    with pytest.raises(ValueError):
        lin(a, activation="swish")
    with pytest.raises(TypeError):
        m.route(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError):
        m.route(torch.zeros(2, 8), 2, scoring="tanh")
    with pytest.raises(TypeError):
        m.combine(a, None)
    with pytest.raises(ValueError):
        m.QuantizedExperts(torch.zeros(10, dtype=torch.uint8),
                           torch.zeros(4, dtype=torch.float16), 2, 64, 128, 64)
    with pytest.raises(TypeError):
        m.QuantizedExperts(torch.zeros(10), torch.zeros(4), 2, 64, 128, 64)


def test_interleave_gate_up(m):
    from sm_120__gemm_b200.linear import interleave_gate_up
    gate = torch.arange(32).view(2, 16)
    up = gate + 100
    both = interleave_gate_up(gate, up)
    assert both.shape == (2, 32)
    for j in range(16):
        at = 16 * (j // 8) + j % 8
        assert torch.equal(both[:, at], gate[:, j]) and torch.equal(both[:, at + 8], up[:, j])
    with pytest.raises(ValueError):
        interleave_gate_up(gate[:, :12], up[:, :12])
    with pytest.raises(ValueError):
        interleave_gate_up(gate, up[:1])


def test_cpp_wrappers_throw(tmp_path):
    """The C++ forms compile and turn a refusal into std::runtime_error."""
    import os
    import shutil
    import subprocess

    from conftest import ROOT
    if shutil.which("g++") is None:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include "int4gemm.hpp"
#include <cstdio>
template <typename F> int throws(F f) {
  try { f(); } catch (const std::runtime_error& e) { std::printf("%s\n", e.what()); return 1; }
  return 0;
}
int main() {
  using namespace int4gemm;
  i4g_epilogue_t e{};
  i4g_route_t r{I4G_SCORE_SOFTMAX, 1, 1, I4G_GROUP_MAX, 1, 1.0f};
  return 4 - throws([&] { launch_final_epilogue(0, 0, 0, 0, 4, 100, 128, 64, e, 0, 0, 0); }) -
         throws([&] { launch_route(0, true, 8, 0, 4, 8, 9, r, 0, 0, 0, 0, 0, 0, 0, 0); }) -
         throws([&] { launch_experts(0, 4, 0, 0, 0, 0, 0, 0, 8, 2, 128, 128, 48, e, 0, 0, 0); }) -
         throws([&] { launch_combine(0, 8, 0, 0, 0, 0, 4, 2, 12, 0); });
}
''')
    pkg = os.path.join(ROOT, "sm_120__gemm_b200")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I",
                    "/usr/local/cuda/include", str(src), "-o", str(tmp_path / "t"), "-L", pkg,
                    "-li4g", f"-Wl,-rpath,{pkg}"], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True)
    assert out.returncode == 0, out


def test_plain_routing_of_a_worked_example():
    """The comparison itself, on numbers worked by hand."""
    import operators_ref as ref
    x = torch.tensor([[0.0, 2.0, 2.0, 1.0], [-np.inf] * 4, [np.nan, 1.0, -np.inf, 3.0]])
    ids, w, off, rows, slots = ref.route(x, 2)
    assert ids.tolist() == [[1, 2], [-1, -1], [3, 1]]
    assert np.allclose(w[0], [0.5, 0.5]) and not w[1].any()
    assert np.allclose(w[2], [1 / (1 + np.exp(-2)), 1 / (1 + np.exp(2))])
    assert off.tolist() == [0, 0, 2, 3, 4]
    assert rows.tolist() == [0, 5, 1, 4, -1, -1]
    assert slots.tolist() == [[0, 2], [-1, -1], [3, 1]]
    # groups: {0, 1} has the best single logit, {2, 3} the best sum
    x = torch.tensor([[5.0, -9.0, 4.0, 4.0]])
    assert ref.route(x, 1, n_group=2)[0].tolist() == [[0]]
    assert ref.route(x, 1, n_group=2, group_score="top2", scoring="sigmoid")[0].tolist() == [[2]]


def test_routings_agree():
    """The plain routing and the definition that the timed cases use pick the same."""
    import importlib.util
    import os

    import operators_ref as ref
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("ops", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    g = torch.Generator().manual_seed(3)
    for scoring in ("softmax", "sigmoid"):
        for bias in (None, 0.1 * torch.randn(24, generator=g)):
            for gs in ("max", "top2"):
                x = torch.randn(40, 24, generator=g)
                x[7] = -np.inf
                case = dict(T=40, E=24, k=3, groups=4, keep=2, scoring=scoring, group_score=gs,
                            renormalize=True, scale=2.0)
                a = ops._plain_route({"logits": x, "bias": bias}, case)
                b = ops._exact_route({"logits": x, "bias": bias}, case)
                c = ref.route(x, 3, scoring, bias, 4, 2, gs, True, 2.0)
                for i, (p, q, r) in enumerate(zip(a, b, (c[0], c[1], c[2], c[3], c[4]))):
                    assert np.allclose(p.numpy(), q, rtol=1e-6), i
                    assert np.allclose(q, r, rtol=1e-12), i
