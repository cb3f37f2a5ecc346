"""Every instance of the epilogue kernel against 64-bit arithmetic: five tile
heights x three scale groups x plain, gated and FP32 results, with whole tiles
and with tails cut along K, dense and over experts. The height that the device
runs is asserted, so a new rule for it shows here instead of moving the coverage."""
import functools

import numpy as np
import pytest
import torch

import operators_ref as ref
import tile_cases

pytestmark = pytest.mark.gpu

# activation, gated, FP32 results
KINDS = [("none", False, False), ("silu", True, False), ("gelu", False, True),
         ("gelu_tanh", True, True)]


@pytest.fixture(scope="module")
def i4g():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import sm_120__gemm_b200 as m
    m.load()
    yield m
    weights.cache_clear()


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def rand(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).half()


@functools.lru_cache(maxsize=1)
def weights(E, K, N, group):
    import sm_120__gemm_b200 as m
    w = rand(max(E, 1), K, N, seed=1, scale=0.05)
    made = m.QuantizedExperts.from_weight(w, group) if E else \
        m.QuantizedLinear.from_weight(w[0], group)
    return made, [ref.weight(x, group) for x in w]


@pytest.mark.parametrize("height,cut,M,N,K,group", tile_cases.by_group(tile_cases.DENSE))
def test_dense(i4g, height, cut, M, N, K, group):
    tile_cases.check_dense(i4g.epilogue_plan(M, N, K, sms()), (height, cut))
    lin, (w64,) = weights(0, K, N, group)
    a, bias = rand(M, K, seed=2), rand(N, seed=3)
    for act, gated, fp32 in KINDS:
        residual = rand(M, N // 2 if gated else N, seed=4)
        got = lin(a, fp32_out=fp32, bias=bias, activation=act, gated=gated, residual=residual)
        ref.check(got, *ref.linear(a, w64, act, gated, bias, residual, fp32))
        again = lin(a, fp32_out=fp32, bias=bias, activation=act, gated=gated, residual=residual)
        assert torch.equal(got, again)
    assert i4g.device_status() == 0


@pytest.mark.parametrize("height,cut,copied,T,E,k,K,N,group",
                         tile_cases.by_group(tile_cases.EXPERTS))
def test_experts(i4g, height, cut, copied, T, E, k, K, N, group):
    counts = tile_cases.expert_rows(T, E, k)
    tile_cases.check_experts(i4g.epilogue_plan(T * k, N, K, sms(), expert_rows=counts),
                             (height, cut, copied))
    ex, w64 = weights(E, K, N, group)
    ids = tile_cases.ids(T, E, k)
    offsets, rows, slots = ref.order(ids, E)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).int().cuda()  # noqa: E731
    r = i4g.Routing(t(ids), torch.ones(T, k, device="cuda"), t(offsets), t(rows), t(slots))
    a, bias = rand(T, K, seed=2), rand(E, N, seed=3)
    sorted_rows = a[(r.rows // k).long()]
    for act, gated, fp32 in KINDS:
        kw = dict(bias=bias, activation=act, gated=gated, fp32_out=fp32)
        got = ex(a, r, **kw)
        # without a workspace: whole tiles, rows gathered inside the product
        bare = torch.empty_like(got)
        i4g.launch_experts(a, T, ex.tiles, ex.scales, bare, r.offsets, r.rows, k, T * k, E, N, K,
                           group, **kw)
        in_order = ex(sorted_rows, r, gather=False, **kw)
        assert torch.equal(got, in_order)
        for e in range(E):
            lo, hi = int(offsets[e]), int(offsets[e + 1])
            want = ref.linear(sorted_rows[lo:hi], w64[e], act, gated, bias[e], None, fp32)
            ref.check(got[lo:hi], *want)
            ref.check(bare[lo:hi], *want)
    assert i4g.device_status() == 0
