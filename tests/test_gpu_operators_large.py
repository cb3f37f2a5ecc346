"""Sizes whose element offsets pass 32 bits, against 64-bit arithmetic at sampled
rows, and a batch of more tokens than 16-bit counts of one block per SM hold."""
import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def i4g():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import sm_120__gemm_b200 as m
    m.load()
    yield m
    torch.cuda.empty_cache()


def rand(*shape, seed=0, scale=1.0, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)


def sampled(M):
    at = torch.linspace(0, M - 1, 61, device="cuda").long()
    return torch.unique(torch.cat([at, torch.arange(M - 3, M, device="cuda")]))


def test_epilogue_product(i4g):
    M, N, K, g = 264_201, 8192, 64, 32
    w = rand(K, N, seed=1, scale=0.05)
    lin, w64 = i4g.QuantizedLinear.from_weight(w, g), ref.weight(w, g)
    a, residual = rand(M, K, seed=2), rand(M, N, seed=3)
    assert residual.numel() > 2 ** 31
    at = sampled(M)
    got = lin(a, activation="silu", residual=residual)
    ref.check(got[at], *ref.linear(a[at], w64, "silu", residual=residual[at]))
    kept = residual[at].clone()
    assert lin(a, activation="silu", residual=residual, out=residual) is residual
    assert torch.equal(residual, got)
    ref.check(residual[at], *ref.linear(a[at], w64, "silu", residual=kept))
    assert i4g.device_status() == 0


def test_experts_and_combination(i4g):
    T, E, k, K, N, g = 132_101, 3, 2, 64, 8192, 32
    w = rand(E, K, N, seed=1, scale=0.05)
    ex = i4g.QuantizedExperts.from_weight(w, g)
    x = rand(T, K, seed=2)
    r = i4g.route(rand(T, E, seed=3, dtype=torch.float32), k)
    y = ex(x, r, activation="relu")
    assert y.numel() > 2 ** 31
    at = sampled(T * k)
    expert = torch.bucketize(at, r.offsets[1:].long(), right=True)
    for e in range(E):
        p = at[expert == e]
        ref.check(y[p], *ref.linear(x[(r.rows[p] // k).long()], ref.weight(w[e], g), "relu"))
    token = sampled(T)
    out = i4g.combine(y, r)
    part = r.weights[token].double()[..., None] * y[r.slots[token].long()].double()
    want = part.sum(1)
    tol = 3 * 2.0 ** -24 * part.abs().sum(1)  # two additions and a product, FP32
    ref.check(out[token], want, tol + 2.0 ** -11 * (want.abs() + tol) + 2.0 ** -25)
    assert i4g.device_status() == 0


@pytest.mark.parametrize("T,E,k,dtype", [(5_000_011, 4, 2, torch.float32),
                                         (4_300_007, 512, 1, torch.float16)])
def test_route(i4g, T, E, k, dtype):
    x = rand(T, E, seed=1, dtype=dtype)
    r = i4g.route(x, k)
    flat = r.ids.reshape(-1).long()
    assert int(flat.min()) >= 0 and int(flat.max()) < E
    assert torch.equal(r.offsets[1:].long(), torch.bincount(flat, minlength=E).cumsum(0))
    rows = torch.argsort(flat, stable=True)
    assert torch.equal(r.rows.long(), rows)
    assert torch.equal(r.slots.reshape(-1).long()[rows], torch.arange(T * k, device="cuda"))
    for t in (0, T // 2, T - 4000):  # the choice itself, where it can be sorted at once
        part = x[t:t + 4000].double()
        best, ids = torch.sort(part, dim=1, descending=True, stable=True)
        assert torch.equal(r.ids[t:t + 4000].long(), ids[:, :k])
        w = torch.softmax(part, 1).gather(1, ids[:, :k])
        w = w / w.sum(1, keepdim=True)
        assert ((r.weights[t:t + 4000].double() - w).abs() <= 64 * 2.0 ** -23 * w).all()
