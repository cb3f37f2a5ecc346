"""Weights made on an explicit stream while the current one is busy: every step
of their making runs on the stream that was given, and what it allocates is that
stream's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def i4g():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import sm_120__gemm_b200 as m
    m.load()
    return m


def rand(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * 0.05).half()


def while_busy(make, temporary):
    """make(stream) with 50 ms of work ahead on the current stream, the memory a
    temporary of that shape would get holding something else."""
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    for stream in (s, s.cuda_stream):
        junk = torch.full(temporary, 3.0, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        del junk
        torch.cuda._sleep(100_000_000)
        made = make(stream)
        # what the current stream frees and takes next must not be in use on s
        torch.full(temporary, -3.0, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        yield made


def same(a, b):
    return torch.equal(a.tiles, b.tiles) and torch.equal(a.scales, b.scales)


def test_linear_from_gate_up(i4g):
    gate, up = rand(1024, 2048, seed=1), rand(1024, 2048, seed=2)
    want = i4g.QuantizedLinear.from_gate_up(gate, up, 64)
    for got in while_busy(lambda s: i4g.QuantizedLinear.from_gate_up(gate, up, 64, stream=s),
                          (1024, 4096)):
        assert same(got, want)


def test_experts_from_gate_up(i4g):
    gate, up = rand(3, 1024, 1024, seed=1), rand(3, 1024, 1024, seed=2)
    want = i4g.QuantizedExperts.from_gate_up(gate, up, 64)
    for got in while_busy(lambda s: i4g.QuantizedExperts.from_gate_up(gate, up, 64, stream=s),
                          (3, 1024, 2048)):
        assert same(got, want)


def test_from_weight_with_strides(i4g):
    w = rand(2048, 1024, seed=3).t()  # made contiguous inside the call
    want = i4g.QuantizedLinear.from_weight(w, 128)
    for got in while_busy(lambda s: i4g.QuantizedLinear.from_weight(w, 128, stream=s),
                          (1024, 2048)):
        assert same(got, want)
    e = rand(2, 1024, 512, seed=4).transpose(1, 2)
    want = i4g.QuantizedExperts.from_weight(e, 32)
    for got in while_busy(lambda s: i4g.QuantizedExperts.from_weight(e, 32, stream=s),
                          (1, 512, 1024)):
        assert same(got, want)


def test_from_packed(i4g):
    K, N, g = 512, 1024, 64
    packed = torch.randint(0, 256, (K * N // 2,), dtype=torch.uint8, device="cuda")
    scales = rand(K // g, N, seed=5).abs()
    want = i4g.QuantizedLinear.from_packed(packed, scales, K, N, g)
    for got in while_busy(lambda s: i4g.QuantizedLinear.from_packed(packed, scales, K, N, g,
                                                                    stream=s), (K, N // 4)):
        assert same(got, want)


@pytest.mark.parametrize("kind", ["plain", "fp32", "epilogue", "experts"])
def test_weights_dropped_after_their_last_call(i4g, kind):
    """A layer and its inputs may go right after a call on another stream: their
    memory is not reused under the kernel."""
    K, N, M = 1024, 2048, 24
    a = rand(M, K, seed=1)
    s = torch.cuda.Stream()

    def layer():
        if kind == "experts":
            return i4g.QuantizedExperts.from_weight(rand(2, K, N, seed=2), 64)
        return i4g.QuantizedLinear.from_weight(rand(K, N, seed=2), 64)

    def call(m, x, **kw):
        if kind == "experts":
            r = i4g.route(torch.zeros(M, 2, device="cuda"), 1, **kw)
            return m(x, r, activation="silu", **kw)
        return m(x, fp32_out=(kind == "fp32"), activation="silu" if kind == "epilogue" else "none",
                 **kw)

    want = call(layer(), a)
    torch.cuda.synchronize()
    for stream in (s, s.cuda_stream):
        m, x = layer(), a.clone()
        sizes = [(t.numel(), t.dtype) for t in (m.tiles, m.scales, x)]
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(50_000_000)
        got = call(m, x, stream=stream)
        del m, x
        taken = [torch.zeros(n, dtype=t, device="cuda") for n, t in sizes]
        s.synchronize()
        assert torch.equal(got, want)
        del taken


def test_strided_rows_on_a_stream(i4g):
    """Rows that the call makes contiguous are copied on the stream that was given."""
    lin = i4g.QuantizedLinear.from_weight(rand(256, 512, seed=2), 64)
    x = rand(256, 40, seed=3)
    want = lin(x.t())
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.full((40, 256), 3.0, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)
    got = lin(x.t(), stream=s)
    s.synchronize()
    assert torch.equal(got, want)


def test_workspace_is_zeroed_on_its_stream(i4g):
    M, N, K = 600, 512, 8192
    need = i4g.gemm_workspace_size(M, N, K)
    assert need > 4096
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        i4g._workspaces.pop((torch.cuda.current_device(), s.cuda_stream), None)
        torch.cuda.empty_cache()
        junk = torch.full((need,), 3, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        del junk
        torch.cuda._sleep(50_000_000)
        ws = i4g.workspace_for(M, N, K, stream=stream)
        with torch.cuda.stream(s):
            seen = ws[:4096].clone()
        s.synchronize()
        assert not seen.any()
        torch.cuda.synchronize()
    i4g._workspaces.pop((None, s.cuda_stream), None)
    assert i4g.workspace_for(M, N, K, device="cuda", stream=s).device == ws.device


def test_refuses_scales_elsewhere(i4g):
    """Codes and scales live on one device: the call says so before it launches."""
    lin = i4g.QuantizedLinear.from_weight(rand(64, 128), 64)
    ex = i4g.QuantizedExperts.from_weight(rand(2, 64, 128), 64)
    a = rand(4, 64)
    r = i4g.route(torch.zeros(4, 2, device="cuda"), 1)
    apart = i4g.QuantizedLinear(lin.tiles, lin.scales.cpu(), 64, 128, 64)
    with pytest.raises(TypeError):
        apart(a, activation="silu")
    with pytest.raises(TypeError):
        i4g.QuantizedExperts(ex.tiles, ex.scales.cpu(), 2, 64, 128, 64)(a, r)


def test_refuses_weights_on_the_cpu(i4g):
    cpu = torch.zeros(64, 128, dtype=torch.float16)
    for call in (lambda: i4g.QuantizedLinear.from_weight(cpu, 64),
                 lambda: i4g.QuantizedLinear.from_gate_up(cpu, cpu, 64),
                 lambda: i4g.QuantizedExperts.from_gate_up(cpu[None], cpu[None], 64)):
        with pytest.raises(TypeError):
            call()
