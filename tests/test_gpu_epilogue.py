"""The GEMM's fused epilogue against 64-bit arithmetic (operators_ref.py)."""
import ctypes

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
    return m


def rand(*shape, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).half()


def make(i4g, K, N, group, seed=1):
    w = rand(K, N, seed=seed, scale=0.05)
    return i4g.QuantizedLinear.from_weight(w, group), ref.weight(w, group)


def run(i4g, M, N, K, group, act="none", gated=False, bias=False, residual=False, fp32=False):
    lin, w64 = make(i4g, K, N, group)
    cols = N // 2 if gated else N
    a = rand(M, K, seed=2)
    b = rand(N, seed=3) if bias else None
    r = rand(M, cols, seed=4) if residual else None
    got = lin(a, fp32_out=fp32, bias=b, activation=act, gated=gated, residual=r)
    torch.cuda.synchronize()
    assert i4g.device_status() == 0
    assert got.dtype == (torch.float32 if fp32 else torch.float16) and got.shape == (M, cols)
    ref.check(got, *ref.linear(a, w64, act, gated, b, r, fp32))


# row counts around every tile height; at this size they run the decode kernel
# and 16-row tiles (test_gpu_tile_heights.py asserts the height it runs)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 128, 129, 255, 257, 700])
@pytest.mark.parametrize("gated", [False, True])
def test_rows(i4g, M, gated):
    run(i4g, M, 384, 320, 64, "silu", gated, bias=True)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gated,residual", [(False, True), (True, True), (False, False)])
@pytest.mark.parametrize("M", [5, 200])
def test_activations(i4g, act, gated, residual, M):
    run(i4g, M, 256, 256, 128, act, gated, bias=True, residual=residual)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("fp32", [False, True])
def test_groups_and_types(i4g, group, M, fp32):
    run(i4g, M, 256, 384, group, "gelu", gated=(group == 64), bias=True, residual=True, fp32=fp32)


# every tile height in turn, by threes and fours: 32, 64, 128 and 256 rows (the
# height follows from how many tiles the SMs get, so small shapes take 16)
@pytest.mark.parametrize("M,N,K", [(17, 18944, 1088), (25, 20480, 2048), (90, 2432, 12416),
                                   (33, 18944, 1088), (63, 14336, 2112), (160, 4096, 4160),
                                   (65, 9600, 2112), (127, 18944, 1088), (513, 9472, 1088),
                                   (1000, 1920, 4160), (129, 18944, 576), (203, 18944, 320),
                                   (255, 18944, 576), (203, 9600, 8256)])
@pytest.mark.parametrize("gated,fp32", [(False, False), (True, False), (False, True)])
def test_tile_heights(i4g, M, N, K, gated, fp32):
    run(i4g, M, N, K, 64, "gelu" if gated else "none", gated, bias=True, residual=True, fp32=fp32)


# few tiles and long K, more tiles than SMs, promotion; up to 16 rows both kernels
# that serve them. Tails are cut along K at 16, 32 and 64 rows here, the last two run
# whole 128-row tiles (test_gpu_tile_heights.py cuts at every height)
@pytest.mark.parametrize("M,N,K", [(1, 128, 14336), (7, 256, 8192), (1, 28672, 2048),
                                   (3, 28672, 8192), (13, 20480, 4160), (16, 57344, 1024),
                                   (40, 4096, 8192), (64, 128, 6144 + 64), (100, 640, 8192),
                                   (300, 640, 8192), (520, 7168, 4160), (1024, 2048, 12288)])
@pytest.mark.parametrize("gated", [False, True])
def test_split_tails(i4g, M, N, K, gated):
    run(i4g, M, N, K, 64, "silu" if gated else "none", gated, bias=True, residual=True)


@pytest.mark.parametrize("M,N,K", [(1, 28672, 2048), (3, 28672, 8192), (40, 4096, 8192),
                                   (100, 640, 8192), (300, 640, 8192), (1024, 3200, 12288), (520, 7168, 4160)])
def test_split_tails_repeat_bit_for_bit(i4g, M, N, K):
    lin, _ = make(i4g, K, N, 64)
    a = rand(M, K, seed=9)
    first = lin(a, activation="silu", gated=True)
    for _ in range(40):
        assert torch.equal(first, lin(a, activation="silu", gated=True))
    assert i4g.device_status() == 0


def test_a_row_does_not_depend_on_the_other_rows_values(i4g):
    """Rows are independent: NaN and infinity in one row stay there."""
    lin, w64 = make(i4g, 256, 256, 64)
    a = rand(40, 256, seed=5)
    a[3] = float("nan")
    a[11, 7] = float("inf")
    got = lin(a, activation="relu")
    assert got[3].isnan().all() and not got[11].isfinite().all()
    keep = [i for i in range(40) if i not in (3, 11)]
    ref.check(got[keep], *ref.linear(a[keep], w64, "relu"))


def test_large_values_saturate_like_fp16(i4g):
    lin, w64 = make(i4g, 256, 128, 64)
    a = rand(4, 256, seed=6, scale=6e4).clamp(-6e4, 6e4)
    got = lin(a, activation="silu").double()
    x = a.double() @ w64
    y = ref.activation(x, "silu")
    big = y.abs() > 70000
    assert big.any() and torch.isinf(got[big]).all()
    assert (got[x < -1000] == 0).all()


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [3, 40, 300])
def test_infinity_stays_infinity(i4g, act, gated, M):
    """act(+infinity) is +infinity for every activation: from a bias, and from a
    sum of an infinite activation row; gated, it takes the sign of the up column."""
    lin, w64 = make(i4g, 128, 256, 64)
    a = rand(M, 128, seed=2)
    bias = rand(256, seed=3)
    bias[[2, 21, 199]] = float("inf")  # gate columns, were they gated
    want, tol = ref.linear(a, w64, act, gated, bias)
    got = lin(a, activation=act, gated=gated, bias=bias)
    lost = torch.isinf(want)
    assert int(lost.sum()) == 3 * M and torch.equal(got[lost].double(), want[lost])
    ref.check(got[~lost], want[~lost], tol[~lost])
    a = torch.zeros_like(a)
    a[1, 7] = float("inf")
    got = lin(a, activation=act)
    assert torch.isposinf(got[1, w64[7] > 0]).all()


def test_residual_in_place_strided_and_out(i4g):
    lin, w64 = make(i4g, 512, 256, 128)
    a = rand(33, 512, seed=7)
    stream = rand(33, 256, seed=8)
    want, tol = ref.linear(a, w64, residual=stream)
    out = stream.clone()
    assert lin(a, out=out, residual=out) is out
    ref.check(out, want, tol)
    wide = rand(33, 300, seed=10)
    view = wide[:, 5:261]  # odd offset, stride 300
    want, tol = ref.linear(a, w64, residual=view)
    ref.check(lin(a, residual=view), want, tol)
    turned = rand(256, 33, seed=11).t()  # columns not contiguous
    ref.check(lin(a, residual=turned), *ref.linear(a, w64, residual=turned))
    row = rand(256, seed=12).expand(33, 256)  # one row for all
    ref.check(lin(a, residual=row), *ref.linear(a, w64, residual=row))
    strided = rand(66, 512, seed=13)[::2]
    ref.check(lin(strided, activation="relu"), *ref.linear(strided, w64, "relu"))


def test_plain_calls_keep_their_path(i4g):
    """Without epilogue arguments the call is what it was, bit for bit."""
    lin, _ = make(i4g, 512, 256, 128)
    for M in (1, 16, 200):
        a = rand(M, 512, seed=M)
        c = torch.empty(M, 256, dtype=torch.float16, device="cuda")
        i4g.launch_final(a, lin.tiles, lin.scales, c, M, 256, 512, 128)
        assert torch.equal(c, lin(a, activation="none"))


def test_empty_batch_and_refusals(i4g):
    lin, _ = make(i4g, 256, 256, 64)
    a = rand(4, 256)
    assert lin(a[:0], activation="silu", gated=True).shape == (0, 128)
    f16 = dict(dtype=torch.float16, device="cuda")
    for bad in (dict(bias=torch.zeros(128, **f16)), dict(bias=torch.zeros(256, device="cuda")),
                dict(residual=torch.zeros(4, 128, **f16)), dict(bias=torch.zeros(256).half()),
                dict(activation="relu", out=torch.zeros(4, 128, **f16)),
                dict(activation="relu", out=torch.zeros(4, 512, **f16)[:, ::2]),
                dict(activation="swish")):
        with pytest.raises((ValueError, TypeError)):
            lin(a, **bad)
    with pytest.raises(ValueError):
        lin(rand(4, 128), activation="relu")
    with pytest.raises(TypeError):
        lin(rand(4, 256).float(), activation="relu")


def test_workspace_none_small_and_enough_agree(i4g):
    M, N, K = 24, 512, 8192
    assert i4g.gemm_epilogue_workspace_size(4, N, K) == 0  # the decode kernel
    lin, w64 = make(i4g, K, N, 64)
    a = rand(M, K, seed=3)
    need = i4g.gemm_epilogue_workspace_size(M, N, K)
    assert need > 4096
    want, tol = ref.linear(a, w64, "gelu")
    for n in (0, need - 1, need):
        ws = torch.zeros(n, dtype=torch.uint8, device="cuda") if n else None
        c = torch.empty(M, N, dtype=torch.float16, device="cuda")
        for _ in range(2):
            i4g.launch_final_epilogue(a, lin.tiles, lin.scales, c, M, N, K, 64, activation="gelu",
                                      workspace=ws)
        ref.check(c, want, tol)
        if n:
            assert int(ws[:4096].count_nonzero()) == 0, "arrival counters not reset"


def test_counters_left_by_a_timeout_are_reset(i4g):
    """What a launch that gave up leaves in the workspaces the package holds does
    not reach later calls: the status call that reports it resets them."""
    import sm_120__gemm_b200._binding as binding
    lin, _ = make(i4g, 8192, 512, 64)
    a, b = rand(24, 8192, seed=1), rand(600, 8192, seed=2)
    assert i4g.gemm_epilogue_workspace_size(24, 512, 8192) > 0
    assert i4g.gemm_workspace_size(600, 512, 8192) > 0
    want, plain = lin(a, activation="silu"), lin(b)
    s = torch.cuda.Stream()
    lin(a, activation="silu", stream=s)
    torch.cuda.synchronize()
    buffers = binding.workspaces() + list(i4g._workspaces.values())
    assert len(binding.workspaces()) >= 2 and i4g._workspaces
    for ws in buffers:
        ws[:4096].view(torch.int32).fill_(1)  # as half-arrived tiles leave them
    i4g.selftest_wait_timeout(1000)
    assert i4g.device_status() == -8
    assert not binding.workspaces()
    assert all(not ws[:4096].any() for ws in i4g._workspaces.values())
    for _ in range(2):
        assert torch.equal(lin(a, activation="silu"), want) and torch.equal(lin(b), plain)
        got = lin(a, activation="silu", stream=s)
        s.synchronize()
        assert torch.equal(got, want)
    assert i4g.device_status() == 0 and binding.workspaces()


def test_graphs_share_nothing(i4g):
    """Two captured graphs replayed on two streams at once, and eager calls
    between: every result as if run alone."""
    M, N, K = 24, 1024, 8192
    assert i4g.gemm_epilogue_workspace_size(M, N, K) > 0
    lin, _ = make(i4g, K, N, 128)
    a = [rand(M, K, seed=20 + i) for i in range(3)]
    want = [lin(x, activation="silu", gated=True) for x in a]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(lin(a[i], activation="silu", gated=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = lin(a[2], activation="silu", gated=True)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(eager, want[2])
    assert i4g.device_status() == 0


def test_explicit_streams(i4g):
    lin, _ = make(i4g, 2048, 512, 64)
    a = rand(16, 2048, seed=1)
    want = lin(a, activation="relu")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        x = a.clone()
        torch.cuda.synchronize()
        got = lin(x, activation="relu", stream=stream)
        del x  # its memory may be reused only after the call
        torch.empty(16, 2048, dtype=torch.float16, device="cuda").fill_(7)
        s.synchronize()
        assert torch.equal(got, want)


def test_sharded_columns_gated(i4g):
    lin, _ = make(i4g, 512, 1024, 128)
    a = rand(9, 512, seed=2)
    bias = rand(1024, seed=3)
    whole = lin(a, activation="silu", gated=True, bias=bias)
    for rank in range(2):
        part = lin.shard(2, rank)
        got = part(a, activation="silu", gated=True, bias=bias[rank * 512:(rank + 1) * 512])
        assert torch.equal(got, whole[:, rank * 256:(rank + 1) * 256])


def test_from_gate_up_columns(i4g):
    gate, up = rand(256, 128, seed=1, scale=0.05), rand(256, 128, seed=2, scale=0.05)
    lin = i4g.QuantizedLinear.from_gate_up(gate, up, 64)
    a = rand(12, 256, seed=3)
    got = lin(a, activation="gelu_tanh", gated=True)
    g, u = a.double() @ ref.weight(gate, 64), a.double() @ ref.weight(up, 64)
    want = ref.activation(g, "gelu_tanh") * u
    from sm_120__gemm_b200.linear import interleave_gate_up
    w64 = interleave_gate_up(ref.weight(gate, 64), ref.weight(up, 64))
    expected, tol = ref.linear(a, w64, "gelu_tanh", True)
    assert torch.allclose(want, expected, rtol=1e-12, atol=1e-12)
    ref.check(got, expected, tol)
