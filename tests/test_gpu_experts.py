"""Routing, the experts' products and their combination against plain 64-bit
implementations (operators_ref.py)."""
import numpy as np
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


def rand(*shape, seed=0, scale=1.0, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def check_route(i4g, x, k, **kw):
    r = i4g.route(x, k, **kw)
    torch.cuda.synchronize()
    ids, w, offsets, rows, slots = ref.route(x, k, **kw)
    np.testing.assert_array_equal(r.ids.cpu().numpy(), ids)
    np.testing.assert_array_equal(r.offsets.cpu().numpy(), offsets)
    np.testing.assert_array_equal(r.rows.cpu().numpy(), rows)
    np.testing.assert_array_equal(r.slots.cpu().numpy(), slots)
    # exp within 2 units in the last place of 2^-23, sums of 512 and 32 terms
    # (16 + 5 and 5 additions on a term's way), two quotients, two products
    tol = (2 + 21 + 5 + 4) * 2.0 ** -23 * 2
    got = r.weights.cpu().double().numpy()
    assert (np.abs(got - w) <= tol * np.abs(w) + 1e-37).all(), np.abs(got - w).max()
    return r


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (1, 64, 8), (3, 7, 7), (17, 33, 5),
                                   (128, 64, 6), (129, 64, 6), (200, 160, 8), (1000, 256, 8),
                                   (333, 512, 32), (5, 512, 10), (2500, 96, 3)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_route(i4g, T, E, k, scoring, dtype):
    check_route(i4g, rand(T, E, seed=T + E, scale=1.5, dtype=dtype), k, scoring=scoring)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("E,groups,keep,k", [(64, 8, 3, 6), (256, 8, 4, 8), (160, 8, 3, 6),
                                             (60, 5, 2, 4), (32, 32, 7, 5), (24, 2, 2, 8),
                                             (512, 16, 1, 32)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_route_groups(i4g, scoring, bias, E, groups, keep, k, group_score):
    x = rand(150, E, seed=E, scale=1.5, dtype=torch.float32)
    b = rand(E, seed=1, scale=0.1, dtype=torch.float32) if bias else None
    check_route(i4g, x, k, scoring=scoring, bias=b, n_group=groups, topk_group=keep,
                group_score=group_score, renormalize=bias, scale=2.5)


def test_route_ties_go_to_the_lowest_index(i4g):
    x = torch.randint(-3, 4, (400, 48), device="cuda",
                      generator=torch.Generator(device="cuda").manual_seed(1)).float()
    x[0] = 0
    x[1, ::2], x[1, 1::2] = 0.0, -0.0  # equal, whatever their sign
    check_route(i4g, x, 8)
    check_route(i4g, x, 8, scoring="sigmoid", bias=torch.zeros(48, device="cuda"))
    check_route(i4g, x.half(), 8, n_group=6, topk_group=2, group_score="top2")
    # sums that only differ far below FP32: decided as in FP64
    b = 0.25 + torch.arange(48, device="cuda").float() * 2.0 ** -24
    check_route(i4g, x * 1e-3, 8, scoring="sigmoid", bias=b)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,G", [(8, 2), (32, 4), (60, 6)])
def test_route_groups_whose_terms_cancel(i4g, scoring, E, G):
    """A group's two best may be large and of opposite sign: the order of their
    sums is still FP64's. Biases that no FP32 score could resolve, masks by the
    type's lowest value and infinite ones among them."""
    x = rand(1000, E, seed=E, dtype=torch.float32)
    bias = torch.full((E,), -2.0 ** 23, device="cuda")
    size = E // G
    for g in range(G):
        bias[g * size], bias[g * size + 1] = 2.0 ** (20 - g % 2), -2.0 ** (20 - g % 2)
    kw = dict(scoring=scoring, n_group=G, group_score="top2")
    check_route(i4g, x, 2, bias=bias, topk_group=1, **kw)
    check_route(i4g, x, 2, bias=-bias, topk_group=G - 1, **kw)
    bias[size:] = torch.finfo(torch.float32).min
    check_route(i4g, x, 2, bias=bias, topk_group=1, **kw)
    bias[-size:] = -2.9e38  # sums that FP32 cannot hold, in order
    check_route(i4g, x, 2, bias=bias, topk_group=min(2, G - 1), **kw)
    bias[:size] = 0.0
    bias[-1] = np.inf
    check_route(i4g, x, 2, bias=bias, topk_group=1, **kw)


def test_route_masks_infinities_and_nan(i4g):
    x = rand(300, 32, seed=4, dtype=torch.float32)
    x[5] = -np.inf          # a padded token
    x[6, 3:] = -np.inf      # three experts left, for k = 6
    x[7, 4] = float("nan")
    x[8] = float("nan")
    x[9, 2] = x[9, 20] = np.inf
    x[10] = torch.finfo(torch.float32).min
    x[11] = torch.finfo(torch.float32).max
    x[12, 1:] = -3e38
    for n in (300, 13):
        for kw in (dict(), dict(renormalize=False), dict(n_group=4, topk_group=2)):
            check_route(i4g, x[:n], 6, **kw)
        r = i4g.route(x[:n], 6, scoring="sigmoid", bias=rand(32, seed=5, dtype=torch.float32))
        assert (r.ids[5] == -1).all() and (r.ids[8] == -1).all() and not r.weights[5].any()
        assert (r.ids[6, 3:] == -1).all() and sorted(r.ids[6, :3].tolist()) == [0, 1, 2]
        assert 4 not in r.ids[7].tolist()
    b = torch.zeros(32, device="cuda")
    b[3], b[9] = -np.inf, float("nan")
    r = i4g.route(x[13:], 32, scoring="sigmoid", bias=b)
    assert not (r.ids == 3).any() and not (r.ids == 9).any() and (r.ids[:, 30:] == -1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("T", [12, 700])
def test_route_weights_of_scores_below_fp32(i4g, dtype, T):
    """Chosen experts whose scores FP32 cannot hold still share a token's weight:
    FP64 holds sigmoids of logits down to -708 (and gives 0 for the last row's)."""
    x = rand(T, 40, seed=T, scale=2.0, dtype=torch.float32)
    top = torch.tensor([-60.0, -79.0, -81.0, -86.0, -87.3, -88.0, -89.0, -95.0, -120.0, -300.0,
                        -650.0, -900.0], device="cuda")
    low = (x + top.repeat((T + 11) // 12)[:T, None]).to(dtype)
    spread = low.clone()
    spread[:, 1:6] -= 40  # some of a token's experts in range, others below it
    spread[:, 20] = -3.0
    one_high = rand(T, 40, seed=1, dtype=dtype)
    bias = torch.zeros(40, device="cuda")
    bias[5:12] = 8.0  # chosen first, far below the largest logit
    one_high[:, 5:12] -= 120
    one_high[T // 2:, 5:12] -= 200
    infinite = one_high.clone()
    infinite[:, 5] = np.inf
    for kw in (dict(), dict(scale=2.5), dict(renormalize=False, scale=3.0),
               dict(n_group=4, topk_group=2, group_score="top2")):
        for logits in (low, spread):
            check_route(i4g, logits, 5, scoring="sigmoid", **kw)
        check_route(i4g, one_high, 5, bias=bias, **kw)
        check_route(i4g, infinite, 5, bias=bias, **kw)
    w = i4g.route(low[:11], 5, scoring="sigmoid").weights.sum(1)
    assert ((w - 1).abs() <= 8 * 2.0 ** -24).all()  # five roundings of the weights


def test_route_all_rows_masked(i4g):
    for T in (4, 600):
        r = check_route(i4g, torch.full((T, 16), -np.inf, device="cuda"), 4)
        assert (r.rows == -1).all() and not r.offsets.any()


def test_route_strided_empty_and_streams(i4g):
    wide = rand(140, 100, seed=1, dtype=torch.float32)
    check_route(i4g, wide[:, 3:67], 4)
    check_route(i4g, wide[::2, 3:66], 4)
    check_route(i4g, rand(40, 30, seed=2).t(), 4)
    check_route(i4g, wide[:1, :20].expand(30, 20), 4)
    r = i4g.route(wide[:0, :64], 4)
    assert r.ids.shape == (0, 4) and not r.offsets.any() and r.offsets.shape == (65,)
    want = i4g.route(wide, 4)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = i4g.route(wide, 4, stream=s)
    s.synchronize()
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    for bad in (dict(n_group=3), dict(n_group=4, topk_group=5), dict(n_group=50, topk_group=1)):
        with pytest.raises(i4g.I4GError):
            i4g.route(wide, 4, **bad)
    with pytest.raises(i4g.I4GError):
        i4g.route(wide, 33)
    with pytest.raises(ValueError):
        i4g.route(wide, 4, bias=torch.zeros(99, device="cuda"))
    with pytest.raises(TypeError):
        i4g.route(wide.double(), 4)


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (5, 7, 3), (40, 65, 5)])
def test_route_results_do_not_overlap(i4g, T, E, k):
    x = rand(T, E, seed=3, dtype=torch.float32)
    want = [t.clone() for t in i4g.route(x, k)]
    for i in range(5):
        got = i4g.route(x, k)
        assert all(t.is_contiguous() and t.data_ptr() % 16 == 0 for t in got)
        got[i].fill_(-7)
        assert (got[i] == -7).all()
        assert all(torch.equal(a, b) for j, (a, b) in enumerate(zip(got, want)) if j != i)


def routing_of(i4g, ids, E):
    offsets, rows, slots = ref.order(ids, E)
    T, k = ids.shape
    w = rand(T, k, seed=5, dtype=torch.float32).abs() if T else torch.zeros(0, k, device="cuda")
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).int().cuda()  # noqa: E731
    return i4g.Routing(t(ids), w, t(offsets), t(rows), t(slots))


def choices(kind, T, E, k, seed=0):
    rng = np.random.default_rng(seed)
    if kind == "one":  # every token the same experts
        return np.tile(np.arange(k), (T, 1))
    if kind == "skewed":  # expert 0 for every token, the others at random
        rest = np.stack([1 + rng.permutation(E - 1)[:k - 1] for _ in range(T)])
        return np.concatenate([np.zeros((T, 1), int), rest], axis=1)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]) if T else np.zeros((0, k), int)
    if kind == "padded":
        ids[rng.random(T) < 0.3] = -1
        ids[rng.random(ids.shape) < 0.1] = -1
    return ids


def check_experts(i4g, kind, T, E, k, K, N, group, act="none", gated=False, bias=False,
                  gather=True, fp32=False):
    w = rand(E, K, N, seed=1, scale=0.05)
    ex = i4g.QuantizedExperts.from_weight(w, group)
    r = routing_of(i4g, choices(kind, T, E, k), E)
    a = rand(T if gather else T * k, K, seed=2)
    b = rand(E, N, seed=3) if bias else None
    cols = N // 2 if gated else N
    out = torch.full((T * k, cols), 77.0, dtype=torch.float32 if fp32 else torch.float16,
                     device="cuda")
    got = ex(a, r, gather=gather, bias=b, activation=act, gated=gated, out=out, fp32_out=fp32)
    torch.cuda.synchronize()
    assert i4g.device_status() == 0 and got is out
    edges = r.offsets.tolist()
    for e in range(E):
        lo, hi = edges[e], edges[e + 1]
        if lo == hi:
            continue
        src = a[(r.rows[lo:hi] // k).long()] if gather else a[lo:hi]
        want, tol = ref.linear(src, ref.weight(w[e], group), act, gated,
                               None if b is None else b[e], None, fp32)
        ref.check(got[lo:hi], want, tol)
    assert (got[edges[E]:] == 77).all()  # rows behind the last expert's
    return ex, r, a


@pytest.mark.parametrize("kind", ["random", "one", "skewed", "padded"])
@pytest.mark.parametrize("T,E,k", [(1, 8, 3), (9, 16, 2), (70, 5, 3), (300, 4, 2), (520, 33, 2)])
@pytest.mark.parametrize("gather", [True, False])
def test_experts(i4g, kind, T, E, k, gather):
    check_experts(i4g, kind, T, E, k, 192, 256, 64, "silu", True, True, gather)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("act,gated", [("none", False), ("gelu", False), ("gelu_tanh", True),
                                       ("relu", False)])
@pytest.mark.parametrize("T", [4, 150])
def test_experts_epilogues(i4g, group, act, gated, T):
    check_experts(i4g, "random", T, 6, 2, 256, 128, group, act, gated, bias=True)


@pytest.mark.parametrize("T,E,k,K,N", [(1, 16, 8, 4096, 256), (3, 8, 2, 8192, 128),
                                       (64, 4, 2, 4160, 640), (900, 3, 1, 8192, 256)])
def test_experts_split_tails(i4g, T, E, k, K, N):
    ex, r, a = check_experts(i4g, "random", T, E, k, K, N, 64, "silu", True)
    first = ex(a, r, activation="silu", gated=True)
    n = int(r.offsets[-1])
    for _ in range(30):
        assert torch.equal(ex(a, r, activation="silu", gated=True)[:n], first[:n])


# tiles of 32 rows (the first two), 64, 128 and 256
@pytest.mark.parametrize("T,E,k,K,N", [(100, 8, 2, 1088, 4864), (150, 4, 2, 4160, 1280),
                                       (240, 8, 2, 1088, 4864), (350, 4, 2, 4160, 1280),
                                       (450, 8, 2, 320, 4864), (1200, 5, 1, 576, 4864),
                                       (1500, 5, 2, 576, 4864), (700, 3, 1, 4160, 4864)])
@pytest.mark.parametrize("kind,gather", [("random", True), ("skewed", True), ("padded", False)])
def test_experts_tile_heights(i4g, T, E, k, K, N, kind, gather):
    if kind == "skewed" and k == 1:
        kind = "one"  # a token has one expert: all of them the first
    check_experts(i4g, kind, T, E, k, K, N, 64, "silu", True, True, gather)


# without a workspace nothing is split or copied ahead: tokens' rows are gathered
# inside the product at every tile height
@pytest.mark.parametrize("T,E,k,K,N", [(9, 8, 2, 320, 384), (100, 8, 2, 1088, 4864),
                                       (240, 8, 2, 1088, 4864), (450, 8, 2, 320, 4864),
                                       (1500, 5, 2, 576, 4864)])
@pytest.mark.parametrize("kind", ["random", "padded"])
def test_experts_without_a_workspace(i4g, T, E, k, K, N, kind):
    w = rand(E, K, N, seed=1, scale=0.05)
    ex = i4g.QuantizedExperts.from_weight(w, 64)
    r = routing_of(i4g, choices(kind, T, E, k), E)
    a = rand(T, K, seed=2)
    got = torch.full((T * k, N), 77.0, dtype=torch.float16, device="cuda")
    i4g.launch_experts(a, T, ex.tiles, ex.scales, got, r.offsets, r.rows, k, T * k, E, N, K, 64,
                       activation="relu")
    torch.cuda.synchronize()
    assert i4g.device_status() == 0
    edges = r.offsets.tolist()
    for e in range(E):
        lo, hi = edges[e], edges[e + 1]
        if lo < hi:
            src = a[(r.rows[lo:hi] // k).long()]
            ref.check(got[lo:hi], *ref.linear(src, ref.weight(w[e], 64), "relu"))
    assert (got[edges[E]:] == 77).all()


def test_experts_fp32_one_expert_and_many(i4g):
    check_experts(i4g, "one", 30, 1, 1, 128, 128, 32, fp32=True, bias=True)
    check_experts(i4g, "padded", 40, 512, 4, 64, 128, 64, "relu")


def test_experts_empty_and_refusals(i4g):
    w = rand(4, 128, 128, seed=1, scale=0.05)
    ex = i4g.QuantizedExperts.from_weight(w, 64)
    empty = i4g.route(torch.zeros(0, 4, device="cuda"), 2)
    assert ex(rand(0, 128), empty).shape == (0, 128)
    assert i4g.combine(rand(0, 128), empty).shape == (0, 128)
    r = i4g.route(rand(6, 4, dtype=torch.float32), 2)
    a = rand(6, 128)
    for bad in (dict(a=rand(5, 128)), dict(a=rand(12, 128)), dict(a=rand(6, 64)),
                dict(a=a.float()), dict(a=a, gather=False), dict(a=a, activation="tanh"),
                dict(a=a, bias=rand(128)), dict(a=a, out=torch.zeros(12, 64).half().cuda()),
                dict(a=a.cpu())):
        bad = dict(bad)
        with pytest.raises((ValueError, TypeError)):
            ex(bad.pop("a"), r, **bad)
    with pytest.raises(ValueError):  # a routing over other experts
        ex(a, i4g.route(rand(6, 5, dtype=torch.float32), 2))


def test_experts_bad_tables_are_clamped(i4g):
    """Offsets outside the rows, falling offsets and rows outside A come to no
    harm: every access stays inside the buffers (guards around them keep)."""
    E, K, N, T, k = 4, 128, 128, 20, 2
    ex = i4g.QuantizedExperts.from_weight(rand(E, K, N, seed=1, scale=0.05), 64)
    good = routing_of(i4g, choices("random", T, E, k), E)
    a = rand(T, K, seed=2)
    guard = torch.full((T * k + 64, N), 5.0, dtype=torch.float16, device="cuda")
    out = guard[32:32 + T * k]
    for offsets in ([0, 10, 20, 30, 1000000], [-5, 10, 5, 30, 40], [40, 30, 20, 10, 0]):
        r = good._replace(offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        ex(a, r, out=out)
    r = good._replace(rows=torch.full_like(good.rows, 1 << 30))
    ex(a, r, out=out)
    assert (out == 0).all()  # rows outside A read as zeros
    r = good._replace(rows=torch.full_like(good.rows, -7))
    ex(a, r, out=out)
    torch.cuda.synchronize()
    assert (guard[:32] == 5).all() and (guard[32 + T * k:] == 5).all()
    assert i4g.device_status() == 0


def test_experts_row_copy_is_the_calls_own(i4g):
    """Of a call's workspace only counters and partial sums stay with the package; the
    copy of the gathered rows goes back when the call returns."""
    T, E, k, K, N = 4096, 64, 8, 2048, 256
    ex = i4g.QuantizedExperts.from_weight(rand(E, K, N, seed=1, scale=0.05), 64)
    r = i4g.route(rand(T, E, seed=1, dtype=torch.float32), k)
    a = rand(T, K, seed=2)
    torch.cuda.synchronize()
    i4g.reset_workspaces()
    before = torch.cuda.memory_allocated()
    y = ex(a, r)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    copy = T * k * K * 2
    assert i4g.experts_workspace_size(T * k, E, N, K) > copy  # rows are copied ahead here
    assert held < copy // 2
    # one buffer for everything gives the same, and so does a graph
    ws = torch.zeros(i4g.experts_workspace_size(T * k, E, N, K), dtype=torch.uint8, device="cuda")
    got = torch.empty_like(y)
    i4g.launch_experts(a, T, ex.tiles, ex.scales, got, r.offsets, r.rows, k, T * k, E, N, K, 64,
                       workspace=ws)
    assert torch.equal(got, y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ex(a, r)
    for _ in range(3):
        out.zero_()
        g.replay()
        assert torch.equal(out, y)
    assert torch.equal(ex(a.repeat_interleave(k, 0)[r.rows.long()], r, gather=False), y)
    assert i4g.device_status() == 0


@pytest.mark.parametrize("T,E,k,K,N", [(9, 8, 2, 320, 384), (40, 12, 8, 128, 128),
                                       (240, 8, 2, 1088, 4864), (1500, 5, 4, 576, 4864)])
def test_experts_rows_outside_a_read_as_zeros(i4g, T, E, k, K, N):
    """-1 (routing's own mark) down to -(k - 1), and rows behind A: zeros, whether
    they are gathered inside the product or copied ahead of it."""
    w = rand(E, K, N, seed=1, scale=0.05)
    ex = i4g.QuantizedExperts.from_weight(w, 64)
    r = routing_of(i4g, choices("random", T, E, k), E)
    a = rand(T, K, seed=2)
    bias = rand(E, N, seed=3)
    rows = r.rows.clone()
    outside = torch.arange(T * k, device="cuda") % 5 < 2
    marks = torch.tensor([-1, 1 - k, T * k, -(2 ** 31), 2 ** 31 - 1], dtype=torch.int32,
                         device="cuda")
    rows[outside] = marks[torch.arange(int(outside.sum()), device="cuda") % 5]
    expert = torch.bucketize(torch.arange(T * k, device="cuda"), r.offsets[1:].long(), right=True)
    zeros = bias[expert].relu()
    whole = ex(a, r, bias=bias, activation="relu")
    need = i4g.experts_workspace_size(T * k, E, N, K)
    for n in (0, need):
        ws = torch.zeros(n, dtype=torch.uint8, device="cuda") if n else None
        got = torch.empty(T * k, N, dtype=torch.float16, device="cuda")
        i4g.launch_experts(a, T, ex.tiles, ex.scales, got, r.offsets, rows, k, T * k, E, N, K, 64,
                           bias=bias, activation="relu", workspace=ws)
        assert torch.equal(got[outside], zeros[outside])
        # elsewhere what the rows inside A gave: two roundings to FP16, and sums of
        # magnitudes up to 60 in another order, 2e-5 of them
        near = (got - whole)[~outside].abs() <= 2.0 ** -9 * whole[~outside].abs() + 2.0 ** -9
        assert near.all()
    assert i4g.device_status() == 0


def test_experts_offsets_that_fall_stay_in_the_workspace(i4g):
    """Offsets that fall and rise again name more tiles than any routing: nothing is
    written, neither to C nor behind the workspace (guards of 1 MB around both)."""
    E, K, N, M = 16, 8192, 128, 64
    ex = i4g.QuantizedExperts.from_weight(rand(E, K, N, seed=1, scale=0.05), 64)
    a = rand(M, K, seed=2)
    need = i4g.experts_workspace_size(M, E, N, K)
    assert need > 4096
    guard = 1 << 20
    held = torch.full((guard + need + guard,), 9, dtype=torch.uint8, device="cuda")
    ws = held[guard:guard + need]
    ws.zero_()
    out = torch.full((M, N), 5.0, dtype=torch.float16, device="cuda")
    rows = torch.arange(M, dtype=torch.int32, device="cuda")
    for offsets in ([0, M] * 8 + [0], [0] + [M, 0] * 8, [0] * 15 + [M, M - 1]):
        t = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        for r in (None, rows):
            i4g.launch_experts(a, M, ex.tiles, ex.scales, out, t, r, 1, M, E, N, K, 64,
                               workspace=ws)
    torch.cuda.synchronize()
    assert i4g.device_status() == 0
    assert (out == 5).all() and not ws[:4096].any()
    assert (held[:guard] == 9).all() and (held[guard + need:] == 9).all()
    # and the workspace still serves a routing
    t = torch.arange(E + 1, dtype=torch.int32, device="cuda") * (M // E)
    i4g.launch_experts(a, M, ex.tiles, ex.scales, out, t, None, 1, M, E, N, K, 64, workspace=ws)
    other = torch.empty_like(out)
    i4g.launch_experts(a, M, ex.tiles, ex.scales, other, t, None, 1, M, E, N, K, 64)
    assert (out != 5).any() and (out - other).abs().max() <= 2.0 ** -9 * other.abs().max()


@pytest.mark.parametrize("T,k,N", [(1, 1, 8), (1, 8, 4096), (7, 2, 1000), (300, 8, 256),
                                   (40, 32, 64), (65, 11, 136)])
@pytest.mark.parametrize("residual", [False, True])
def test_combine(i4g, T, k, N, residual):
    E = max(40, k)
    r = routing_of(i4g, choices("padded", T, E, k), E)
    y = rand(T * k, N, seed=3)
    res = rand(T, N, seed=4) if residual else None
    got = i4g.combine(y, r, residual=res)
    slot = r.slots.long()
    part = r.weights.double()[..., None] * y.double()[slot.clamp(min=0)]
    part = torch.where((slot >= 0)[..., None], part, torch.zeros_like(part))
    want = part.sum(1) + (res.double() if residual else 0)
    # k + 1 additions of FP32 terms, one rounding to FP16
    tol = (k + 1) * 2.0 ** -24 * (part.abs().sum(1) + (res.double().abs() if residual else 0))
    ref.check(got, want, tol + 2.0 ** -11 * (want.abs() + tol) + 2.0 ** -25)


def test_combine_skips_and_in_place(i4g):
    r = routing_of(i4g, np.array([[0, 1], [-1, 1], [-1, -1]]), 2)
    y = rand(6, 64, seed=1)
    y[3:] = float("nan")  # rows no slot names
    x = rand(3, 64, seed=2)
    want = i4g.combine(y, r, residual=x)
    assert want.isfinite().all() and torch.equal(want[2], x[2])
    out = x.clone()
    i4g.combine(y, r, residual=out, out=out)
    assert torch.equal(out, want)
    bad = r._replace(slots=torch.full_like(r.slots, 1 << 20))
    assert torch.equal(i4g.combine(y, bad, residual=x), x)
    for kw in (dict(residual=rand(3, 32)), dict(out=rand(2, 64)), dict(out=rand(3, 128)[:, ::2])):
        with pytest.raises(ValueError):
            i4g.combine(y, r, **kw)
    with pytest.raises(i4g.I4GError):
        i4g.combine(rand(6, 12), r)


def test_launch_functions(i4g):
    """The C ABI's Python mirrors, as a caller with its own buffers uses them."""
    T, E, k, K, N, g = 9, 6, 2, 128, 128, 64
    ex = i4g.QuantizedExperts.from_weight(rand(E, K, N, seed=1, scale=0.05), g)
    x = rand(T, K, seed=2)
    logits = rand(T, E, seed=3, dtype=torch.float32)
    want = i4g.route(logits, k, scoring="sigmoid", scale=0.5)
    i32 = dict(dtype=torch.int32, device="cuda")
    r = i4g.Routing(torch.empty(T, k, **i32), torch.empty(T, k, device="cuda"),
                    torch.empty(E + 1, **i32), torch.empty(T * k, **i32),
                    torch.empty(T, k, **i32))
    assert i4g.route_workspace_size(T, E) == 0 and i4g.route_workspace_size(5000, E) > 0
    options = i4g.RouteOptions(i4g.SCORINGS["sigmoid"], 1, 1, i4g.GROUP_SCORES["max"], 1, 0.5)
    i4g.launch_route(logits, True, E, None, T, E, k, options, *r)
    for p, q in zip(r, want):
        assert torch.equal(p, q)
    y = torch.empty(T * k, N, dtype=torch.float16, device="cuda")
    ws = torch.zeros(max(256, i4g.experts_workspace_size(T * k, E, N, K)), dtype=torch.uint8,
                     device="cuda")
    i4g.launch_experts(x, T, ex.tiles, ex.scales, y, r.offsets, r.rows, k, T * k, E, N, K, g,
                       activation="relu", workspace=ws)
    assert torch.equal(y, ex(x, want, activation="relu"))
    out = torch.empty(T, N, dtype=torch.float16, device="cuda")
    i4g.launch_combine(y, T * k, r.slots, r.weights, None, out, T, k, N)
    assert torch.equal(out, i4g.combine(y, want))
    with pytest.raises(i4g.I4GError):
        i4g.launch_route(logits, True, E, None, 5000, E, k, options, *r)  # no workspace


def plain_moe(x, logits, k, wg, wu, wd, group, act, residual, **route_kw):
    """The block in 64 bits, rounded to fp16 where the block rounds."""
    ids, w, *_ = ref.route(logits, k, **route_kw)
    out = residual.double().clone()
    for t in range(x.shape[0]):
        for j, e in enumerate(ids[t]):
            if e < 0:
                continue
            a = x[t:t + 1].double()
            h = (ref.activation(a @ wg[e], act) * (a @ wu[e])).half().double()
            out[t] += float(w[t, j]) * (h @ wd[e]).half().double()[0]
    return out


@pytest.mark.parametrize("T", [1, 5, 150])
def test_block_together(i4g, T):
    """Dense gate/up -> down as one MLP, and the routed block: as they are used."""
    E, k, K, F = 8, 2, 256, 128
    g, u = rand(E, K, F, seed=1, scale=0.08), rand(E, K, F, seed=2, scale=0.08)
    d = rand(E, F, K, seed=3, scale=0.08)
    mlp = i4g.ExpertMLP(i4g.QuantizedExperts.from_gate_up(g, u, 64),
                        i4g.QuantizedExperts.from_weight(d, 64))
    x = rand(T, K, seed=4)
    logits = rand(T, E, seed=5, dtype=torch.float32)
    if T > 3:
        logits[2] = -np.inf  # a padded token
    r = i4g.route(logits, k, scoring="sigmoid", scale=2.0)
    got = mlp(x, r, residual=x)
    w64 = [[ref.weight(w[e], 64) for e in range(E)] for w in (g, u, d)]
    want = plain_moe(x, logits, k, *w64, 64, "silu", x, scoring="sigmoid", scale=2.0)
    # an intermediate rounding may fall the other way: 2^-10 of each term, and
    # the final half step
    scale = want.abs().max() + 1
    assert (got.double() - want).abs().max() <= scale * (2.0 ** -9)
    if T > 3:
        assert torch.equal(got[2], x[2])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (s, s.cuda_stream):
        other = mlp(x, r, residual=x, stream=stream)
        s.synchronize()
        assert torch.equal(other, got)


def test_block_in_a_graph(i4g):
    """The routed block captured once and replayed over new inputs: the routing
    changes from replay to replay."""
    E, k, K, F, T = 16, 4, 512, 256, 20
    mlp = i4g.ExpertMLP(
        i4g.QuantizedExperts.from_gate_up(rand(E, K, F, seed=1, scale=0.05),
                                          rand(E, K, F, seed=2, scale=0.05), 128),
        i4g.QuantizedExperts.from_weight(rand(E, F, K, seed=3, scale=0.05), 128))
    x = rand(T, K, seed=4)
    logits = rand(T, E, seed=5, dtype=torch.float32)
    bias = rand(E, seed=6, scale=0.1, dtype=torch.float32)

    def block():
        r = i4g.route(logits, k, scoring="sigmoid", bias=bias, n_group=4, topk_group=2,
                      group_score="top2")
        return mlp(x, r, residual=x)

    block()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = block()
    for i in range(10):
        x.copy_(rand(T, K, seed=100 + i))
        logits.copy_(rand(T, E, seed=200 + i, dtype=torch.float32))
        if i == 4:
            logits[3:9] = -np.inf
        g.replay()
        got = out.clone()
        assert torch.equal(got, block())
    assert i4g.device_status() == 0
