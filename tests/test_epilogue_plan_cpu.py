"""The host's plan of the epilogue product and of the experts' products
(i4g_epilogue_plan), and that the shapes of the GPU tests reach every instance
of the kernel. No GPU."""
import ctypes

import pytest

import tile_cases

NULL, SHAPE = -1, -2
HEIGHTS = {16, 32, 64, 128, 256}


@pytest.fixture(scope="module")
def m():
    import sm_120__gemm_b200 as mod
    mod.load()
    return mod


@pytest.mark.parametrize("case", tile_cases.DENSE)
def test_dense_cases(m, case):
    _, _, M, N, K = case
    tile_cases.check_dense(m.epilogue_plan(M, N, K, 148), case)


@pytest.mark.parametrize("case", tile_cases.EXPERTS)
def test_expert_cases(m, case):
    _, _, _, T, E, k, K, N = case
    plan = m.epilogue_plan(T * k, N, K, 148, expert_rows=tile_cases.expert_rows(T, E, k))
    tile_cases.check_experts(plan, case)


def test_every_instance_is_reached():
    for cases in (tile_cases.DENSE, tile_cases.EXPERTS):
        reached = {(c[0], c[-1], c[1]) for c in tile_cases.by_group(cases)}
        assert reached == {(h, g, cut) for h in HEIGHTS for g in (32, 64, 128)
                           for cut in (False, True)}


def test_heights_of_the_other_tests(m):
    """The shapes that the tests of tile heights and of row gathers are written for."""
    dense = {32: [(17, 18944, 1088), (25, 20480, 2048), (90, 2432, 12416)],
             64: [(33, 18944, 1088), (63, 14336, 2112), (160, 4096, 4160)],
             128: [(65, 9600, 2112), (127, 18944, 1088), (513, 9472, 1088), (1000, 1920, 4160)],
             256: [(129, 18944, 576), (203, 18944, 320), (255, 18944, 576), (203, 9600, 8256)]}
    for height, shapes in dense.items():
        for s in shapes:
            assert m.epilogue_plan(*s, 148)["tile_rows"] == height, s
    experts = {32: [(100, 8, 2, 1088, 4864), (150, 4, 2, 4160, 1280)],
               64: [(240, 8, 2, 1088, 4864), (350, 4, 2, 4160, 1280)],
               128: [(450, 8, 2, 320, 4864), (1200, 5, 1, 576, 4864)],
               256: [(1500, 5, 2, 576, 4864), (700, 3, 1, 4160, 4864)]}
    for height, shapes in experts.items():
        for T, E, k, K, N in shapes:
            assert m.epilogue_plan(T * k, N, K, 148, E=E)["tile_rows"] == height, (T, E, k, K, N)


def test_decode_kernel_and_whole_waves(m):
    assert m.epilogue_plan(1, 4096, 4096, 148)["tile_rows"] == 0
    assert m.epilogue_plan(1, 4096, 4096, 148, E=1)["tile_rows"] != 0  # experts: never decode
    assert m.epilogue_plan(17, 18944, 8192, 148)["shares"] == 0  # 148 tiles: no tail
    assert m.epilogue_plan(40, 4096, 64, 148)["shares"] == 0     # too short to cut


def test_rows_up_to_32_bits(m):
    """Row counts that a tile's height more would take past 32 bits are refused by every
    entry point that takes them; the largest others have a plan."""
    most = 2 ** 31 - 1 - 256
    n = ctypes.c_size_t()
    for E in (0, 1, 3):
        assert m.epilogue_plan(most, 128, 64, 148, E=E)["tile_rows"] == 256
        for rows in (most + 1, 2 ** 31 - 1):
            with pytest.raises(m.I4GError):
                m.epilogue_plan(rows, 128, 64, 148, E=E)
    for rows in (most + 1, 2 ** 31 - 1):
        lib = m.load()
        assert lib.i4g_gemm_epilogue_workspace_size(rows, 128, 64, ctypes.byref(n)) == SHAPE
        assert lib.i4g_experts_workspace_size(rows, 3, 128, 64, ctypes.byref(n)) == SHAPE


def test_rows_of_experts_beyond_the_pairs(m):
    rows = [5, 0, 3]
    plan = m.epilogue_plan(8, 128, 8192, 148, expert_rows=rows)
    assert plan["tail_tiles"] == 2 and plan["shares"] == 16
    with pytest.raises(m.I4GError):
        m.epilogue_plan(7, 128, 8192, 148, expert_rows=rows)
    with pytest.raises(m.I4GError):
        m.epilogue_plan(8, 128, 8192, 148, expert_rows=[-1, 3])
    for bad in ((0, 128, 128, 148), (8, 100, 128, 148), (8, 128, 100, 148), (8, 128, 128, 0)):
        with pytest.raises(m.I4GError):
            m.epilogue_plan(*bad)
    with pytest.raises(m.I4GError):
        m.epilogue_plan(8, 128, 128, 148, E=513)
    n = ctypes.c_int()
    assert m.load().i4g_epilogue_plan(8, 0, None, 128, 128, 148, None, n, n, n) == NULL
