"""Shapes that run every instance of the epilogue kernel on 148 SMs: each tile
height with whole tiles and with a tail cut along K, for each scale group.

K / 64 is odd where the group allows (32, 64: the last stage of two or four
blocks is short), and for group 128 even but no multiple of four: the last of
a 16- to 64-row tile's stages holds two blocks, and at 256 rows, where a stage
is one block, a scale group spans two stages and a share may start between them.
"""

# (tile height, tail cut along K, M, N, K)
DENSE = [
    (16, False, 17, 128, 320), (16, False, 17, 128, 384),
    (16, True, 17, 128, 4160), (16, True, 17, 128, 4224),
    (32, False, 150, 1920, 320), (32, False, 150, 1920, 384),
    (32, True, 400, 384, 6464), (32, True, 400, 384, 6528),
    (64, False, 300, 1920, 320), (64, False, 300, 1920, 384),
    (64, True, 100, 1920, 8384), (64, True, 100, 1920, 8320),
    (128, False, 65, 9600, 320), (128, False, 65, 9600, 384),
    (128, True, 600, 1920, 12480), (128, True, 600, 1920, 12416),
    (256, False, 129, 9600, 320), (256, False, 129, 9600, 384),
    (256, True, 1000, 2432, 6464), (256, True, 1000, 2432, 6528),
]

# (tile height, tail cut, rows copied into expert order first, T, E, top_k, K, N),
# tokens spread by expert_rows()
EXPERTS = [
    (16, False, False, 7, 2, 1, 320, 128), (16, False, False, 7, 2, 1, 384, 128),
    (16, True, False, 7, 2, 1, 4160, 128), (16, True, True, 1100, 2, 1, 6528, 128),
    (32, False, False, 700, 3, 2, 320, 256), (32, False, True, 700, 3, 2, 1152, 256),
    (32, True, True, 1100, 2, 1, 8384, 128), (32, True, True, 1100, 2, 1, 8320, 128),
    (64, False, False, 1100, 2, 1, 320, 640), (64, False, True, 1100, 2, 1, 640, 640),
    (64, True, True, 700, 3, 2, 12480, 128), (64, True, True, 700, 3, 2, 12416, 128),
    (128, False, False, 450, 5, 2, 320, 1280), (128, False, True, 700, 3, 2, 384, 896),
    (128, True, True, 1100, 2, 1, 6464, 1920), (128, True, True, 1100, 2, 1, 6528, 1920),
    (256, False, True, 1100, 9, 3, 320, 640), (256, False, True, 1100, 9, 3, 384, 640),
    (256, True, True, 700, 5, 2, 4160, 1920), (256, True, True, 700, 5, 2, 4224, 1920),
]


def groups(K):
    return (128,) if K % 128 == 0 else (32, 64)


def ids(T, E, k):
    """Each token's experts, at random."""
    import numpy as np
    rng = np.random.default_rng(0)
    return np.stack([rng.permutation(E)[:k] for _ in range(T)])


def expert_rows(T, E, k):
    import numpy as np
    return np.bincount(ids(T, E, k).reshape(-1), minlength=E).tolist()


def by_group(cases):
    """The cases with each scale group they run."""
    return [(*c, g) for c in cases for g in groups(c[-1] if len(c) == 5 else c[-2])]


def check_dense(plan, case):
    height, cut = case[:2]
    assert plan["tile_rows"] == height and (plan["shares"] > 0) == cut, (case, plan)


def check_experts(plan, case):
    height, cut, copied = case[:3]
    assert plan["tile_rows"] == height and (plan["shares"] > 0) == cut, (case, plan)
    assert bool(plan["copy_rows"]) == copied, (case, plan)
