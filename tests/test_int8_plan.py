"""How attention over an 8-bit cache is shared out: in its own tiles."""

import numpy as np
import pytest


def plan(api, lengths, heads, ctas, **cache):
    work, join = [], []
    for line in api.attention_plan(lengths, heads, ctas, **cache).splitlines():
        kind, *v = line.split()
        (work if kind == "work" else join).append([int(x) for x in v])
    return work, join


@pytest.mark.parametrize("dtype,dim,tile", [("int8", 16, 128), ("int8", 128, 128), ("int8", 144, 64), ("int8", 256, 64),
                                            ("bf16", 128, 64), ("f32", 8, 64)])
@pytest.mark.parametrize("seed", range(6))
def test_tiles_are_those_of_the_cache(api, dtype, dim, tile, seed):
    rng = np.random.default_rng(seed)
    lengths = [int(x) for x in np.exp(rng.uniform(0, 9, int(rng.integers(1, 20))))]
    lengths[0] = 9000  # longer than a row that has a CTA of its own
    heads, ctas = int(rng.integers(1, 4)), int(rng.integers(1, 300))
    work, join = plan(api, lengths, heads, ctas, dtype=dtype, head_dim=dim)
    tiles = np.repeat([-(-n // tile) for n in lengths], heads)
    first = np.concatenate([[0], np.cumsum(tiles)])
    seen = np.zeros(first[-1], int)
    touched = {}
    for c, (row, at, count) in enumerate(work):
        seen[first[row] + at : first[row] + at + count] += 1
        for r in range(row, int(np.searchsorted(first, first[row] + at + count))):
            touched.setdefault(r, []).append(c)
    assert (seen == 1).all()
    assert {r: (cs[0], len(cs)) for r, cs in touched.items() if len(cs) > 1} == {r: (c, k) for r, c, k, _ in join}


def test_short_rows_have_a_cta_each(api):
    # Up to 512 slots, whatever the tile.
    for lengths, tiles in (([512, 129], [4, 2]), ([511], [4])):
        work, join = plan(api, lengths, 1, 100, dtype="int8", head_dim=64)
        assert not join and [w[2] for w in work] == tiles
    assert plan(api, [513], 1, 100, dtype="int8", head_dim=64)[1]


def test_the_plan_without_a_type_is_that_of_wider_caches(api):
    assert api.attention_plan([1000, 70], 2, 9) == api.attention_plan([1000, 70], 2, 9, dtype="bf16", head_dim=64)
    assert api.attention_plan([1000, 70], 2, 9) != api.attention_plan([1000, 70], 2, 9, dtype="int8")


@pytest.mark.parametrize("dtype,dim", [("int8", 24), ("int8", 0), ("f32", 12), ("f32", 264), ("int4", 64)])
def test_caches_that_there_are_not(api, dtype, dim):
    with pytest.raises(api.InvalidArgument, match="plan|dtype"):
        api.attention_plan([64], 1, 8, dtype=dtype, head_dim=dim)
