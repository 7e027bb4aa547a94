"""Whether a shared prefix is worked through once: where each sequence is better off
by itself the results are, to the bit, those of a batch that names no prefix."""

import numpy as np
import pytest


def same_as_alone(gpu, dtype, members, shared, heads, group, dim):
    rng = np.random.default_rng(members + shared)
    page = 64
    before = shared // page
    tables = np.concatenate([np.tile(np.arange(before), (members, 1)), before + np.arange(members)[:, None]], 1)
    cache = gpu.KVCache(before + members, page, heads, dim, dtype=dtype)
    total = (before + members) * page
    everything = cache.batch(np.arange(before + members)[None], [total], appended=[total])
    x = rng.normal(0, 1, (total, heads, dim)).astype(np.float32)
    t = gpu.tensor([total, heads, dim], x)
    everything.append(t, t)
    y = rng.normal(0, 1, (members, heads * group, dim)).astype(np.float32)
    q = gpu.tensor(list(y.shape), y)
    lengths = [shared + 1 + s % 60 for s in range(members)]
    batch = cache.batch(tables, lengths, appended=[0] * members, prefix=[shared] * members)
    alone = cache.batch(tables, lengths, appended=[0] * members)
    got, want = (gpu.paged_attention(q, b).cpu() for b in (batch, alone))
    # Two orders of sums: each is off by the roundings of its logits and of its sum of
    # weight x value; eight bits add units of 2^-22 of a tile's largest, 127 of them.
    logit = np.linalg.norm(x, axis=-1).max() * np.linalg.norm(y, axis=-1).max() * dim**-0.5
    rel = 2.0**-24 * (2 * (2 * dim + 64) * logit + 2 * max(lengths) + 128) + (2.0**-15 if dtype == "int8" else 0)
    assert np.abs(got - want).max() <= 2 * rel * np.abs(x).max()
    return np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,members,shared,heads,group,dim", [
    ("f32", 64, 384, 8, 4, 128),
    ("f32", 64, 256, 8, 4, 128),
    ("int8", 64, 1024, 8, 4, 128),
    ("bf16", 64, 256, 8, 4, 256),
    ("bf16", 8, 2048, 8, 4, 128),
    ("int8", 16, 4096, 8, 4, 256),
    # Eight queries a row at this head size, so that nothing is spared.
    ("f32", 2, 8192, 4, 8, 256),
    ("f32", 4, 4096, 4, 8, 256),
])
def test_by_themselves(gpu, dtype, members, shared, heads, group, dim):
    assert same_as_alone(gpu, dtype, members, shared, heads, group, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,members,shared,heads,group,dim", [
    ("f32", 16, 4096, 8, 2, 64),
    ("f32", 8, 4096, 4, 1, 256),
    ("int8", 64, 4096, 8, 2, 64),
    ("bf16", 64, 512, 8, 4, 128),
    ("bf16", 8, 4096, 8, 1, 256),
    ("bf16", 2, 16384, 8, 4, 128),
])
def test_once_for_all(gpu, dtype, members, shared, heads, group, dim):
    assert not same_as_alone(gpu, dtype, members, shared, heads, group, dim)
