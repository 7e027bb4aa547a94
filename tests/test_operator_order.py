"""Operators see what the calls before them wrote, on one stream, where each launch
begins beside the last one's end."""

import re

import numpy as np
import pytest


def test_every_kernel_waits_for_those_before_it(api):
    # Unconditionally: a launch that may begin early and does not wait has no
    # promise that it sees what was written before.
    sources = re.split(r"^kernel \S+ : operator$", api.operator_sources(), flags=re.M)[1:]
    assert len(sources) > 20
    for source in sources:
        waits = [line for line in source.splitlines() if "griddepcontrol.wait" in line and not line.lstrip().startswith("//")]
        assert waits and all(re.fullmatch(r'\s*asm volatile\("griddepcontrol\.wait;" ::: "memory"\);', w) for w in waits)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32", "int8"])
@pytest.mark.parametrize("members,shared,own", [(64, 1024, 400), (40, 4096, 30)])
def test_queries_and_rows_that_were_just_written(gpu, dtype, members, shared, own):
    # Each step writes over the same rows of the cache and makes queries in memory
    # that the step before used, by launches of a few CTAs, and attention follows at
    # once. A query is +-1 in every channel, the newest key 1, the others near 0, so
    # a head's result is the newest value or the others' mean.
    from porch_b200._lib import lib

    rng = np.random.default_rng(own)
    heads, group, dim, page, steps = 2, 4, 128, 16, 24
    before, after = shared // page, -(-own // page)
    pages = before + members * after
    order = rng.permutation(pages).astype(np.int32)
    tables = np.concatenate([np.tile(order[:before], (members, 1)), order[before:].reshape(members, after)], 1)
    cache = gpu.KVCache(pages, page, heads, dim, dtype=dtype)
    small = [rng.normal(0, 0.02, (pages * page, heads, dim)).astype(np.float32) for _ in range(2)]
    cache.batch(np.arange(pages)[None], [pages * page], appended=[pages * page]).append(
        *(gpu.tensor(list(x.shape), x) for x in small))
    lengths = [shared + own] * members
    signs = rng.choice([-1.0, 1.0], (steps, members, heads * group)).astype(np.float32)
    values = rng.normal(0, 1, (steps, members, heads, dim)).astype(np.float32)
    q = [gpu.tensor([members, heads * group, dim], np.repeat(s[..., None], dim, -1)) for s in signs]
    v = [gpu.tensor([members, heads, dim], x) for x in values]
    one = gpu.full([members, heads, dim], 1.0)
    unit, cos, sin, at = gpu.full([dim], 1.0), gpu.full([4, dim // 2], 1.0), gpu.zeros([4, dim // 2]), gpu.zeros([members])
    assert lib().pb_test_share_prefix(1) == 0
    try:
        batch = cache.batch(tables, lengths, prefix=[shared] * members)
        got = []
        for i in range(steps):
            turned, _ = gpu.qk_norm_rope(q[i], one, unit, unit, cos, sin, at)
            batch.append(one, v[i])
            got.append(gpu.paged_attention(turned, batch))
            del turned
        got = [x.cpu().reshape(members, heads * group, dim) for x in got]
    finally:
        assert lib().pb_test_share_prefix(0) == 0
    # Logits: 128 / sqrt(128) = 11.3 for the newest slot, the others' are sums of
    # 128 terms of size 0.02 times that rate, so below 0.2 but for one in millions;
    # 4200 of them weigh at most 4200 e^-11.1 = 6.4 % beside it, and average to 0.
    for i in range(steps):
        newest = np.repeat(values[i], group, 1)
        says = signs[i][..., None] > 0
        assert np.abs(np.where(says, got[i] - newest, 0)).max() <= 0.07 * np.abs(newest).max() + 0.05
        assert np.abs(np.where(says, 0, got[i])).max() <= 0.05
