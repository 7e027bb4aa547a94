"""Attention over an 8-bit cache with logits of any size. The slots that count have
the same key, so their logits are the same to the bit, the others' lie so far
below that they weigh nothing, and the result is the mean of their values, however
large the logit is.

Tolerance, beside a mean v: weights are whole units of at most 2^-21.99 of the
largest weight x scale in a tile, off by half a unit, and meet codes of up to 127
(whatever a tile has: the whole sum is off by n of those); exponentials of 0 and of
whole numbers, sums of n equal weights and the products that follow stay within
(2 n + 128) 2^-24 of the sum of weight x |v|."""

import numpy as np
import pytest

import int8_cache
from test_shared_prefix import Shared

U = 2.0**-24
LOGITS = [s * 2.0**e for e in (10, 14, 15, 16, 17, 18, 20, 22) for s in (1.0, -1.37)]


def sizes(rng, n):
    """Rows' largest sizes whose scales lie closely above, on and below a power of two."""
    return (127 * 2.0 ** rng.integers(-30, 30, n) * (1 + rng.uniform(-0.001, 0.01, n))).astype(np.float32)


def of_size(rng, top, dim):
    x = rng.uniform(-1, 1, (*top.shape, dim)).astype(np.float32) * top[..., None]
    x[..., 3] = top
    return x


def means(host, hot, group):
    """(result, tolerance, scores) where the slots `hot`[s] of sequence s count alike."""
    n = len(host.lengths)
    out, tol = np.zeros((n, host.heads * group, host.dim)), np.zeros((n, host.heads * group, host.dim))
    scores = np.zeros((n, host.heads, max(host.lengths)))
    for s in range(n):
        v, at = host.stored(host.v[s])[hot[s]], len(hot[s])
        unit = int8_cache.quantise(host.v[s])[1].astype(np.float64)[hot[s]]
        whole = 127 * 2.0**-22.9 * unit.max(0)
        out[s] = np.repeat(v.mean(0), group, 0)
        tol[s] = np.repeat((2 * at + 128) * U * np.abs(v).mean(0) + whole[:, None], group, 0) + 1e-37
        scores[s][:, hot[s]] = group / at
    return out, tol, scores


def scale_for(logit, dim):
    """q = k = 16 in every channel: a logit of `logit` in units of log2."""
    return logit / (256 * dim * 1.4426950408889634)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [16, 128, 256])
def test_one_slot_gives_its_value(gpu, dim):
    rng = np.random.default_rng(dim)
    n, heads, group = 3000, 2, 2
    host = int8_cache.Host(rng, [1] * n, heads, dim, 8)
    for s in range(n):
        host.k[s][:] = 16
        host.v[s] = of_size(rng, sizes(rng, heads)[None], dim)
    _, batch = host.build(gpu)
    q = gpu.tensor([n, heads * group, dim], np.full((n, heads * group, dim), 16, np.float32))
    out, tol, scores = means(host, [[0]] * n, group)
    for logit in LOGITS:
        got = gpu.paged_attention(q, batch, scale=scale_for(logit, dim)).cpu().reshape(out.shape)
        assert (np.abs(got - out) <= tol).all(), logit
        again, new = gpu.paged_attention_scored(q, batch, scale=scale_for(logit, dim))
        assert np.array_equal(again.cpu().reshape(out.shape), got)
        assert (np.abs(new.cpu().reshape(scores.shape) - scores) <= 64 * U * scores).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 4), (128, 12), (192, 3)])
def test_slots_that_count_alike_among_others(gpu, dim, group):
    # In one tile and in several, split over CTAs and joined.
    rng = np.random.default_rng(dim + group)
    lengths = [2, 127, 128, 129, 500, 3000] * 20 + [30000]
    host = int8_cache.Host(rng, lengths, 1, dim, 64)
    hot = []
    for s, n in enumerate(lengths):
        hot.append(np.sort(rng.choice(n, min(n, int(rng.integers(1, 9))), replace=False)))
        host.k[s][:] = 0
        host.k[s][hot[s]] = 16
        # What does not count has values of any size; what does, of about one.
        top = sizes(rng, n) if s % 2 else np.repeat(sizes(rng, 1), n)
        top[hot[s]] = sizes(rng, 1) * (1 + rng.uniform(0, 0.002, len(hot[s])))
        host.v[s] = of_size(rng, top[:, None], dim)
    _, batch = host.build(gpu)
    q = gpu.tensor([len(lengths), group, dim], np.full((len(lengths), group, dim), 16, np.float32))
    out, tol, scores = means(host, hot, group)
    for logit in [x for x in LOGITS if x > 0]:
        got, new = gpu.paged_attention_scored(q, batch, scale=scale_for(logit, dim))
        assert (np.abs(got.cpu().reshape(out.shape) - out) <= tol).all(), logit
        assert (np.abs(new.cpu().reshape(scores.shape) - scores) <= 64 * U * scores).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [80, 128])
def test_behind_a_shared_prefix(gpu, dim):
    from porch_b200._lib import lib

    rng = np.random.default_rng(dim)
    members, shared, groups = 6, 192, 50
    n = members * groups
    host = Shared(rng, [(members, shared)] * groups, [shared + 1 + s % 3 for s in range(n)], 1, dim, 64, "int8")
    hot = []
    for s in range(n):
        first = s // members * members
        host.k[s][:] = 0
        if s == first:
            host.v[s] = of_size(rng, sizes(rng, len(host.v[s]))[:, None], dim)
        else:
            host.v[s][:shared] = host.v[first][:shared]
            host.v[s][shared:] = of_size(rng, sizes(rng, len(host.v[s]) - shared)[:, None], dim)
        # Of every group's slots one in the prefix counts, or each sequence's last one.
        hot.append([7 * (first // members) % shared if first // members % 2 else host.lengths[s] - 1])
        host.k[s][hot[s]] = 16
    assert lib().pb_test_share_prefix(1) == 0
    try:
        _, batch = host.build(gpu)
        q = gpu.tensor([n, 4, dim], np.full((n, 4, dim), 16, np.float32))
        out, tol, _ = means(host, hot, 4)
        for logit in [x for x in LOGITS if x > 0]:
            got = gpu.paged_attention(q, batch, scale=scale_for(logit, dim)).cpu().reshape(out.shape)
            assert (np.abs(got - out) <= tol).all(), logit
    finally:
        assert lib().pb_test_share_prefix(0) == 0
