"""Eviction against its definition: the kept slots, their scores and positions,
and the rows that moved, bit for bit."""

import numpy as np
import pytest

import paged

pytestmark = pytest.mark.gpu


def rows_of(pool, host, s, length):
    """[length, heads, dim] of sequence s as the pool holds it, in raw bits."""
    import torch

    x = torch.as_tensor(pool, device="cuda")
    x = (x.view(torch.int16) if host.dtype == "bf16" else x.view(torch.int32)).cpu().numpy()
    at = host.tables[s, : -(-length // host.page)] if length else []
    return x[at].transpose(0, 2, 1, 3).reshape(-1, host.heads, host.dim)[:length]


def bits(host, x):
    x = np.ascontiguousarray(host.stored(x))
    return (x.view(np.uint32) >> 16).astype(np.uint16).view(np.int16) if host.dtype == "bf16" else x.view(np.int32)


CASES = [
    # lengths, heads, head size, page, type, budget, recent, sinks
    ([40], 1, 8, 8, "f32", 8, 2, 1),
    ([40, 8, 7, 0, 1, 9], 2, 64, 16, "bf16", 8, 0, 0),
    ([33, 34], 3, 80, 8, "f32", 32, 32, 0),
    ([500, 499], 2, 24, 32, "bf16", 1, 0, 0),
    ([500, 499], 2, 24, 32, "bf16", 1, 1, 0),
    ([5000, 1025, 1024, 1023], 2, 128, 64, "bf16", 1024, 100, 4),
    ([3001], 5, 72, 256, "f32", 2900, 1000, 16),
    ([70001, 20], 1, 16, 128, "bf16", 4097, 1024, 4),
    ([200000], 1, 8, 256, "bf16", 100000, 1000, 4),
    ([300, 250], 1, 40, 8, "f32", 280, 20, 260),
    ([9000] * 3 + [8, 8999], 8, 16, 64, "bf16", 700, 64, 4),
    ([33000, 32999, 5], 2, 16, 64, "bf16", 20000, 64, 4),
    ([420000, 1500], 1, 8, 256, "bf16", 3000, 500, 4),
    ([420000, 1500], 1, 8, 256, "f32", 419000, 500, 4),
    ([30, 20], 2, 8, 8, "f32", 5000, 500, 4),
    ([393217, 4096, 4097], 1, 8, 256, "bf16", 4096, 0, 0),
]


@pytest.mark.parametrize("lengths,heads,dim,page,dtype,budget,recent,sinks", CASES)
@pytest.mark.parametrize("seen", [False, True])
def test_against_the_definition(gpu, lengths, heads, dim, page, dtype, budget, recent, sinks, seen):
    rng = np.random.default_rng(sum(lengths) + budget + seen)
    host = paged.Host(rng, lengths, heads, dim, page, dtype)
    n, longest = len(lengths), max(lengths)
    newest = [max(0, 2 * x - 1) if seen else max(0, x - 1) for x in lengths]
    cache, batch = host.build(gpu, newest)
    scores = np.exp(rng.normal(0, 2, (n, heads, longest))).astype(np.float32)
    scores[rng.random(scores.shape) < 0.3] = 0.25  # many ties
    scores[rng.random(scores.shape) < 0.05] = 0.0
    places = None
    if seen:  # some places known, some not, fewer than there are slots
        places = rng.integers(0, max(1, longest), (n, heads, max(1, longest // 2))).astype(np.float32)
        places[rng.random(places.shape) < 0.2] = -1
    given = None if places is None else gpu.tensor(list(places.shape), places)
    t = gpu.tensor(list(scores.shape), scores)
    out, where = gpu.cache_evict(batch, t, given, budget=budget, recent=recent, sinks=sinks)
    source, want, want_where = paged.evict(lengths, newest, scores, places, budget, recent, sinks)
    assert np.array_equal(out.cpu().reshape(want.shape), want)
    assert np.array_equal(where.cpu().reshape(want.shape), want_where)
    assert np.array_equal(t.cpu().reshape(scores.shape), scores)
    for pool, rows in zip(cache.pools(), (host.k, host.v)):
        for s, length in enumerate(lengths):
            m = min(length, budget)
            got = rows_of(pool, host, s, m)
            for h in range(heads):
                assert np.array_equal(got[:, h], bits(host, rows[s][source[s, h, :m], h]))
    # The same call once more gives the same: nothing that it reads has changed.
    out, where = gpu.cache_evict(batch, t, given, budget=budget, recent=recent, sinks=sinks)
    assert np.array_equal(out.cpu().reshape(want.shape), want)
    assert np.array_equal(where.cpu().reshape(want.shape), want_where)


def test_scores_that_are_not_finite_and_signed_zeros(gpu):
    rng = np.random.default_rng(1)
    host = paged.Host(rng, [64], 1, 8, 8, "f32")
    _, batch = host.build(gpu)
    scores = rng.choice(np.array([0.0, -0.0, -1.0, np.inf, -np.inf, np.nan, 3e38, -3e38, 1e-40, -1e-40], np.float32),
                        (1, 1, 60))  # four slots without a score
    for budget in (5, 20, 40, 63):
        source, want, where = paged.evict([64], [63], scores, None, budget, 3, 2)
        out, got = gpu.cache_evict(batch, gpu.tensor([1, 1, 60], scores), budget=budget, recent=3, sinks=2)
        assert np.array_equal(got.cpu().reshape(where.shape), where)
        assert np.array_equal(out.cpu().reshape(want.shape), want, equal_nan=True)


def test_decoding_with_eviction(gpu):
    """Steps of append, scored attention and eviction, against the same in numpy."""
    rng = np.random.default_rng(12)
    heads, group, dim, page, budget = 2, 3, 32, 8, 24
    host = paged.Host(rng, [20, 23], heads, dim, page, "bf16", spare=4)
    host.tables = np.concatenate([host.tables, [[p] for p in set(range(host.pages)) - set(host.tables.ravel())][:2]], 1)
    cache, batch = host.build(gpu)
    scores, places = None, None
    w_scores, w_places = np.zeros((2, heads, 0), np.float32), None
    newest = [19, 22]
    for step in range(12):
        k, v = (rng.normal(0, 1, (2, heads, dim)).astype(np.float32) for _ in range(2))
        host.lengths = [n + 1 for n in host.lengths]
        newest = [n + 1 for n in newest]
        for s in range(2):
            host.k[s] = np.concatenate([host.k[s], k[s : s + 1]])
            host.v[s] = np.concatenate([host.v[s], v[s : s + 1]])
        batch = cache.batch(host.tables, host.lengths, newest=newest)
        batch.append(gpu.tensor([2, heads, dim], k), gpu.tensor([2, heads, dim], v))
        q = rng.normal(0, 2, (2, heads * group, dim)).astype(np.float32)
        want, tol, w_new, new_tol = host.attend(q, 0.2, w_scores)
        out, scores = gpu.paged_attention_scored(gpu.tensor(list(q.shape), q), batch, scores, scale=0.2)
        assert (np.abs(out.cpu().reshape(want.shape) - want) <= tol).all()
        got = scores.cpu().reshape(w_new.shape)
        assert (np.abs(got - w_new) <= new_tol).all()
        w_scores = got  # the device's own, so that both sides rank the same numbers
        if max(host.lengths) > budget + 3:
            source, w_scores, w_places = paged.evict(host.lengths, newest, w_scores, w_places, budget, 6, 2)
            scores, places = gpu.cache_evict(batch, scores, places, budget=budget, recent=6, sinks=2)
            assert np.array_equal(scores.cpu().reshape(w_scores.shape), w_scores)
            assert np.array_equal(places.cpu().reshape(w_places.shape), w_places)
            for s in range(2):
                m = min(host.lengths[s], budget)
                at = source[s, :, :m].T[..., None]
                host.k[s], host.v[s] = (np.take_along_axis(x[s], at, 0) for x in (host.k, host.v))
            host.lengths = [min(n, budget) for n in host.lengths]
