"""Attention of sequences that share a prefix, against the definition in 64
bits and the same cache without the prefix. Tolerances: paged.Host.attend and
int8_cache.Host.attend, whose sums may be taken in any order and parts."""

import numpy as np
import pytest

import int8_cache


@pytest.fixture(autouse=True)
def shared(request):
    """Prefixes are shared at these sizes, too, which the library would not do."""
    if request.node.get_closest_marker("gpu") is None:
        yield
        return
    from porch_b200._lib import lib

    assert lib().pb_test_share_prefix(1) == 0
    yield
    assert lib().pb_test_share_prefix(0) == 0


class Shared(int8_cache.Host):
    """Groups of (members, shared slots); lengths are whole ones."""

    def __init__(self, rng, groups, lengths, heads, dim, page, dtype):
        super().__init__(rng, lengths, heads, dim, page, dtype)
        self.prefix = [n for members, n in groups for _ in range(members)]
        first = 0
        for members, n in groups:
            for s in range(first + 1, first + members):
                self.tables[s, : n // page] = self.tables[first, : n // page]
                self.k[s][:n], self.v[s][:n] = self.k[first][:n], self.v[first][:n]
            first += members
        assert len(lengths) == first and all(n >= p for n, p in zip(lengths, self.prefix))

    def build(self, api):
        """Every slot that no sequence uses is NaN; shared ones are written again with the same values."""
        cache = api.KVCache(self.pages, self.page, self.heads, self.dim, dtype=self.dtype)
        total = self.pages * self.page
        everything = cache.batch(np.arange(self.pages)[None], [total], appended=[total])
        nan = api.tensor([total, self.heads, self.dim], np.full(total * self.heads * self.dim, np.nan, np.float32))
        everything.append(nan, nan)
        for s, n in enumerate(self.lengths):
            if n:
                one = cache.batch(self.tables[s : s + 1], [n], appended=[n])
                one.append(api.tensor([n, self.heads, self.dim], self.k[s]), api.tensor([n, self.heads, self.dim], self.v[s]))
        return cache, cache.batch(self.tables, self.lengths, appended=[0] * len(self.lengths), prefix=self.prefix)


CASES = [
    # groups (members, shared slots), lengths, kv heads, query heads per kv head, head size, page
    ([(2, 8)], [9, 8], 1, 1, 16, 8),
    ([(3, 64)], [65, 64, 200], 2, 4, 64, 16),
    ([(2, 16), (1, 0), (2, 48)], [17, 21, 5, 49, 50], 3, 5, 80, 16),
    ([(1, 0), (3, 2000), (1, 0)], [0, 2100, 2000, 2017, 0], 2, 3, 128, 8),
    ([(8, 640)], [641] * 8, 1, 2, 128, 64),
    ([(9, 640)], [700] * 9, 1, 2, 128, 64),
    ([(40, 1024)], list(range(1024, 1064)), 2, 4, 128, 32),
    ([(70, 256), (3, 512)], [256 + i % 5 for i in range(70)] + [600, 513, 512], 1, 2, 96, 256),
    ([(6, 4096), (5, 4096)], [4100] * 11, 1, 8, 112, 128),
    ([(130, 128)], [129] * 130, 1, 1, 64, 16),
    ([(2, 20000)], [20001, 20777], 1, 16, 128, 8),
    ([(5, 320)], [330] * 5, 2, 7, 256, 64),
    ([(3, 8)], [9, 9, 9], 1, 40, 32, 8),
    ([(33, 8200)], [8300] * 33, 1, 4, 48, 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32", "int8"])
@pytest.mark.parametrize("groups,lengths,heads,group,dim,page", CASES)
def test_against_the_definition(gpu, groups, lengths, heads, group, dim, page, dtype):
    rng = np.random.default_rng(sum(lengths) + dim)
    host = Shared(rng, groups, lengths, heads, dim, page, dtype)
    _, batch = host.build(gpu)
    q = rng.normal(0, 2, (len(lengths), heads * group, dim)).astype(np.float32)
    out, tol, _, _ = host.attend(q, dim**-0.5)
    got = gpu.paged_attention(gpu.tensor(list(q.shape), q), batch).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()
    # Few of the same batch's heads, and another scale: a plan of its own.
    few = np.ascontiguousarray(q[:, ::group])
    out, tol, _, _ = host.attend(few, 0.2)
    got = gpu.paged_attention(gpu.tensor(list(few.shape), few), batch, scale=0.2).cpu().reshape(few.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32", "int8"])
def test_logits_far_apart_and_queries_read_in_place(gpu, dtype):
    # The weight lies wholly in the prefix, wholly behind it, or on one slot of each.
    rng = np.random.default_rng(5)
    lengths = [400 + i for i in range(20)]
    host = Shared(rng, [(20, 384)], lengths, 2, 64, 32, dtype)
    fused = rng.normal(0, 1, (20, 11, 66)).astype(np.float32)
    for s in range(20):
        at = [(3 * s) % 384, lengths[s] - 1][s % 2]
        fused[s, 2:6, 1:65] = 8 * host.stored(host.k[s])[at].repeat(2, 0)
    q = fused[:, 2:6, 1:65]
    _, batch = host.build(gpu)
    view = gpu.materialize(gpu.tensor([20, 11, 66], fused)[gpu.all, 2:6, 1:65])
    out, tol, _, _ = host.attend(np.ascontiguousarray(q), 1.0)
    got = gpu.paged_attention(view, batch, scale=1.0).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32", "int8"])
def test_values_that_are_not_finite_stay_with_their_readers(gpu, dtype):
    rng = np.random.default_rng(2)
    host = Shared(rng, [(20, 128), (2, 64)], [140] * 20 + [70, 80], 2, 64, 16, dtype)
    q = rng.normal(0, 1, (22, 4, 64)).astype(np.float32)
    _, batch = host.build(gpu)
    want = gpu.paged_attention(gpu.tensor([22, 4, 64], q), batch).cpu().reshape(q.shape)
    host.v[1][139, 0, 5] = np.nan  # behind the prefix: one sequence
    for s in range(20):
        host.k[s][64, 1, 0] = np.nan  # in it: all that share it
    q2 = q.copy()
    q2[7, 0, 60] = np.nan
    q2[8, 1, 60] = np.inf
    bad = np.zeros(q.shape, bool)
    bad[1, :2, :] = True if dtype == "int8" else np.arange(64) == 5
    bad[:20, 2:] = bad[7, 0] = bad[8, 1] = True
    _, batch = host.build(gpu)
    got = gpu.paged_attention(gpu.tensor([22, 4, 64], q2), batch).cpu().reshape(q.shape)
    assert not np.isfinite(got[bad]).any() and np.array_equal(got[~bad], want[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32", "int8"])
@pytest.mark.parametrize("below", [128, 384])
def test_logits_below_the_range_of_float32_weigh_nothing(gpu, dtype, below):
    # Whole tiles of the prefix, or all of it, have logits past float32's range.
    rng = np.random.default_rng(below)
    host = Shared(rng, [(20, 384)], [400] * 20, 1, 64, 32, dtype)
    for s in range(20):
        host.k[s][:, :, 0] = 0
        host.k[s][:below] = 0
        host.k[s][:below, :, 0] = -(2.0**84)
    q = rng.normal(0, 1, (20, 2, 64)).astype(np.float32)
    q[:, :, 0] = 2.0**50
    q[:, :, 1:] *= np.float32(2.0**45)
    _, batch = host.build(gpu)
    t = gpu.tensor([20, 2, 64], q)
    scale = 2.0**-47
    host.k, host.v = ([x[below:] for x in y] for y in (host.k, host.v))
    host.lengths = [400 - below] * 20
    out, tol, _, _ = host.attend(q if dtype == "int8" else np.where(np.arange(64) == 0, 0, q).astype(np.float32), scale)
    got = gpu.paged_attention(t, batch, scale=scale).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_scores_and_appending_and_another_layer(gpu, dtype):
    rng = np.random.default_rng(9)
    lengths = [200 + i for i in range(18)]
    host = Shared(rng, [(18, 192)], lengths, 2, 64, 64, dtype)
    cache, _ = host.build(gpu)
    # A step: every sequence's newest token goes in behind the prefix.
    batch = cache.batch(host.tables, lengths, prefix=host.prefix)
    for s, n in enumerate(lengths):
        host.k[s][n - 1], host.v[s][n - 1] = rng.normal(0, 1, (2, 2, 64)).astype(np.float32)
    rows = [gpu.tensor([18, 2, 64], np.stack([x[n - 1] for x, n in zip(y, lengths)])) for y in (host.k, host.v)]
    batch.append(*rows)
    q = rng.normal(0, 1, (18, 8, 64)).astype(np.float32)
    t = gpu.tensor([18, 8, 64], q)
    out, tol, new, new_tol = host.attend(q, 0.125)
    first = gpu.paged_attention(t, batch).cpu().reshape(q.shape)
    assert (np.abs(first - out) <= tol).all()
    # Scored attention takes no notice of the prefix.
    got, weights = gpu.paged_attention_scored(t, batch)
    plain, same = gpu.paged_attention_scored(t, cache.batch(host.tables, lengths))
    assert np.array_equal(got.cpu(), plain.cpu()) and np.array_equal(weights.cpu(), same.cpu())
    assert (np.abs(weights.cpu().reshape(new.shape) - new) <= new_tol).all()
    k, v = (x.cpu().reshape(-1, 2, 64) for x in batch.read())
    assert len(k) == sum(lengths)
    other = gpu.KVCache(host.pages, 64, 2, 64, dtype=dtype)
    for s, n in enumerate(lengths):
        one = other.batch(host.tables[s : s + 1], [n], appended=[n])
        one.append(gpu.tensor([n, 2, 64], host.v[s]), gpu.tensor([n, 2, 64], host.k[s]))
    host.k, host.v = host.v, host.k
    out, tol, _, _ = host.attend(q, 0.125)
    assert (np.abs(gpu.paged_attention(t, batch.on(other)).cpu().reshape(q.shape) - out) <= tol).all()
    for _ in range(3):
        assert np.array_equal(gpu.paged_attention(t, batch).cpu().reshape(q.shape), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_by_size(gpu, dtype):
    # Without the hook: a small prefix is each sequence's own, to the bit; a large
    # one is shared, and its attention the definition's.
    from porch_b200._lib import lib

    assert lib().pb_test_share_prefix(0) == 0
    rng = np.random.default_rng(8)
    for members, shared, heads, same in ((20, 512, 2, True), (120, 2048, 4, False)):
        lengths = [shared + 1 + i % 3 for i in range(members)]
        host = Shared(rng, [(members, shared)], lengths, heads, 128, 64, dtype)
        cache, batch = host.build(gpu)
        q = rng.normal(0, 1, (members, heads, 128)).astype(np.float32)
        t = gpu.tensor(list(q.shape), q)
        got = gpu.paged_attention(t, batch).cpu()
        plain = gpu.paged_attention(t, cache.batch(host.tables, lengths, appended=[0] * members)).cpu()
        assert np.array_equal(got, plain) == same
        out, tol, _, _ = host.attend(q, 128**-0.5)
        assert (np.abs(got.reshape(q.shape) - out) <= tol).all()
        # Again, by a batch whose plan was made with it.
        again = cache.batch(host.tables, lengths, appended=[0] * members, prefix=host.prefix)
        assert np.array_equal(gpu.paged_attention(t, again).cpu(), got)


@pytest.mark.gpu
def test_a_prefix_that_nobody_shares(gpu):
    rng = np.random.default_rng(3)
    host = Shared(rng, [(1, 32), (1, 32), (1, 0)], [40, 50, 33], 2, 64, 16, "bf16")
    cache, batch = host.build(gpu)
    q = rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    t = gpu.tensor([3, 4, 64], q)
    plain = cache.batch(host.tables, host.lengths)
    assert np.array_equal(gpu.paged_attention(t, batch).cpu(), gpu.paged_attention(t, plain).cpu())


@pytest.mark.gpu
def test_from_several_threads(gpu):
    import threading

    rng = np.random.default_rng(4)
    host = Shared(rng, [(30, 1024)], [1100] * 30, 2, 128, 64, "bf16")
    cache, batch = host.build(gpu)
    q = rng.normal(0, 1, (30, 8, 128)).astype(np.float32)
    t = gpu.tensor([30, 8, 128], q)
    want, wrong = gpu.paged_attention(t, batch).cpu(), []

    def work():
        try:
            mine = cache.batch(host.tables, host.lengths, appended=[0] * 30, prefix=host.prefix)
            for _ in range(5):
                wrong.extend(x for x in [gpu.paged_attention(t, mine).cpu()] if not np.array_equal(x, want))
        except Exception as e:  # a thread's exception would be lost
            wrong.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [1, 2])
def test_waits_that_run_out_are_reported_and_the_gpu_recovers(gpu, mode):
    # Mode 1: the first CTA multiplies nothing, so its other roles' waits run out;
    # 2: its softmax gives up at once, while loads and products are on their way.
    from porch_b200._lib import lib

    rng = np.random.default_rng(6)
    host = Shared(rng, [(30, 1024)], [1100] * 30, 2, 128, 64, "bf16")
    _, batch = host.build(gpu)
    q = rng.normal(0, 1, (30, 4, 128)).astype(np.float32)
    t = gpu.tensor([30, 4, 128], q)
    want = gpu.paged_attention(t, batch).cpu()
    assert lib().pb_test_attention_stall(mode) == 0
    try:
        with pytest.raises(RuntimeError, match="kernel error code"):
            gpu.paged_attention(t, batch).cpu()
    finally:
        assert lib().pb_test_attention_stall(0) == 0
    for _ in range(2):
        assert np.array_equal(gpu.paged_attention(t, batch).cpu(), want)


@pytest.mark.gpu
def test_refusals(gpu):
    cache = gpu.KVCache(20, 16, 2, 64, dtype="bf16")
    tables = np.array([[0, 1, 2, 5], [0, 1, 3, 6], [0, 4, 7, 8]])
    for prefix, message in (([8, 8, 0], "whole pages"), ([-16, 0, 0], "whole pages"), ([32, 32, 32], "other pages"),
                            ([64, 64, 0], "before its length"), ([48, 48, 0], "other pages"), ([32, 32], "one whole length"),
                            ([32.0, 32.0, 0.0], "one whole length")):
        with pytest.raises(gpu.InvalidArgument, match=message):
            cache.batch(tables, [50, 49, 60], prefix=prefix)
    for lengths, appended in (([32, 50, 60], [1, 0, 0]), ([50, 31, 60], [0, 0, 0]), ([31, 50, 60], None)):
        with pytest.raises(gpu.InvalidArgument, match="before its length and its new tokens"):
            cache.batch(tables, lengths, appended=appended, prefix=[32, 32, 0])
    cache.batch(tables, [32, 50, 60], prefix=[32, 32, 0]).append(gpu.zeros([2, 2, 64]), gpu.zeros([2, 2, 64]))
    batch = cache.batch(tables, [50, 49, 60], prefix=[32, 32, 16])
    with pytest.raises(gpu.InvalidArgument, match="more than one place"):
        gpu.cache_evict(batch, gpu.zeros([3, 2, 60]), budget=20)
    with pytest.raises(gpu.InvalidArgument, match="q must be"):
        gpu.paged_attention(gpu.zeros([2, 4, 64]), batch)


@pytest.mark.gpu
def test_a_prefix_past_two_to_the_32_bytes(gpu):
    pages, page, dim = ((1 << 24) + (1 << 20)) // 64, 64, 128
    cache = gpu.KVCache(pages, page, 1, dim, dtype="bf16")
    rng = np.random.default_rng(2)
    host = Shared(rng, [(30, 128)], [150] * 30, 1, dim, page, "bf16")
    host.tables = pages - 1 - np.maximum(host.tables, 0)
    for s in range(30):
        one = cache.batch(host.tables[s : s + 1], [150], appended=[150])
        one.append(gpu.tensor([150, 1, dim], host.k[s]), gpu.tensor([150, 1, dim], host.v[s]))
    q = rng.normal(0, 1, (30, 2, dim)).astype(np.float32)
    out, tol, _, _ = host.attend(q, dim**-0.5)
    batch = cache.batch(host.tables, [150] * 30, prefix=host.prefix)
    got = gpu.paged_attention(gpu.tensor(list(q.shape), q), batch).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
def test_many_parts_and_many_rows(gpu):
    # One long prefix of one key head in more parts than a warp joins, beside
    # groups and sequences of all kinds in one batch.
    rng = np.random.default_rng(12)
    groups = [(17, 12800), (1, 0), (2, 64), (1, 64), (40, 128), (3, 0), (5, 64)]
    lengths = [12800 + i for i in range(17)] + [0, 64, 65, 100] + [130] * 40 + [3, 0, 700] + [64, 65, 66, 67, 200]
    lengths = lengths[: sum(m for m, _ in groups)]
    host = Shared(rng, groups, lengths, 1, 64, 64, "bf16")
    _, batch = host.build(gpu)
    q = rng.normal(0, 2, (len(lengths), 2, 64)).astype(np.float32)
    out, tol, _, _ = host.attend(q, 0.125)
    got = gpu.paged_attention(gpu.tensor(list(q.shape), q), batch).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("members,shared,own,heads,group,dim", [
    (64, 4096, 250, 8, 4, 128), (64, 4096, 400, 8, 2, 64), (60, 1024, 700, 8, 1, 80), (63, 6144, 70, 8, 8, 16)])
def test_what_follows_runs_beside_the_prefix(gpu, members, shared, own, heads, group, dim):
    # More tiles behind the prefix than CTAs at once: the launches share the SMs.
    rng = np.random.default_rng(members + own)
    lengths = [shared + own + s % 5 for s in range(members)]
    lengths[7] = shared
    host = Shared(rng, [(members, shared)], lengths, heads, dim, 64, "bf16")
    _, batch = host.build(gpu)
    q = rng.normal(0, 1, (members, heads * group, dim)).astype(np.float32)
    t = gpu.tensor(list(q.shape), q)
    got = [gpu.paged_attention(t, batch).cpu() for _ in range(3)]
    out, tol, _, _ = host.attend(q, dim**-0.5)
    assert (np.abs(got[0].reshape(q.shape) - out) <= tol).all()
    assert all(np.array_equal(got[0], x) for x in got[1:])
