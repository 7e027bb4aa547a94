"""A paged cache in 8 bits: what is written, read back, attended to and evicted,
against the definitions in 64 bits (tolerances: int8_cache.Host.attend)."""

import numpy as np
import pytest

import int8_cache
import paged


def pools(cache):
    """(codes, scales) of keys and of values, from the device."""
    torch = pytest.importorskip("torch")
    cache_codes = [torch.as_tensor(p, device="cuda") for p in cache.pools()]
    cache_scales = [torch.as_tensor(p, device="cuda") for p in cache.scales()]
    torch.cuda.synchronize()
    return [(c.cpu().numpy(), s.cpu().numpy()) for c, s in zip(cache_codes, cache_scales)]


def rows_of(pool, table, length, page):
    """[length, heads, ...] of a pool [pages, heads, page, ...]."""
    at = np.arange(length)
    return pool[table[at // page], :, at % page]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,page", [(1, 16, 8), (2, 64, 16), (3, 80, 32), (8, 128, 64), (5, 256, 256), (1, 240, 8)])
def test_what_is_written(gpu, heads, dim, page):
    rng = np.random.default_rng(dim)
    host = int8_cache.Host(rng, [37, 1, 100], heads, dim, page)
    host.k[0] *= np.exp(rng.uniform(-60, 60, host.k[0].shape[:2]))[..., None].astype(np.float32)
    host.v[2] *= rng.integers(0, 2, host.v[2].shape)
    # Borders: multiples of a half, of a power of two and of an odd largest size.
    top = np.array([127, 254, 127 * 3, 1, 2.0**-60, 3.3e38], np.float32)[rng.integers(0, 6, host.k[2].shape[:2])]
    host.k[2] = (rng.integers(-254, 255, host.k[2].shape) / 254 * top[..., None]).astype(np.float32)
    host.k[2][..., 3] = top
    cache, _ = host.build(gpu)
    for (codes, scales), x in zip(pools(cache), (host.k, host.v)):
        for s, length in enumerate(host.lengths):
            want, unit = int8_cache.quantise(x[s])
            assert np.array_equal(rows_of(codes, host.tables[s], length, page), want)
            assert np.array_equal(rows_of(scales, host.tables[s], length, page), unit)


@pytest.mark.gpu
def test_rows_that_have_no_codes(gpu):
    rng = np.random.default_rng(1)
    host = int8_cache.Host(rng, [9], 2, 32, 8)
    host.k[0][1, 0, 5], host.k[0][2, 1, 31], host.k[0][3, 0, 0] = np.nan, np.inf, -np.inf
    host.k[0][4] = 0
    host.k[0][5, 0] = np.float32(2.0**-97)
    host.k[0][5, 1, 0] = np.float32(2.0**-96)
    host.k[0][5, 1, 1:] = 0
    host.k[0][6, 0] = np.float32(1e-44)
    cache, batch = host.build(gpu)
    (codes, scales), _ = pools(cache)
    codes, scales = (rows_of(x, host.tables[0], 9, 8) for x in (codes, scales))
    want, unit = int8_cache.quantise(host.k[0])
    assert np.array_equal(codes, want) and np.array_equal(scales, unit, equal_nan=True)
    assert np.isnan(scales[[1, 2, 3], [0, 1, 0]]).all() and not scales[4].any() and scales[5, 0] == 0 and codes[5, 1, 0] == 127
    k, v = (x.cpu().reshape(9, 2, 32) for x in batch.read())
    bad = np.zeros((9, 2), bool)
    bad[[1, 2, 3], [0, 1, 0]] = True
    assert np.isnan(k[bad]).all() and np.isfinite(k[~bad]).all() and np.isfinite(v).all()


@pytest.mark.gpu
@pytest.mark.parametrize("first", [0, 1, 4])
def test_new_tokens_read_in_place(gpu, first):
    rng = np.random.default_rng(first)
    fused = rng.normal(0, 1, (33, 6, 52)).astype(np.float32)
    f = gpu.tensor([33, 6, 52], fused)
    k, v = (gpu.materialize(f[gpu.all, h : h + 2, first : first + 48]) for h in (1, 4))
    cache = gpu.KVCache(9, 8, 2, 48, dtype="int8")
    tables = np.array([[3, 1, -1], [0, 5, 2], [7, -1, -1]])
    batch = cache.batch(tables, [9, 20, 4], appended=[9, 20, 4])
    batch.append(k, v)
    ends = np.cumsum([0, 9, 20, 4])
    for (codes, scales), h in zip(pools(cache), (1, 4)):
        for s in range(3):
            want, unit = int8_cache.quantise(fused[ends[s] : ends[s + 1], h : h + 2, first : first + 48])
            assert np.array_equal(rows_of(codes, tables[s], len(want), 8), want)
            assert np.array_equal(rows_of(scales, tables[s], len(want), 8), unit)


@pytest.mark.gpu
def test_rows_behind_the_new_tokens_stay(gpu):
    rng = np.random.default_rng(4)
    host = int8_cache.Host(rng, [21, 8], 2, 32, 8)
    cache, _ = host.build(gpu)
    before = pools(cache)
    batch = cache.batch(host.tables, [21, 8], appended=[2, 0])
    x = rng.normal(0, 1, (2, 2, 32)).astype(np.float32)
    batch.append(gpu.tensor([2, 2, 32], x), gpu.tensor([2, 2, 32], -x))
    for (c0, s0), (c1, s1), y in zip(before, pools(cache), (x, -x)):
        at = [host.tables[0][i // 8] for i in (19, 20)]
        for i, p in zip((19, 20), at):
            want, unit = int8_cache.quantise(y[i - 19])
            assert np.array_equal(c1[p, :, i % 8], want) and np.array_equal(s1[p, :, i % 8], unit)
            c1[p, :, i % 8], s1[p, :, i % 8] = c0[p, :, i % 8], s0[p, :, i % 8]
        assert np.array_equal(c0, c1) and np.array_equal(s0, s1, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "int8"])
@pytest.mark.parametrize("lengths,heads,dim,page", [
    ([1], 1, 16, 8), ([0, 17, 0, 0, 5, 0], 3, 64, 16), ([300, 5, 129, 64], 5, 80, 128), ([7] * 300, 1, 16, 8),
    ([2000, 0, 3], 8, 128, 64), ([33, 70], 64, 256, 32), ([515], 1000, 16, 256), ([0, 0], 2, 32, 8)])
def test_reading_back(gpu, dtype, lengths, heads, dim, page):
    rng = np.random.default_rng(sum(lengths))
    host = int8_cache.Host(rng, lengths, heads, dim, page, dtype)
    _, batch = host.build(gpu)
    k, v = batch.read()
    assert k.shape() == v.shape() == [sum(lengths), heads, dim]
    if sum(lengths):
        for got, x in ((k, host.k), (v, host.v)):
            want = np.concatenate(x)
            if dtype == "int8":
                codes, scale = int8_cache.quantise(want)
                want = codes.astype(np.float32) * scale[..., None]
            else:
                want = host.stored(want)
            assert np.array_equal(got.cpu().reshape(want.shape), want)


@pytest.mark.gpu
def test_reading_pages_that_serve_two_sequences_and_writing_them_elsewhere(gpu):
    # What was read of one cache goes into another of another type.
    rng = np.random.default_rng(6)
    host = int8_cache.Host(rng, [40], 2, 64, 8)
    cache, _ = host.build(gpu)
    both = cache.batch(np.repeat(host.tables, 2, 0), [40, 33], appended=[0, 0])
    k, v = both.read()
    x = k.cpu().reshape(73, 2, 64)
    assert np.array_equal(x[:33], x[40:])
    other = gpu.KVCache(20, 16, 2, 64, dtype="f32")
    copy = other.batch(np.arange(6).reshape(2, 3), [40, 33], appended=[40, 33])
    copy.append(k, v)
    again = copy.read()
    assert np.array_equal(again[0].cpu(), k.cpu()) and np.array_equal(again[1].cpu(), v.cpu())


CASES = [
    # lengths, kv heads, query heads per kv head, head size, page
    ([1], 1, 1, 16, 8),
    ([17], 2, 4, 64, 16),
    ([64, 63, 65, 1], 2, 3, 128, 64),
    ([0, 130, 0], 1, 8, 96, 8),
    ([0, 0], 2, 2, 64, 8),
    ([300, 5, 129], 3, 5, 80, 128),
    ([257], 1, 12, 48, 256),
    ([200, 90], 2, 17, 64, 16),
    ([200, 90], 1, 40, 32, 16),
    ([513, 70], 2, 2, 256, 64),
    ([4099], 1, 1, 64, 16),
    ([9001, 3], 2, 6, 128, 128),
    ([20000], 1, 9, 112, 64),
    ([7] * 300, 1, 2, 16, 8),
    ([1000, 70], 1, 12, 256, 16),
    ([700, 500], 2, 16, 128, 64),
    ([385, 384, 0], 1, 1, 128, 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,heads,group,dim,page", CASES)
def test_attention_against_the_definition(gpu, lengths, heads, group, dim, page):
    rng = np.random.default_rng(sum(lengths) + dim)
    host = int8_cache.Host(rng, lengths, heads, dim, page)
    for x in host.v:  # rows of different size
        x *= rng.uniform(0.1, 3, x.shape[:2])[..., None].astype(np.float32)
    _, batch = host.build(gpu)
    q = rng.normal(0, 2, (len(lengths), heads * group, dim)).astype(np.float32)
    t = gpu.tensor(list(q.shape), q)
    out, tol, new, new_tol = host.attend(q, dim**-0.5)
    got = gpu.paged_attention(t, batch).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()
    again, weights = gpu.paged_attention_scored(t, batch)
    assert np.array_equal(again.cpu().reshape(q.shape), got)
    assert (np.abs(weights.cpu().reshape(new.shape) - new) <= new_tol).all()
    scores = rng.uniform(0, 3, (len(lengths), heads, max(lengths) // 2)).astype(np.float32)
    _, _, new, new_tol = host.attend(q, 0.3, scores)
    _, weights = gpu.paged_attention_scored(t, batch, gpu.tensor(list(scores.shape), scores), scale=0.3)
    assert (np.abs(weights.cpu().reshape(new.shape) - new) <= new_tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("length", [70, 700, 9001])
def test_rows_and_queries_of_very_different_size(gpu, length):
    # Values' scales over 2^80, a value that outweighs its tile, logits of
    # thousands, heads of tiny, huge and lopsided queries, rows of zeros.
    rng = np.random.default_rng(length)
    host = int8_cache.Host(rng, [length, 64, 65], 2, 64, 32)
    for s in range(3):
        host.v[s] *= np.exp2(rng.uniform(-40, 40, host.v[s].shape[:2]))[..., None].astype(np.float32)
        host.k[s][1] *= 60
        host.k[s][2] = 0
        host.v[s][3] = 0
    host.v[1][:] = 0
    q = rng.normal(0, 1, (3, 12, 64)).astype(np.float32)
    q[:, 0] *= np.float32(2.0**-50)
    q[:, 1] = 0
    q[:, 2, 7] *= 2000
    q[:, 3] *= 30
    q[:, 4] = np.float32(2.0**-110)
    q[:, 5, 0] = np.nextafter(np.float32(2), np.float32(0))
    _, batch = host.build(gpu)
    t = gpu.tensor(list(q.shape), q)
    out, tol, new, new_tol = host.attend(q, 0.125)
    got, weights = gpu.paged_attention_scored(t, batch)
    got = got.cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all() and not got[1].any()
    assert (np.abs(weights.cpu().reshape(new.shape) - new) <= new_tol).all()


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_row(gpu):
    rng = np.random.default_rng(2)
    host = int8_cache.Host(rng, [100, 90, 65], 2, 64, 16)
    q = rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    _, batch = host.build(gpu)
    want = gpu.paged_attention(gpu.tensor([3, 4, 64], q), batch).cpu().reshape(q.shape)
    host.v[1][89, 0, 5] = np.nan  # the whole row is one that is not finite
    host.k[2][64, 1, 0] = np.inf
    bad = np.zeros(q.shape, bool)
    bad[1, :2] = bad[2, 2:] = True
    q2 = q.copy()
    q2[0, 3, 60] = np.nan
    q2[1, 3, 0] = np.inf
    bad[0, 3] = bad[1, 3] = True
    _, batch = host.build(gpu)
    got = gpu.paged_attention(gpu.tensor([3, 4, 64], q2), batch).cpu().reshape(q.shape)
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], want[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("length,below", [(100, 64), (9001, 8000)])
def test_logits_below_the_range_of_float32_weigh_nothing(gpu, length, below):
    rng = np.random.default_rng(length)
    host = int8_cache.Host(rng, [length], 2, 64, 32)
    host.k[0][:, :, 0] = 0
    host.k[0][:below] = 0
    host.k[0][:below, :, 0] = -(2.0**84)
    q = rng.normal(0, 1, (1, 6, 64)).astype(np.float32)
    q[:, :, 0] = 2.0**50
    q[:, :, 1:] *= np.float32(2.0**45)
    _, batch = host.build(gpu)
    host.k[0], host.v[0], host.lengths = host.k[0][below:], host.v[0][below:], [length - below]
    scale = 2.0**-47
    out, tol, _, _ = host.attend(q, scale)
    got = gpu.paged_attention(gpu.tensor([1, 6, 64], q), batch, scale=scale).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,budget", [([30, 9, 200], 24), ([700, 650], 600), ([5000], 300)])
def test_eviction_moves_codes_and_scales(gpu, lengths, budget):
    rng = np.random.default_rng(budget)
    heads, dim, page = 2, 48, 16
    host = int8_cache.Host(rng, lengths, heads, dim, page)
    cache, batch = host.build(gpu)
    scores = rng.uniform(0, 1, (len(lengths), heads, max(lengths))).astype(np.float32)
    before = pools(cache)
    gpu.cache_evict(batch, gpu.tensor(list(scores.shape), scores), budget=budget, recent=5, sinks=2)
    source, _, _ = paged.evict(lengths, [n - 1 for n in lengths], scores, None, budget, 5, 2)
    for old, new in zip(before, pools(cache)):
        for part in range(2):
            for s, length in enumerate(lengths):
                was, now = (rows_of(x[part], host.tables[s], length, page) for x in (old, new))
                for h in range(heads):
                    kept = source[s, h][: min(length, budget)]
                    assert np.array_equal(now[: len(kept), h], was[kept, h])


@pytest.mark.gpu
def test_a_step_from_writing_to_eviction_on_two_layers(gpu):
    rng = np.random.default_rng(9)
    lengths, heads, dim = [100, 37], 2, 64
    host = int8_cache.Host(rng, lengths, heads, dim, 16)
    cache, batch = host.build(gpu)
    other = gpu.KVCache(host.pages, 16, heads, dim, dtype="int8")
    on = batch.on(other)
    on.append(gpu.tensor([137, heads, dim], np.concatenate(host.v)), gpu.tensor([137, heads, dim], np.concatenate(host.k)))
    q = rng.normal(0, 1, (2, 4, dim)).astype(np.float32)
    t = gpu.tensor([2, 4, dim], q)
    got = gpu.paged_attention(t, batch).cpu().reshape(q.shape)
    out, tol, _, _ = host.attend(q, dim**-0.5)
    assert (np.abs(got - out) <= tol).all()
    host.k, host.v = host.v, host.k
    out, tol, new, new_tol = host.attend(q, dim**-0.5)
    got, weights = gpu.paged_attention_scored(t, on)
    assert (np.abs(got.cpu().reshape(q.shape) - out) <= tol).all()
    assert (np.abs(weights.cpu().reshape(new.shape) - new) <= new_tol).all()
    kept, _ = gpu.cache_evict(on, weights, budget=30, recent=4)
    source, _, _ = paged.evict(lengths, [99, 36], weights.cpu().reshape(new.shape), None, 30, 4, 0)
    at = np.arange(heads)
    host.k = [x[source[s].T, at] for s, x in enumerate(host.k)]
    host.v = [x[source[s].T, at] for s, x in enumerate(host.v)]
    host.lengths = [30, 30]
    out, tol, _, _ = host.attend(q, dim**-0.5)
    got = gpu.paged_attention(t, other.batch(host.tables, [30, 30])).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
def test_writing_and_reading_from_two_threads(gpu):
    import threading

    n, heads, dim = 3000, 2, 64
    rng = np.random.default_rng(6)
    host = int8_cache.Host(rng, [n], heads, dim, 32)
    cache = gpu.KVCache(host.pages, 32, heads, dim, dtype="int8")
    write = cache.batch(host.tables, [n], appended=[n])
    read = cache.batch(host.tables, [n], appended=[0])
    values = [gpu.tensor([n, heads, dim], np.full(n * heads * dim, 2.0**f, np.float32)) for f in range(8)]
    write.append(values[0], values[0])
    failed, got = [], []

    def writer():
        try:
            for _ in range(10):
                for v in values:
                    write.append(v, v)
            gpu.synchronize()
        except Exception as e:  # a thread's exception would be lost
            failed.append(e)

    th = threading.Thread(target=writer)
    th.start()
    while th.is_alive() or len(got) < 20:
        got.append(read.read()[1])
        if len(got) % 10 == 0:
            gpu.synchronize()
    th.join()
    assert not failed
    for x in got[:60]:
        x = x.cpu()  # one write's, each value within a rounding of code 127 times its scale
        assert (np.abs(x / 2.0 ** np.round(np.log2(x.flat[0])) - 1) <= 2.0**-22).all()


def test_refusals_that_need_no_device(api):
    for dim in (8, 24, 136):
        with pytest.raises(api.InvalidArgument, match="multiple of 16 in int8"):
            api.KVCache(4, 16, 2, dim, dtype="int8")
    with pytest.raises(api.InvalidArgument, match="dtype"):
        api.KVCache(4, 16, 2, 64, dtype="int4")
    from ctypes import byref, c_int64, c_uint64, c_void_p

    from porch_b200._lib import lib

    a, b = c_int64(), c_int64()
    assert lib().pb_kv_attention_shape(24, 3, 1, byref(a), byref(b)) == 1
    assert lib().pb_kv_attention_shape(128, 4, 1, byref(a), byref(b)) == 1
    assert lib().pb_kv_attention_shape(128, 3, 1, byref(a), byref(b)) == 0
    k = c_uint64()
    assert lib().pb_kv_cache_scales(None, byref(k), byref(k)) == 1
    t = c_void_p()
    assert lib().pb_kv_read(None, byref(t), byref(t)) == 1


@pytest.mark.parametrize("dim", range(16, 257, 16))
@pytest.mark.parametrize("group", [1, 9])
def test_what_the_attention_takes_of_an_sm(api, dim, group):
    from ctypes import byref, c_int64

    from porch_b200._lib import lib

    ctas, shared = c_int64(), c_int64()
    assert lib().pb_kv_attention_shape(dim, 3, group, byref(ctas), byref(shared)) == 0
    assert ctas.value >= 1 and ctas.value * shared.value <= 228 * 1024 and shared.value <= 228 * 1024


@pytest.mark.gpu
def test_refusals(gpu):
    cache = gpu.KVCache(4, 16, 2, 64, dtype="int8")
    batch = cache.batch([[0, 1]], [20])
    with pytest.raises(gpu.InvalidArgument, match="k and v must be"):
        batch.append(gpu.zeros([1, 2, 32]), gpu.zeros([1, 2, 32]))
    with pytest.raises(gpu.InvalidArgument, match="another shape, type or device"):
        batch.on(gpu.KVCache(4, 16, 2, 64, dtype="bf16"))
    with pytest.raises(gpu.InvalidArgument, match="only an int8 cache has scales"):
        gpu.KVCache(4, 16, 2, 64, dtype="bf16").scales()
    with pytest.raises(RuntimeError, match="placeholder"):
        batch.append(gpu.placeholder([1, 2, 64]), gpu.zeros([1, 2, 64]))


@pytest.mark.gpu
def test_pools_past_two_to_the_32_bytes(gpu):
    # 2^24 + 2^20 rows of 256 codes: the last pages lie past 2^32 bytes, and the
    # scales behind them.
    pages, page, dim = ((1 << 24) + (1 << 20)) // 64, 64, 256
    cache = gpu.KVCache(pages, page, 1, dim, dtype="int8")
    rng = np.random.default_rng(2)
    host = int8_cache.Host(rng, [150], 1, dim, page)
    host.tables = np.array([[pages - 1, 3, pages - 2]], dtype=np.int32)
    batch = cache.batch(host.tables, [150], appended=[150])
    batch.append(gpu.tensor([150, 1, dim], host.k[0]), gpu.tensor([150, 1, dim], host.v[0]))
    for got, x in zip(batch.read(), (host.k[0], host.v[0])):
        codes, scale = int8_cache.quantise(x)
        assert np.array_equal(got.cpu().reshape(x.shape), codes.astype(np.float32) * scale[..., None])
    q = rng.normal(0, 0.2, (1, 3, dim)).astype(np.float32)
    out, tol, _, _ = host.attend(q, 1.0)
    got = gpu.paged_attention(gpu.tensor([1, 3, dim], q), batch, scale=1.0).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()
    scores = rng.uniform(0, 1, (1, 1, 150)).astype(np.float32)
    gpu.cache_evict(batch, gpu.tensor([1, 1, 150], scores), budget=70, recent=9)
    source, _, _ = paged.evict([150], [149], scores, None, 70, 9, 0)
    k, _ = cache.batch(host.tables, [70], appended=[0]).read()
    codes, scale = int8_cache.quantise(host.k[0][source[0, 0]])
    assert np.array_equal(k.cpu().reshape(70, 1, dim), codes.astype(np.float32) * scale[..., None])
