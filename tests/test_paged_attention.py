"""Attention over a paged cache against its definition in 64 bits (the
tolerances are derived in paged.Host.attend). Every slot that no sequence uses
holds NaN throughout."""

import numpy as np
import pytest

import paged

CASES = [
    # lengths, kv heads, query heads per kv head, head size, page, type
    ([1], 1, 1, 8, 8, "f32"),
    ([1], 1, 1, 8, 8, "bf16"),
    ([17], 2, 4, 64, 16, "bf16"),
    ([64, 63, 65, 1], 2, 3, 128, 64, "bf16"),
    ([64, 63, 65, 1], 2, 3, 128, 64, "f32"),
    ([0, 130, 0], 1, 8, 96, 8, "bf16"),
    ([0, 0], 2, 2, 64, 8, "bf16"),
    ([300, 5, 129], 3, 5, 80, 128, "bf16"),
    ([300, 5, 129], 3, 5, 80, 128, "f32"),
    ([257], 1, 12, 40, 256, "bf16"),
    ([257, 100], 1, 16, 72, 32, "f32"),
    ([200, 90], 2, 17, 64, 16, "bf16"),
    ([200, 90], 1, 40, 32, 16, "f32"),
    ([513, 70], 2, 2, 256, 64, "bf16"),
    ([513, 70], 2, 2, 256, 64, "f32"),
    ([4099], 1, 1, 64, 16, "f32"),
    ([9001, 3], 2, 6, 128, 128, "bf16"),
    ([20000], 1, 9, 112, 64, "bf16"),
    ([7] * 300, 1, 2, 24, 8, "bf16"),
    ([1000, 70], 1, 12, 256, 16, "f32"),
    ([700, 500], 2, 16, 128, 64, "bf16"),
    ([700, 3], 1, 10, 256, 32, "bf16"),
    ([385, 384, 0], 1, 1, 128, 8, "bf16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,heads,group,dim,page,dtype", CASES)
def test_against_the_definition(gpu, lengths, heads, group, dim, page, dtype):
    rng = np.random.default_rng(sum(lengths) + dim)
    host = paged.Host(rng, lengths, heads, dim, page, dtype)
    _, batch = host.build(gpu)
    q = rng.normal(0, 2, (len(lengths), heads * group, dim)).astype(np.float32)
    t = gpu.tensor(list(q.shape), q)
    out, tol, new, new_tol = host.attend(q, dim**-0.5)
    got = gpu.paged_attention(t, batch).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()
    again, weights = gpu.paged_attention_scored(t, batch)
    assert np.array_equal(again.cpu().reshape(q.shape), got)
    assert (np.abs(weights.cpu().reshape(new.shape) - new) <= new_tol).all()
    # Running scores, of fewer slots than there are now, and of more.
    for slots in (max(lengths) // 2, max(lengths) + 9):
        scores = rng.uniform(0, 3, (len(lengths), heads, slots)).astype(np.float32)
        _, _, new, new_tol = host.attend(q, 0.3, scores)
        _, weights = gpu.paged_attention_scored(t, batch, gpu.tensor(list(scores.shape), scores), scale=0.3)
        assert weights.shape() == list(new.shape)
        assert (np.abs(weights.cpu().reshape(new.shape) - new) <= new_tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logits_far_apart(gpu, dtype):
    # One slot with nearly all the weight, wherever it stands; logits of
    # thousands; and equal logits, whose weights are 1 / n.
    rng = np.random.default_rng(2)
    host = paged.Host(rng, [700, 129, 64], 1, 64, 32, dtype)
    for s, at in enumerate([0, 128, 40]):
        host.k[s][at] *= 60
    _, batch = host.build(gpu)
    q = np.concatenate([5 * paged.bf16(host.k[s][at])[None] for s, at in enumerate([0, 128, 40])])
    q = np.concatenate([q, -q, 0 * q], 1)
    out, tol, new, new_tol = host.attend(q, 1.0)
    got, weights = gpu.paged_attention_scored(gpu.tensor(list(q.shape), q), batch, scale=1.0)
    assert (np.abs(got.cpu().reshape(q.shape) - out) <= tol).all()
    assert (np.abs(weights.cpu().reshape(new.shape) - new) <= new_tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("length,below", [(100, 64), (200, 130), (9001, 8000), (9001, 9000), (70000, 60001)])
def test_logits_below_the_range_of_float32_weigh_nothing(gpu, dtype, length, below):
    # The first `below` slots' logits are -2^134 x scale, past float32's range:
    # whole tiles, and whole parts of a row, with a maximum of -inf. What is left
    # is the attention of the other slots.
    rng = np.random.default_rng(length)
    host = paged.Host(rng, [length], 2, 64, 32, dtype)
    host.k[0][:, :, 0] = 0
    host.k[0][:below, :, 0] = -(2.0**84)
    _, batch = host.build(gpu)
    q = rng.normal(0, 1, (1, 6, 64)).astype(np.float32)
    q[:, :, 0] = 2.0**50
    t = gpu.tensor([1, 6, 64], q)
    host.k[0], host.v[0], host.lengths = host.k[0][below:], host.v[0][below:], [length - below]
    out, tol, new, new_tol = host.attend(np.where(np.arange(64) == 0, 0, q).astype(np.float32), 0.125)
    assert (np.abs(gpu.paged_attention(t, batch, scale=0.125).cpu().reshape(q.shape) - out) <= tol).all()
    got, weights = gpu.paged_attention_scored(t, batch, scale=0.125)
    assert (np.abs(got.cpu().reshape(q.shape) - out) <= tol).all()
    w = weights.cpu().reshape(1, 2, length)
    assert not w[:, :, :below].any() and (np.abs(w[:, :, below:] - new) <= new_tol).all()


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_row(gpu):
    rng = np.random.default_rng(2)
    host = paged.Host(rng, [100, 90, 65], 2, 64, 16, "bf16")
    q = rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    _, batch = host.build(gpu)
    want = gpu.paged_attention(gpu.tensor([3, 4, 64], q), batch).cpu().reshape(q.shape)
    host.v[1][89, 0, 5] = np.nan
    host.k[2][64, 1, 0] = np.nan
    _, batch = host.build(gpu)
    got = gpu.paged_attention(gpu.tensor([3, 4, 64], q), batch).cpu().reshape(q.shape)
    bad = np.zeros(q.shape, bool)
    bad[1, :2, 5] = True
    bad[2, 2:] = True
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], want[~bad])


@pytest.mark.gpu
def test_pools_past_two_to_the_31_values(gpu):
    # 2^24 + 2^20 rows of 128 values: the last pages lie past 2^31 values and
    # past 2^32 bytes.
    pages, page, dim = ((1 << 24) + (1 << 20)) // 64, 64, 128
    cache = gpu.KVCache(pages, page, 1, dim, dtype="bf16")
    rng = np.random.default_rng(2)
    host = paged.Host(rng, [150], 1, dim, page, "bf16")
    host.tables = np.array([[pages - 1, 3, pages - 2]], dtype=np.int32)
    batch = cache.batch(host.tables, [150], appended=[150])
    batch.append(gpu.tensor([150, 1, dim], host.k[0]), gpu.tensor([150, 1, dim], host.v[0]))
    q = rng.normal(0, 1, (1, 3, dim)).astype(np.float32)
    out, tol, _, _ = host.attend(q, 1.0)
    got = gpu.paged_attention(gpu.tensor([1, 3, dim], q), batch, scale=1.0).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()
    scores = gpu.tensor([1, 1, 150], rng.uniform(0, 1, 150).astype(np.float32))
    kept, _ = gpu.cache_evict(batch, scores, budget=70, recent=9)
    source, _, _ = paged.evict([150], [149], scores.cpu().reshape(1, 1, 150), None, 70, 9, 0)
    host.k[0], host.v[0], host.lengths = host.k[0][source[0, 0]], host.v[0][source[0, 0]], [70]
    out, tol, _, _ = host.attend(q, 1.0)
    got = gpu.paged_attention(gpu.tensor([1, 3, dim], q), cache.batch(host.tables, [70]), scale=1.0)
    assert (np.abs(got.cpu().reshape(q.shape) - out) <= tol).all()


@pytest.mark.gpu
def test_queries_read_in_place_and_pages_shared_by_sequences(gpu):
    rng = np.random.default_rng(6)
    host = paged.Host(rng, [40, 40], 2, 64, 8, "f32")
    host.tables[1] = host.tables[0]
    host.k[1], host.v[1] = host.k[0], host.v[0]
    cache = gpu.KVCache(host.pages, 8, 2, 64)
    one = cache.batch(host.tables[:1], [40], appended=[40])
    one.append(gpu.tensor([40, 2, 64], host.k[0]), gpu.tensor([40, 2, 64], host.v[0]))
    both = cache.batch(host.tables, [40, 40], appended=[0, 0])
    fused = rng.normal(0, 1, (2, 10, 65)).astype(np.float32)
    q = gpu.materialize(gpu.tensor([2, 10, 65], fused)[gpu.all, 3:7, 1:65])
    out, tol, _, _ = host.attend(fused[:, 3:7, 1:], 0.125)
    assert (np.abs(gpu.paged_attention(q, both).cpu().reshape(out.shape) - out) <= tol).all()
    # Another layer's cache, the same tables: other values.
    other = gpu.KVCache(host.pages, 8, 2, 64)
    one.on(other).append(gpu.tensor([40, 2, 64], host.v[0]), gpu.tensor([40, 2, 64], host.k[0]))
    assert (np.abs(gpu.paged_attention(q, both).cpu().reshape(out.shape) - out) <= tol).all()
    host.k, host.v = host.v, host.k
    out, tol, _, _ = host.attend(fused[:, 3:7, 1:], 0.125)
    assert (np.abs(gpu.paged_attention(q, both.on(other)).cpu().reshape(out.shape) - out) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("first", [0, 1, 4])
def test_new_tokens_read_in_place(gpu, dtype, first):
    # Keys and values as heads of a fused projection, at aligned and odd channels.
    rng = np.random.default_rng(first)
    host = paged.Host(rng, [9, 20, 4], 2, 24, 8, dtype)
    fused = rng.normal(0, 1, (33, 6, 28)).astype(np.float32)
    ends = np.cumsum([0, 9, 20, 4])
    for s in range(3):
        host.k[s] = fused[ends[s] : ends[s + 1], 1:3, first : first + 24]
        host.v[s] = fused[ends[s] : ends[s + 1], 4:6, first : first + 24]
    cache = gpu.KVCache(host.pages, 8, 2, 24, dtype=dtype)
    f = gpu.tensor([33, 6, 28], fused)
    k, v = (gpu.materialize(f[gpu.all, h : h + 2, first : first + 24]) for h in (1, 4))
    batch = cache.batch(host.tables, [9, 20, 4], appended=[9, 20, 4])
    batch.append(k, v)
    q = rng.normal(0, 1, (3, 4, 24)).astype(np.float32)
    out, tol, _, _ = host.attend(q, 0.2)
    got = gpu.paged_attention(gpu.tensor([3, 4, 24], q), batch, scale=0.2).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
def test_a_cache_written_by_one_thread_and_read_by_another(gpu):
    import threading

    rng = np.random.default_rng(6)
    host = paged.Host(rng, [3000], 2, 64, 32, "f32")
    cache = gpu.KVCache(host.pages, 32, 2, 64)
    q = rng.normal(0, 1, (1, 4, 64)).astype(np.float32)
    t = gpu.tensor([1, 4, 64], q)
    batch = cache.batch(host.tables, [3000], appended=[3000])
    read = cache.batch(host.tables, [3000], appended=[0])
    rows = [(gpu.tensor([3000, 2, 64], host.k[0] * f), gpu.tensor([3000, 2, 64], host.v[0] * f)) for f in (1, 0.5, 2)]
    for f, (k, v) in zip((1, 0.5, 2), rows):  # each write waits for the reads before it
        th = threading.Thread(target=lambda: batch.append(gpu.materialize(k * 1.0), gpu.materialize(v * 1.0)))
        th.start()
        th.join()
        got = gpu.paged_attention(t, read)
        copy = paged.Host(np.random.default_rng(6), [3000], 2, 64, 32, "f32")
        copy.k[0], copy.v[0] = copy.k[0] * np.float32(f), copy.v[0] * np.float32(f)
        out, tol, _, _ = copy.attend(q, 0.125)
        assert (np.abs(got.cpu().reshape(q.shape) - out) <= tol).all()


@pytest.mark.gpu
def test_a_read_beside_writes_of_another_thread_sees_one_of_them(gpu):
    # All values of a write are one power of two, so the attention is that
    # number, within the weighted sum's (2 n + 128) u; of two writes at once it
    # would be something between.
    import threading

    n, heads, dim = 6000, 4, 64
    rng = np.random.default_rng(6)
    host = paged.Host(rng, [n], heads, dim, 32, "f32")
    cache = gpu.KVCache(host.pages, 32, heads, dim)
    write = cache.batch(host.tables, [n], appended=[n])
    read = cache.batch(host.tables, [n], appended=[0])
    k = gpu.tensor([n, heads, dim], host.k[0])
    values = [gpu.tensor([n, heads, dim], np.full(n * heads * dim, 2.0**f, np.float32)) for f in range(12)]
    write.append(k, values[0])
    q = gpu.tensor([1, 2 * heads, dim], rng.normal(0, 1, (1, 2 * heads, dim)).astype(np.float32))
    failed = []

    def writer():
        try:
            for _ in range(20):
                for v in values:
                    write.append(k, v)
            gpu.synchronize()
        except Exception as e:  # a thread's exception would be lost
            failed.append(e)

    th = threading.Thread(target=writer)
    th.start()
    got = []
    while th.is_alive() or len(got) < 50:
        got.append(gpu.paged_attention(q, read))
        if len(got) % 20 == 0:
            gpu.synchronize()
    th.join()
    assert not failed
    for out in got:
        x = out.cpu()
        seen = 2.0 ** np.round(np.log2(x[0]))
        assert (np.abs(x - seen) <= (2 * n + 128) * 2.0**-24 * seen).all()


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported_and_the_gpu_recovers(gpu):
    # Block 0's loads are never issued: its bounded waits give up (about two
    # seconds), the kernel records 0x7d00 + site and returns.
    from porch_b200._lib import lib

    rng = np.random.default_rng(6)
    host = paged.Host(rng, [500, 40], 2, 64, 32, "bf16")
    q = rng.normal(0, 1, (2, 4, 64)).astype(np.float32)
    _, batch = host.build(gpu)
    t = gpu.tensor([2, 4, 64], q)
    assert lib().pb_test_attention_stall(1) == 0
    try:
        with pytest.raises(RuntimeError, match="kernel error code 32003"):  # 0x7d00 + site 3
            gpu.paged_attention(t, batch).cpu()
    finally:
        assert lib().pb_test_attention_stall(0) == 0
    out, tol, _, _ = host.attend(q, 0.125)
    for _ in range(2):
        assert (np.abs(gpu.paged_attention(t, batch).cpu().reshape(q.shape) - out) <= tol).all()


def test_a_unit_is_handed_back_only_after_its_load_has_landed(api):
    # Both places where a computing warp hands a unit back to the producer: the
    # first stands before the barrier at which a wait that gave up makes all
    # warps leave, so it has a condition; the second stands behind that barrier.
    text = api.operator_sources()
    text = text[text.index("extern \"C\" __global__ void __launch_bounds__(160, PB_PER_SM) pb_paged_attention") :]
    text = text[: text.index("---- the row ends")]
    waits, leaves = "bad |= !pb_wait(full", "if (pb_bar_any(bad)) { bad = true; break; }"
    first, second = [i for i in range(len(text)) if text.startswith("pb_mbar_arrive(empty", i)]
    assert text.count(waits) == 2 and text[:first].endswith("if (lane == 0 && !bad) ")
    assert text.rindex(waits) < text.rindex(leaves) < second


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[40, 30], [70, 5], [5000, 40]])
def test_giving_up_while_loads_are_on_their_way(gpu, lengths):
    # Block 0's computing warps give up at their first tile. Where its row has
    # few tiles the producer has issued every load by then: it has to stay until
    # they have landed, since shared memory is the next block's after it.
    from porch_b200._lib import lib

    rng = np.random.default_rng(7)
    host = paged.Host(rng, lengths, 2, 64, 32, "bf16")
    q = rng.normal(0, 1, (2, 4, 64)).astype(np.float32)
    _, batch = host.build(gpu)
    t = gpu.tensor([2, 4, 64], q)
    assert lib().pb_test_attention_stall(2) == 0
    try:
        for _ in range(3):
            with pytest.raises(RuntimeError, match="kernel error code 32005"):  # 0x7d00 + site 5
                gpu.paged_attention(t, batch).cpu()
    finally:
        assert lib().pb_test_attention_stall(0) == 0
    out, tol, _, _ = host.attend(q, 0.125)
    for _ in range(2):
        assert (np.abs(gpu.paged_attention(t, batch).cpu().reshape(q.shape) - out) <= tol).all()


def test_the_producer_waits_for_its_loads_whoever_gave_up(api):
    # Its last waits stand under no condition but the lane's.
    text = api.operator_sources()
    at = text.index("Nothing may land after this CTA is gone")
    assert "if (lane == 0) {" in text[at : at + 400] and "bad" not in text[at : text.index("pb_mbar_try", at)]


@pytest.mark.gpu
def test_the_same_every_time_and_from_another_thread(gpu):
    import threading

    rng = np.random.default_rng(6)
    host = paged.Host(rng, [3000, 40, 777], 2, 64, 32, "bf16")
    q = rng.normal(0, 1, (3, 8, 64)).astype(np.float32)
    cache, batch = host.build(gpu)
    t = gpu.tensor([3, 8, 64], q)
    first = [x.cpu() for x in gpu.paged_attention_scored(t, batch)]
    got = []

    def work():
        for _ in range(3):
            got.append([x.cpu() for x in gpu.paged_attention_scored(t, batch)])

    th = threading.Thread(target=work)
    th.start()
    work()
    th.join()
    assert len(got) == 6 and all(np.array_equal(a, b) for g in got for a, b in zip(first, g))


def test_refusals_that_need_no_device(api):
    for bad in ((0, 16, 1, 64), (4, 12, 1, 64), (4, 4, 1, 64), (4, 512, 1, 64), (4, 16, 0, 64), (4, 16, 1, 60),
                (4, 16, 1, 264), (4, 16, 1, 0), (1 << 25, 256, 1, 64)):
        with pytest.raises(api.InvalidArgument, match="cache"):
            api.KVCache(*bad)
    with pytest.raises(api.InvalidArgument, match="dtype"):
        api.KVCache(4, 16, 1, 64, dtype="f16")


def test_the_ctas_that_a_plan_counts_on_fit_an_sm(api):
    # An SM has 228 KB of shared memory for its CTAs; of one's, 1 KB is the
    # system's and at most 227 KB the kernel's. A group of 1, and of 9, which
    # may take the wider form.
    from ctypes import byref, c_int64

    from porch_b200._lib import lib

    for dim in range(8, 257, 8):
        for kind in (0, 1):
            for group in (1, 9):
                ctas, shared = c_int64(), c_int64()
                assert lib().pb_kv_attention_shape(dim, kind, group, byref(ctas), byref(shared)) == 0
                assert ctas.value >= 1 and ctas.value * shared.value <= 228 * 1024, (dim, kind, group)
    for bad in ((0, 0, 1), (12, 0, 1), (264, 0, 1), (64, 2, 1), (64, 0, 0)):
        assert lib().pb_kv_attention_shape(*bad, byref(ctas), byref(shared)) != 0


@pytest.mark.parametrize("seed", range(40))
def test_every_tile_is_worked_on_once_and_every_split_row_joined(api, seed):
    # Walks the CTAs as the kernel does.
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 30))
    lengths = [int(x) if rng.random() > 0.2 else 0 for x in np.exp(rng.uniform(0, 9, n))]
    heads, chunks, ctas = int(rng.integers(1, 6)), int(rng.integers(1, 4)), int(rng.integers(1, 600))
    if seed == 0:
        lengths = [0] * n
    if seed > 30:
        lengths = [x % 513 for x in lengths]
    tiles = np.repeat([-(-x // 64) for x in lengths], heads * chunks)
    work, join = [], {}
    for line in api.attention_plan(lengths, heads, ctas, chunks).splitlines():
        kind, *v = line.split()
        if kind == "work":
            work.append([int(x) for x in v])
        else:
            row, *rest = (int(x) for x in v)
            assert row not in join
            join[row] = rest
    # Rows without slots have a CTA each, at the end.
    clear = [w[0] for w in work if w[2] == 0]
    assert clear == list(np.flatnonzero(tiles == 0)) and [w[2] for w in work[len(work) - len(clear):]] == [0] * len(clear)
    work = work[: len(work) - len(clear)]
    if tiles.max() <= 8 and (tiles > 0).sum() <= ctas:  # short rows: a CTA each
        assert not join and [w[2] for w in work] == list(tiles[tiles > 0])
    else:
        # Tiles and rows begun: as even as whole tiles let them be.
        assert len(work) <= min(ctas, tiles.sum())
        even = -(-(tiles.sum() + (tiles > 0).sum()) // max(1, min(ctas, tiles.sum())))
        assert all(w[2] <= even for w in work)
    seen, parts = np.zeros(tiles.sum(), int), {}
    first = np.concatenate([[0], np.cumsum(tiles)])
    for c, (row, tile, count) in enumerate(work):
        segment, at_zero = 0, tile == 0
        for i in range(count):
            assert tile < tiles[row]
            seen[first[row] + tile] += 1
            ends = tile + 1 == tiles[row]
            if ends or i + 1 == count:
                if not (at_zero and ends):
                    parts.setdefault(row, []).append((c, 1 if segment else 0))
                segment += 1
            if i + 1 < count:
                tile += 1
                if ends:
                    tile, at_zero = 0, True
                    row += 1
                    while tiles[row] == 0:
                        row += 1
    assert (seen == 1).all()
    assert parts == {r: [(c + i, 0 if i else place) for i in range(k)] for r, (c, k, place) in join.items()}


@pytest.mark.parametrize("lengths,heads,ctas,chunks", [
    ([2**63 - 1], 1, 8, 1), ([1 << 30], 1, 8, 1), ([-1], 1, 8, 1), ([64], 0, 8, 1), ([64], 1025, 8, 1), ([64], 1, 0, 1),
    ([64], 1, 1 << 40, 1), ([64], 1, 8, 0), ([64], 1, 8, 1 << 50), ([1] * 200, 1024, 8, 1024), ([1] * 65536, 1, 8, 1),
])
def test_plans_of_sizes_that_no_batch_has_are_refused(api, lengths, heads, ctas, chunks):
    with pytest.raises(api.InvalidArgument, match="plan"):
        api.attention_plan(lengths, heads, ctas, chunks)


@pytest.mark.gpu
def test_refusals(gpu):
    cache = gpu.KVCache(6, 16, 2, 64)
    tables = np.array([[0, 1], [2, 3]], np.int32)
    batch = cache.batch(tables, [20, 32])

    def refused(error, match, call, *args, **more):
        with pytest.raises(error, match=match):
            call(*args, **more)

    bad = gpu.InvalidArgument
    refused(bad, "too short", cache.batch, tables, [20, 33])
    refused(bad, "length", cache.batch, tables, [20, -1])
    refused(gpu.OutOfRange, "page 6", cache.batch, [[0, 6]], [32])
    refused(gpu.OutOfRange, "page -1", cache.batch, [[0, -1]], [32])
    refused(gpu.OutOfRange, "page", cache.batch, [[0, 1 << 40]], [32])
    refused(bad, "new tokens", cache.batch, tables, [20, 32], appended=[21, 0])
    refused(bad, "newest", cache.batch, tables, [20, 32], newest=[19, 30])
    refused(bad, "newest", cache.batch, tables, [20, 32], newest=[19, 1 << 24])
    refused(bad, "same row", cache.batch, [[0, 1], [0, 1]], [20, 20])
    refused(bad, "one whole length", cache.batch, tables, [20])
    refused(bad, "one whole length", cache.batch, tables, [20.5, 32.0])
    refused(bad, "whole numbers", cache.batch, tables + 0.5, [20, 32])
    assert cache.batch([[]], [0]).lengths.tolist() == [0]
    refused(bad, "width", cache.batch, [0, 1], [20])
    refused(bad, "sequences", cache.batch, np.zeros((0, 2), np.int32), [])
    refused(bad, "shape, type or device", batch.on, gpu.KVCache(6, 16, 2, 64, dtype="bf16"))
    zeros = gpu.zeros
    refused(bad, "new tokens", batch.append, zeros([3, 2, 64]), zeros([2, 2, 64]))
    refused(bad, "new tokens", batch.append, zeros([2, 2, 64]), zeros([2, 2, 32]))
    refused(bad, "q must be", gpu.paged_attention, zeros([2, 4, 32]), batch)
    refused(bad, "q must be", gpu.paged_attention, zeros([1, 4, 64]), batch)
    refused(bad, "multiple", gpu.paged_attention, zeros([2, 3, 64]), batch)
    refused(bad, "multiple", gpu.paged_attention, zeros([2, 1, 64]), batch)
    refused(bad, "finite", gpu.paged_attention, zeros([2, 4, 64]), batch, scale=float("nan"))
    refused(bad, "scores must be", gpu.paged_attention_scored, zeros([2, 4, 64]), batch, zeros([2, 4, 32]))
    scores = zeros([2, 2, 32])
    refused(bad, "scores must be", gpu.cache_evict, batch, zeros([2, 32]), budget=8)
    refused(bad, "positions must be", gpu.cache_evict, batch, scores, zeros([1, 2, 8]), budget=8)
    refused(bad, "budget", gpu.cache_evict, batch, scores, budget=0)
    refused(bad, "recent and sinks", gpu.cache_evict, batch, scores, budget=8, recent=9)
    refused(bad, "recent and sinks", gpu.cache_evict, batch, scores, budget=8, recent=5, sinks=4)
    refused(bad, "recent and sinks", gpu.cache_evict, batch, scores, budget=8, sinks=-1)
    shared = cache.batch([[0, 1], [0, 2]], [20, 20], appended=[0, 0])
    refused(bad, "more than one place", gpu.cache_evict, shared, scores, budget=8)
    with pytest.raises(RuntimeError, match="placeholder"):
        gpu.paged_attention(gpu.placeholder([2, 4, 64]), batch)
