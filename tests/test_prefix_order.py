"""What a call over a shared prefix enqueues: both launches behind all that came
before the call, beside each other, and the join and all that follows behind both.
Over a stand-in for the driver, whose log tells; needs no GPU."""

import pytest

import fake_driver

SETUP = """
from porch_b200._lib import lib
assert lib().pb_test_share_prefix(1) == 0
rng = np.random.default_rng(1)
n, shared = 20, 256
cache = api.KVCache(64, 64, 2, 64, "{dtype}")
tables = np.concatenate([np.tile(np.arange(4), (n, 1)), 4 + np.arange(2 * n).reshape(n, 2)], 1)
lengths = [shared + 1 + s * 4 for s in range(n)]
batch = cache.batch(tables, lengths, prefix=[shared] * n)
x = api.tensor([n, 4, 64], rng.normal(0, 1, n * 256).astype(np.float32))
k = api.tensor([n, 2, 64], rng.normal(0, 1, n * 128).astype(np.float32))
one, turn, at = api.full([64], 1.0), api.zeros([4, 32]), api.zeros([n])
def step():
    q, y = api.qk_norm_rope(x, k, one, one, turn, turn, at)
    batch.append(y, k)
    out = api.paged_attention(q, batch)
    return api.qk_norm_rope(out, k, one, one, turn, turn, at)
"""

READ = {"pb_prefix_attention", "pb_paged_attention"}


def conflict(a, b):
    """Whether one reads what the other writes: queries, cache, parts, results."""
    return (b in READ and a not in READ) or (a in READ and b not in READ) or (a == "pb_shared_finish") != (b == "pb_shared_finish")


@pytest.mark.parametrize("dtype", ["bf16", "f32", "int8"])
def test_steps_one_after_the_other(api, tmp_path, dtype):
    _, log = fake_driver.run(SETUP.format(dtype=dtype) + "kept = [step() for _ in range(3)]\n", tmp_path)
    launched = [line[3] for line in log if line[1] == "launch"]
    assert launched.count("pb_shared_finish") == 3 and launched.count("pb_paged_attention") == 3
    assert launched.count("pb_prefix_attention") == (3 if dtype == "bf16" else 0)
    assert fake_driver.unordered(log, conflict) == []
    # Of one call the two are beside each other, and of different calls they are not.
    beside = fake_driver.unordered(log, lambda a, b: a in READ and b in READ)
    assert beside == ([("pb_prefix_attention", "pb_paged_attention")] * 3 if dtype == "bf16" else [])


@pytest.mark.parametrize("slow", [None, "cuEventRecord", "pb_prefix_attention"])
def test_steps_of_two_threads(api, tmp_path, slow):
    # A cache's writes and reads are in the order of their launches, whoever makes them.
    program = SETUP.format(dtype="bf16") + """
kept = []
def work():
    q = api.tensor([n, 4, 64], np.ones(n * 256, np.float32))
    v = api.tensor([n, 2, 64], np.ones(n * 128, np.float32))
    for _ in range(2):
        kept.append(api.paged_attention(q, batch))
        batch.append(v, v)
threads = [threading.Thread(target=work) for _ in range(2)]
for t in threads:
    t.start()
for t in threads:
    t.join()
"""
    _, log = fake_driver.run(program, tmp_path, slow=slow)
    assert [line[3] for line in log if line[1] == "launch"].count("pb_prefix_attention") == 4
    assert fake_driver.unordered(log, lambda a, b: {a, b} & READ and "pb_cache_append" in (a, b)) == []
