"""Calls that write a cache and calls that read it, from two threads: what they
enqueue is ordered on the device in the order in which it was launched. Over a
stand-in for the driver, whose log tells; needs no GPU."""

import pytest

import fake_driver

SETUP = """
rng = np.random.default_rng(1)
cache = api.KVCache(64, 64, 2, 64, "bf16")
table = np.arange(64).reshape(1, 64)
# 4000 slots to 1000: more rows to move than the select takes along
batch = cache.batch(table, [4000], appended=[4000])
q = api.tensor([1, 4, 64], rng.normal(0, 1, 256).astype(np.float32))
k = api.tensor([4000, 2, 64], rng.normal(0, 1, 4000 * 128).astype(np.float32))
scores = api.tensor([1, 2, 4000], rng.uniform(0, 1, 8000).astype(np.float32))
calls = {
    "append": lambda: batch.append(k, k),
    "attend": lambda: api.paged_attention(q, batch),
    "score": lambda: api.paged_attention_scored(q, batch, scores),
    "evict": lambda: api.cache_evict(batch, scores, budget=1000),
}
kept = []
def wait_for(kernel):
    for _ in range(2000):
        if any(" begin " in line and line.split()[-1] == kernel for line in open(os.environ["FAKE_CUDA_LOG"])):
            return
        time.sleep(0.005)
    raise SystemExit("no launch of " + kernel)
"""

WRITES = {"pb_cache_append", "pb_evict_select", "pb_evict_move"}
TOUCHES = WRITES | {"pb_paged_attention"}


def conflict(a, b):
    return a in TOUCHES and b in TOUCHES and (a in WRITES or b in WRITES)


@pytest.mark.parametrize("first,slow,second", [
    ("attend", "pb_paged_attention", "append"),
    ("attend", "pb_paged_attention", "evict"),
    ("score", "pb_paged_attention", "evict"),
    ("append", "pb_cache_append", "attend"),
    ("append", "pb_cache_append", "evict"),
    ("evict", "pb_evict_select", "attend"),
    ("evict", "pb_evict_move", "attend"),
    ("evict", "pb_evict_move", "append"),
])
def test_a_call_that_comes_in_while_another_is_being_launched(api, tmp_path, first, slow, second):
    # The second thread's call begins while the first one's launch is under way.
    program = SETUP + f"""
other = threading.Thread(target=lambda: kept.append(calls["{first}"]()))
other.start()
wait_for("{slow}")
kept.append(calls["{second}"]())
other.join()
"""
    _, log = fake_driver.run(program, tmp_path, slow=slow)
    launched = [line[3] for line in log if line[1] == "launch"]
    assert slow in launched and len([n for n in launched if n in TOUCHES]) >= 2
    assert fake_driver.unordered(log, conflict) == []


def test_calls_of_threads_that_take_turns(api, tmp_path):
    program = SETUP + """
def turn(*names):
    t = threading.Thread(target=lambda: kept.append([calls[n]() for n in names]))
    t.start()
    t.join()
turn("append", "attend")
turn("score", "evict")
turn("attend")
calls["append"]()
turn("evict", "append")
calls["score"]()
"""
    _, log = fake_driver.run(program, tmp_path)
    assert fake_driver.unordered(log, conflict) == []
