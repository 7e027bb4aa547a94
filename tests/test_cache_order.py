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


def test_the_pools_interface_names_a_stream_behind_every_call(api, tmp_path):
    # A reader enqueues its work on the stream that a pool's interface names: a
    # launch of its own stands for it in the log. Asked from the thread that
    # called the operators, and from another one.
    program = SETUP + """
pools = cache.pools()
def faces():
    a, b = (p.__cuda_array_interface__ for p in pools)
    assert a["stream"] == b["stream"] == q.__cuda_array_interface__["stream"]
    k, v, _ = cache.device_data()
    assert (a["data"], b["data"]) == ((k, False), (v, False)) and a["typestr"] == "<u2"
    assert a["shape"] == (64, 2, 64, 64)
    return a["stream"]
for name in ("append", "evict"):
    kept.append(calls[name]())
    print(hex(faces()), flush=True)
seen = []
kept.append(calls["append"]())
q = api.tensor([1, 4, 64], np.zeros(256, np.float32))
t = threading.Thread(target=lambda: (api.zeros([1]).realize(), seen.append(pools[0].__cuda_array_interface__["stream"])))
t.start()
t.join()
print(hex(seen[0]))
"""
    out, log = fake_driver.run(program, tmp_path)
    here, again, other = out.split()
    assert here == again != other
    streams = {line[2] for line in log if line[1] == "launch" and line[3] in WRITES}
    assert streams == {here}
    log += [["0", "launch", stream, "reader", "1", "1", "0"] for stream in (here, other)]
    assert fake_driver.unordered(log, lambda a, b: a in WRITES and b == "reader") == []


def test_a_scale_that_overflows_in_units_of_log2_is_refused(api, tmp_path):
    out, log = fake_driver.run(SETUP + """
for scale in (float("nan"), float("inf"), 2.5e38, -3.4e38):
    for call in (api.paged_attention, api.paged_attention_scored):
        try:
            call(q, batch, scale=scale)
        except api.InvalidArgument as e:
            assert "scale" in str(e)
            print("refused")
api.paged_attention(q, batch, scale=-2.3e38)
""", tmp_path)
    assert out.split() == ["refused"] * 8
    assert [line[3] for line in log if line[1] == "launch"] == ["pb_paged_attention", "pb_paged_finish"]


def test_a_kernel_that_compiles_holds_up_only_those_who_need_it(api, tmp_path):
    # Head size 24 takes a second to compile. Two threads want it, and get it
    # with one compilation of each kernel; this one runs a kernel that is there.
    program = SETUP + """
calls["append"]()
other = api.KVCache(8, 8, 1, 24)
wide = other.batch([[0, 1]], [16], appended=[16])
x = api.tensor([16, 1, 24], np.ones(384, np.float32))
threads = [threading.Thread(target=lambda: wide.append(x, x)) for _ in range(2)]
for t in threads:
    t.start()
while not any(l.split()[1:] == ["compile", "1"] for l in open(os.environ["FAKE_CUDA_LOG"])):
    time.sleep(0.005)
began = time.perf_counter()
calls["append"]()
took = time.perf_counter() - began
assert any(t.is_alive() for t in threads)
for t in threads:
    t.join()
assert took < 0.3, took
"""
    _, log = fake_driver.run(program, tmp_path, slow_compile="#define PB_D 24")
    assert sum(line[1:] == ["compile", "1"] for line in log) == 1


@pytest.mark.parametrize("group,dim,dtype", [(1, 64, "bf16"), (12, 128, "f32"), (17, 64, "bf16"), (40, 64, "f32")])
def test_a_step_uploads_and_waits_only_where_its_batch_is_made(api, tmp_path, group, dim, dtype):
    # From the second step on an attention only enqueues, whatever the number of
    # query heads, over the batch's own cache and another layer's, and a batch
    # makes two uploads.
    program = f"""
caches = [api.KVCache(8, 64, 2, {dim}, "{dtype}") for _ in range(2)]
q = api.tensor([2, 2 * {group}, {dim}], np.ones(4 * {group} * {dim}, np.float32))
lines = lambda: [l.split()[1] for l in open(os.environ["FAKE_CUDA_LOG"])]
busy = lambda l: (l.count("copy"), l.count("sync"))
for step in range(3):
    a = len(lines())
    batch = caches[0].batch(np.arange(8).reshape(2, 4), [100 + step, 50])
    b = len(lines())
    for c in caches:
        api.paged_attention_scored(q, batch.on(c))
    log = lines()
    print(*busy(log[a:b]), *busy(log[b:]))
"""
    out, _ = fake_driver.run(program, tmp_path)
    assert out.splitlines()[1:] == ["2 2 0 0"] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pools_read_behind_the_stream_of_their_interface(gpu, dtype):
    # Nothing but the stream orders the copy behind a write that takes long.
    import numpy as np

    torch = pytest.importorskip("torch")
    n = 1 << 17
    cache = gpu.KVCache(n // 256, 256, 2, 64, dtype)
    batch = cache.batch(np.arange(n // 256)[None], [n], appended=[n])
    pools = cache.pools()
    rows = [gpu.tensor([n, 2, 64], np.full(n * 128, x, np.float32)) for x in (1.0, 2.0, 4.0)]
    for x, r in zip((1.0, 2.0, 4.0), rows):
        for other in rows:
            batch.append(other, other)
        batch.append(r, r)
        stream = torch.cuda.ExternalStream(pools[1].__cuda_array_interface__["stream"])
        with torch.cuda.stream(stream):
            got = torch.as_tensor(pools[1], device="cuda").clone()
        stream.synchronize()
        assert bool((got.view(torch.bfloat16 if dtype == "bf16" else torch.float32) == x).all())
