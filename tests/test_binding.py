"""The compiled part of the Python binding: argument kinds, errors, lifetimes."""

import gc
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import fake_driver

ROOT = Path(__file__).resolve().parent.parent
# Before the import of porch_b200.api, as on an interpreter without the compiled module.
NOT_COMPILED = """
from pathlib import Path
from porch_b200 import _lib
_lib.binding_path = lambda: Path("/nowhere/_binding.so")
"""


def python(program):
    done = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    return done.stdout


@pytest.mark.parametrize("before", ["", NOT_COMPILED])
def test_an_import_loads_no_native_library(api, before):
    python(before + """
loaded = lambda: "libporch_b200.so" in open("/proc/self/maps").read()
from porch_b200 import api
assert not loaded()
assert api.placeholder([2, 3]).shape() == [2, 3]
assert loaded()
""")


@pytest.mark.parametrize("before", ["", NOT_COMPILED])
def test_a_library_that_is_not_built_fails_at_its_first_use(api, before):
    python(before + """
from pathlib import Path
from porch_b200 import _lib
path = _lib.binding_path() # the compiled part stays where it is
_lib.binding_path = lambda: path
_lib.LIBRARY = Path("/nowhere/libporch_b200.so")
from porch_b200 import api
for use in (lambda: api.placeholder([2]), lambda: api.Tensor(None).__cuda_array_interface__,
            lambda: api.qk_norm_rope(*[api.Tensor(None)] * 7)):
    try:
        use()
        raise SystemExit("no error")
    except ImportError as e:
        assert "is not built" in str(e), e
""")


OPERATORS = """
x = lambda *shape: api.tensor(list(shape), np.arange(np.prod(shape), dtype=np.float32))
cache = api.KVCache(8, 8, 2, 16)
batch = cache.batch(np.arange(8).reshape(2, 4), [20, 30])
q, k = api.qk_norm_rope(x(2, 4, 16), x(2, 2, 16) + 1.0, x(16), x(16), x(9, 8), x(9, 8), x(2), interleaved=True)
grads = api.qk_norm_rope_backward(q, k, q, k, x(16), x(16), x(9, 8), x(9, 8), x(2), eps=0.5)
batch.append(k, k)
out = api.paged_attention(q, batch)
out, scores = api.paged_attention_scored(q, batch, None, 0.25)
out, scores = api.paged_attention_scored(q, batch, scores + 0.0)
kept, places = api.cache_evict(batch, scores, budget=np.int64(12), recent=3)
kept, places = api.cache_evict(batch, scores, places, budget=12, sinks=1)
for t in (q, k, *grads, out, scores, kept, places):
    assert type(t) is api.Tensor and isinstance(t._h, int)
    face = t.__cuda_array_interface__
    assert face is t.__cuda_array_interface__ and face["stream"] == q.__cuda_array_interface__["stream"]
    print(t.shape(), face["shape"], face["typestr"], face["version"], face["data"] == (t.device_data()[0], False))
p = api.placeholder
good = [p([3, 4, 8]), p([3, 2, 8]), p([8]), p([8]), p([16, 4]), p([16, 4]), p([3])]
for call in (lambda: api.qk_norm_rope(*good, eps="small"), lambda: api.qk_norm_rope("q", *good[1:]),
             lambda: api.qk_norm_rope(None, *good[1:]), lambda: api.qk_norm_rope(api.Tensor(None), *good[1:]),
             lambda: api.qk_norm_rope(1.0, *good[1:]), lambda: api.Tensor("text"), lambda: api.Tensor(None).shape(),
             lambda: api.Tensor(None).__cuda_array_interface__, lambda: p([2]).__cuda_array_interface__,
             lambda: api.paged_attention(q, batch, scale="1"), lambda: api.paged_attention(p([2, 4, 16]), batch),
             lambda: api.cache_evict(batch, scores, budget="4"), lambda: api.cache_evict(batch, scores, budget=0),
             lambda: api.paged_attention(q, cache)):
    try:
        call()
        raise SystemExit("no error")
    except Exception as e:
        print(type(e).__name__, e if isinstance(e, (api.InvalidArgument, RuntimeError)) else "")
"""


def test_without_the_compiled_module_everything_is_the_same(api, tmp_path):
    # Over the driver's stand-in: shapes, interfaces, errors, and what is launched.
    seen = []
    for name, before in (("compiled", ""), ("ctypes", NOT_COMPILED)):
        folder = tmp_path / name
        folder.mkdir()
        out, log = fake_driver.run(OPERATORS, folder, before=before)
        launches = [line[3:] for line in log if line[1] == "launch"]
        assert {n[0] for n in launches} >= {"pb_norm_rope", "pb_norm_rope_grad", "pb_cache_append", "pb_paged_attention",
                                            "pb_paged_finish", "pb_evict_select"}
        seen.append((out, launches))
    assert seen[0] == seen[1]


def test_an_array_of_another_library_is_refused_where_a_copy_would_not_be_it(api):
    class Face:
        def __init__(self, **more):
            self.__cuda_array_interface__ = dict(shape=(2, 3), typestr="<f4", data=(0, False), version=3, **more)

    for more, match in ((dict(mask=Face()), "mask"), (dict(strides=(4, 8)), "contiguous")):
        with pytest.raises(api.InvalidArgument, match=match):
            api.tensor_from_device(Face(**more))


@pytest.mark.parametrize("before", ["", NOT_COMPILED])
@pytest.mark.parametrize("slow,what", [
    (dict(slow_compile="pb_elem"), "lazy.__cuda_array_interface__"),  # compiles a kernel: a second
    (dict(slow="cuEventRecord"), "tensors.clear()"),  # a tensor that another stream reads: 0.4 s
])
def test_other_threads_run_meanwhile(api, tmp_path, before, slow, what):
    fake_driver.run("""
tensors = [api.tensor([1000], np.ones(1000, np.float32))]
lazy = api.as_tensor(tensors[0] * 2.0)
q = [api.tensor([1, 1, 8], np.ones(8, np.float32))] * 2
def read():
    w = api.tensor([8], np.ones(8, np.float32))
    c = api.tensor([4, 4], np.ones(16, np.float32))
    tensors.append(api.qk_norm_rope(*q, w, w, c, c, api.tensor([1], np.ones(1, np.float32)))[0])
t = threading.Thread(target=read)
t.start()
t.join()
tensors.append(q.pop())
q.clear()
if """ + repr("lazy" not in what) + """:
    del lazy
def work():
    began = time.perf_counter()
    """ + what + """
    took.append(time.perf_counter() - began)
took, gap, last = [], 0.0, time.perf_counter()
t = threading.Thread(target=work)
t.start()
while t.is_alive():
    time.sleep(0.002)
    now = time.perf_counter()
    gap, last = max(gap, now - last), now
assert took[0] > 0.35 and gap < 0.25, (took, gap)
""", tmp_path, before=before, **slow)


@pytest.mark.gpu
def test_without_the_compiled_module_results_are_the_same(gpu):
    program = """
import numpy as np
from porch_b200 import api, _lib
""" + OPERATORS[: OPERATORS.index("for t in")] + """
for t in (q, k, *grads, out, scores, kept, places):
    print(t.cpu().tobytes().hex())
print(type(_lib.binding().paged_attention).__name__)
"""
    (*a, compiled), (*b, plain) = python(program).split(), python(NOT_COMPILED + program).split()
    assert a == b and compiled == "builtin_function_or_method" and plain == "function"


def test_handles(api):
    t = api.placeholder([2, 3])
    assert isinstance(t, api.Tensor) and isinstance(t._h, int) and t._h != 0
    with pytest.raises(RuntimeError):
        t.__cuda_array_interface__
    with pytest.raises(RuntimeError):  # again: an error is not kept
        t.__cuda_array_interface__
    none = api.Tensor(None)
    assert none._h is None
    with pytest.raises(api.InvalidArgument, match="null"):
        none.shape()
    with pytest.raises(api.InvalidArgument, match="null"):
        none.__cuda_array_interface__
    with pytest.raises(TypeError):
        api.Tensor("text")
    for _ in range(1000):
        api.placeholder([4])
    gc.collect()


def test_argument_kinds(api):
    p = api.placeholder
    good = [p([3, 4, 8]), p([3, 2, 8]), p([8]), p([8]), p([16, 4]), p([16, 4]), p([3])]
    with pytest.raises(TypeError):
        api.qk_norm_rope(*good, eps="small")
    with pytest.raises(TypeError):
        api.qk_norm_rope("q", *good[1:])
    with pytest.raises(TypeError):
        api.qk_norm_rope(None, *good[1:])
    with pytest.raises(api.InvalidArgument, match="q is null"):
        api.qk_norm_rope(api.Tensor(None), *good[1:])
    with pytest.raises(api.InvalidArgument):  # a number is no tensor expression
        api.qk_norm_rope(1.0, *good[1:])


@pytest.mark.gpu
def test_expressions_are_realised_and_results_outlive_their_inputs(gpu):
    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (4, 3, 16)).astype(np.float32)
    ones, table = np.ones(16, np.float32), np.ones((8, 8), np.float32)

    def call(lazy):
        q = gpu.tensor([4, 3, 16], x)
        parts = [q, q, gpu.tensor([16], ones), gpu.tensor([16], ones), gpu.tensor([8, 8], table),
                 gpu.tensor([8, 8], 0 * table), gpu.tensor([4], np.arange(4, dtype=np.float32))]
        return gpu.qk_norm_rope(*[(t + 0.0) if lazy else t for t in parts])

    want = [t.cpu() for t in call(False)]
    got = call(True)
    gc.collect()
    assert all(np.array_equal(a, b.cpu()) for a, b in zip(want, got))


@pytest.mark.gpu
def test_interface(gpu):
    t = gpu.tensor([2, 5], np.arange(10, dtype=np.float32))
    face = t.__cuda_array_interface__
    assert face["shape"] == (2, 5) and face["typestr"] == "<f4" and face["version"] == 3
    assert face["data"] == (t.device_data()[0], False) and face["stream"]
    assert t.__cuda_array_interface__ is face
    assert gpu.tensor([0, 3], np.zeros(0, np.float32)).__cuda_array_interface__["data"] == (0, False)
    lazy = gpu.as_tensor(t * 2.0)
    assert lazy.__cuda_array_interface__["shape"] == (2, 5)
    torch = pytest.importorskip("torch")
    view = torch.as_tensor(lazy, device="cuda")
    del lazy, t
    gc.collect()
    gpu.synchronize()
    assert view.sum().item() == 90


@pytest.mark.gpu
def test_interface_of_a_placeholder(gpu):
    for _ in range(2):
        with pytest.raises(RuntimeError, match="placeholder"):
            gpu.placeholder([2, 3]).__cuda_array_interface__


@pytest.mark.gpu
def test_batch_arguments(gpu):
    cache = gpu.KVCache(4, 8, 1, 8)
    batch = cache.batch([[0, 1]], [9])
    q = gpu.zeros([1, 1, 8])
    scores = gpu.zeros([1, 1, 9])
    with pytest.raises(TypeError):
        gpu.cache_evict(batch, scores, budget="4")
    with pytest.raises(TypeError):
        gpu.paged_attention(q, batch, scale="1")
    with pytest.raises(AttributeError):
        gpu.paged_attention(q, cache)
    out, _ = gpu.cache_evict(batch, scores + 1.0, None, budget=np.int64(4))
    assert out.shape() == [1, 1, 4] and (out.cpu() == 1).all()
