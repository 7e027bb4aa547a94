"""The compiled part of the Python binding: argument kinds, errors, lifetimes."""

import gc

import numpy as np
import pytest


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
