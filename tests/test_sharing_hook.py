"""The hook that makes tests share small prefixes is a matter of the batches made
while it is on: others', before and after, go on as they were."""

import numpy as np
import pytest

from test_shared_prefix import Shared


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_a_batch_keeps_what_it_was_made_with(gpu, dtype):
    from porch_b200._lib import lib

    rng = np.random.default_rng(4)
    host = Shared(rng, [(20, 256)], [300 + s for s in range(20)], 2, 64, 64, dtype)
    cache, before = host.build(gpu)
    q = rng.normal(0, 1, (20, 4, 64)).astype(np.float32)
    t = gpu.tensor(list(q.shape), q)
    alone = gpu.paged_attention(t, cache.batch(host.tables, host.lengths, appended=[0] * 20)).cpu()
    assert lib().pb_test_share_prefix(1) == 0
    try:
        shared = cache.batch(host.tables, host.lengths, appended=[0] * 20, prefix=host.prefix)
        assert np.array_equal(gpu.paged_attention(t, before).cpu(), alone)
        once = gpu.paged_attention(t, shared).cpu()
    finally:
        assert lib().pb_test_share_prefix(0) == 0
    assert not np.array_equal(once, alone)
    assert np.array_equal(gpu.paged_attention(t, shared).cpu(), once)
    assert np.array_equal(gpu.paged_attention(t, shared.on(cache)).cpu(), once)
    out, tol, _, _ = host.attend(q, 0.125)
    assert (np.abs(once.reshape(q.shape) - out) <= tol).all()
