"""Norms and rotation of query and key heads, and their gradient, against the
formulas in 64 bits.

Bounds, from the arithmetic (u = 2^-24, one rounding): a head's mean square is
a chain of at most 32 fused adds per lane, 5 shuffled adds and one more, so 40 u
at most, which the square root halves; rsqrtf is within 2 ulp (4 u); two
products, and the rotation's products and sum are 5 u of |a c| + |b s|. In all
below 32 u = 2^-19 of |a c| + |b s|. The gradient's inner mean adds another
chain and its products: below 64 u = 2^-18 of the terms' absolute sum. A
weight's gradient is a sum of N = tokens x heads terms, each within 64 u: below
(64 + N) u of the sum of their absolute values.
"""

import numpy as np
import pytest

U = 2.0**-24


def turn(x, c, s, rot, interleaved):
    y = x.copy()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2 : rot])
    p, q = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = p, q
    else:
        y[..., : rot // 2], y[..., rot // 2 : rot] = p, q
    return y


def turned_size(x, c, s, rot, interleaved):
    """|a c| + |b s| and its partner: what the rotation's rounding is relative to."""
    c, s = np.abs(c), np.abs(s)
    y = np.abs(x)
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., : rot // 2], y[..., rot // 2 : rot])
    p, q = a * c + b * s, b * c + a * s
    out = y.copy()
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = p, q
    else:
        out[..., : rot // 2], out[..., rot // 2 : rot] = p, q
    return out


def forward(x, w, c, s, rot, eps, interleaved):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return turn(x * r * w, c, s, rot, interleaved), turned_size(x * r * w, c, s, rot, interleaved)


def backward(dy, x, w, c, s, rot, eps, interleaved):
    g = turn(dy, c, -s, rot, interleaved)
    size = turned_size(dy, c, s, rot, interleaved)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = x * r
    dx = r * (g * w - n * (g * w * n).mean(-1, keepdims=True))
    dx_size = r * (size * np.abs(w) + np.abs(n) * (size * np.abs(w * n)).mean(-1, keepdims=True))
    return dx, dx_size, (g * n).sum((0, 1)), (size * np.abs(n)).sum((0, 1))


def inputs(rng, t, hq, hk, d, rot, table, interleaved=False):
    x = {
        "q": rng.normal(0, 2, (t, hq, d)),
        "k": rng.normal(0, 0.1, (t, hk, d)),
        "qw": rng.normal(1, 0.3, d),
        "kw": rng.normal(1, 0.3, d),
        "pos": rng.integers(0, table, t).astype(np.float64),
    }
    angle = np.arange(table)[:, None] * 100.0 ** (-np.arange(rot // 2) / (rot // 2))
    x["cos"], x["sin"] = np.cos(angle), np.sin(angle)
    return {k: v.astype(np.float32) for k, v in x.items()}


def rows(x):
    at = x["pos"].astype(int)
    return x["cos"][at][:, None].astype(np.float64), x["sin"][at][:, None].astype(np.float64)


def test_the_formula_is_the_gradient_of_differences():
    rng = np.random.default_rng(3)
    for interleaved in (False, True):
        x = {k: v.astype(np.float64) for k, v in inputs(rng, 2, 3, 1, 10, 6, 5).items()}
        c, s = rows(x)
        dy = rng.normal(0, 1, x["q"].shape)
        dx, _, dw, _ = backward(dy, x["q"], x["qw"], c, s, 6, 1e-6, interleaved)

        def loss(q, w):
            return (forward(q, w, c, s, 6, 1e-6, interleaved)[0] * dy).sum()

        h = 1e-6
        for at in [(0, 0, 0), (1, 2, 9), (0, 1, 5)]:
            e = np.zeros_like(x["q"])
            e[at] = h
            assert abs((loss(x["q"] + e, x["qw"]) - loss(x["q"] - e, x["qw"])) / (2 * h) - dx[at]) < 1e-6
        for i in (0, 4, 9):
            e = np.zeros(10)
            e[i] = h
            assert abs((loss(x["q"], x["qw"] + e) - loss(x["q"], x["qw"] - e)) / (2 * h) - dw[i]) < 1e-6


def test_refusals(api):
    p = api.placeholder
    good = [p([3, 4, 8]), p([3, 2, 8]), p([8]), p([8]), p([16, 4]), p([16, 4]), p([3])]

    def refuse(message, at, shape, **more):
        bad = list(good)
        bad[at] = p(shape)
        with pytest.raises(api.InvalidArgument, match=message):
            api.qk_norm_rope(*bad, **more)

    refuse("tokens, heads, head_dim", 0, [3, 32])
    refuse("same tokens and head_dim", 1, [2, 2, 8])
    refuse("same tokens and head_dim", 1, [3, 2, 4])
    refuse("heads", 1, [3, 0, 8])
    refuse("weights", 2, [4])
    refuse("weights", 3, [1, 8])
    refuse("cos and sin", 5, [16, 3])
    refuse("positions must be", 6, [4])
    wide = list(good)
    wide[4] = wide[5] = p([16, 5])
    with pytest.raises(api.InvalidArgument, match="rot must be"):
        api.qk_norm_rope(*wide)
    with pytest.raises(api.InvalidArgument, match="eps"):
        api.qk_norm_rope(*good, eps=-1.0)
    with pytest.raises(api.InvalidArgument, match="shapes of q and k"):
        api.qk_norm_rope_backward(p([3, 2, 8]), good[1], *good)
    with pytest.raises(RuntimeError, match="placeholder"):
        api.qk_norm_rope(*good)
    with pytest.raises(RuntimeError, match="placeholder"):
        api.qk_norm_rope_backward(good[0], good[1], *good)


def test_shared_memory_written_in_vectors_is_aligned(api):
    # pb_store_head writes a group's row of `sums` in up to 16 bytes; the
    # language only promises a float's alignment for an array of floats.
    text = api.operator_sources()
    declared = [line for line in text.splitlines() if "__shared__" in line and " sums[PB_GPB]" in line]
    assert declared and all("__align__(16)" in line for line in declared)


CASES = [
    # tokens, q heads, k heads, head size, rotated, interleaved
    (1, 1, 1, 2, 2, False),
    (1, 8, 2, 64, 64, False),
    (1, 8, 2, 64, 64, True),
    (7, 5, 3, 80, 40, False),
    (7, 5, 3, 80, 40, True),
    (3, 4, 4, 37, 18, False),
    (3, 4, 4, 37, 18, True),
    (33, 3, 1, 128, 128, False),
    (33, 9, 2, 96, 32, True),
    (5, 2, 1, 256, 128, False),
    (2, 2, 1, 1024, 64, False),
    (2, 2, 1, 1023, 1022, False),
    (257, 6, 1, 6, 4, True),
    (600, 7, 2, 72, 72, False),
    (1500, 5, 3, 64, 64, False),
    (2500, 3, 1, 40, 24, True),
    (1300, 3, 2, 513, 512, False),
]


def tensors(api, x):
    return {k: api.tensor(list(v.shape), v) for k, v in x.items()}


def call(t):
    return [t[k] for k in ("q", "k", "qw", "kw", "cos", "sin", "pos")]


@pytest.mark.gpu
@pytest.mark.parametrize("t,hq,hk,d,rot,interleaved", CASES)
def test_forward_and_gradient(gpu, t, hq, hk, d, rot, interleaved):
    rng = np.random.default_rng(d * 131 + t)
    x = inputs(rng, t, hq, hk, d, rot, 50)
    dq, dk = (rng.normal(0, 1, (t, h, d)).astype(np.float32) for h in (hq, hk))
    m = tensors(gpu, x)
    c, s = rows(x)
    got = gpu.qk_norm_rope(*call(m), eps=1e-5, interleaved=interleaved)
    for name, weight, out in (("q", "qw", got[0]), ("k", "kw", got[1])):
        want, size = forward(x[name].astype(np.float64), x[weight].astype(np.float64), c, s, rot, 1e-5, interleaved)
        assert (np.abs(out.cpu().reshape(want.shape) - want) <= 2.0**-19 * size + 1e-37).all()
    grads = gpu.qk_norm_rope_backward(gpu.tensor([t, hq, d], dq), gpu.tensor([t, hk, d], dk), *call(m), eps=1e-5,
                                      interleaved=interleaved)
    for name, weight, dy, dx, dw in (("q", "qw", dq, grads[0], grads[2]), ("k", "kw", dk, grads[1], grads[3])):
        want, size, wsum, wsize = backward(dy.astype(np.float64), x[name].astype(np.float64),
                                           x[weight].astype(np.float64), c, s, rot, 1e-5, interleaved)
        assert (np.abs(dx.cpu().reshape(want.shape) - want) <= 2.0**-18 * size + 1e-37).all()
        terms = t * dy.shape[1]
        assert (np.abs(dw.cpu() - wsum) <= (64 + terms) * U * wsize + 1e-37).all()


@pytest.mark.gpu
def test_strided_views_are_read_in_place(gpu):
    # Heads of a fused projection, at a channel offset that breaks 16-byte
    # alignment, tokens in reversed roles (a permuted axis), and every other token.
    rng = np.random.default_rng(9)
    x = inputs(rng, 12, 4, 2, 16, 8, 20)
    m = tensors(gpu, x)
    fused = rng.normal(0, 1, (12, 9, 19)).astype(np.float32)
    f = gpu.tensor([12, 9, 19], fused)
    want_q, want_k = fused[:, 1:5, 3:19], fused[:, 5:7, 3:19]
    q = gpu.materialize(f[gpu.all, 1:5, 3:19])
    k = gpu.materialize(f[gpu.all, 5:7, 3:19])
    a = gpu.qk_norm_rope(q, k, *call(m)[2:])
    b = gpu.qk_norm_rope(gpu.tensor([12, 4, 16], want_q), gpu.tensor([12, 2, 16], want_k), *call(m)[2:])
    for x1, x2 in zip(a, b):
        assert np.allclose(x1.cpu(), x2.cpu(), rtol=1e-6, atol=1e-6)
    heads_first = gpu.tensor([4, 12, 16], np.ascontiguousarray(want_q.transpose(1, 0, 2)))
    p = gpu.materialize(gpu.permute(heads_first, [1, 0, 2]))
    c = gpu.qk_norm_rope(p, k, *call(m)[2:])
    assert np.allclose(c[0].cpu(), b[0].cpu(), rtol=1e-6, atol=1e-6)
    inner = gpu.materialize(gpu.permute(gpu.tensor([12, 16, 4], np.ascontiguousarray(want_q.transpose(0, 2, 1))),
                                        [0, 2, 1]))
    d = gpu.qk_norm_rope(inner, k, *call(m)[2:])
    assert np.array_equal(d[0].cpu(), b[0].cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_outside_the_table_and_values_that_are_not_finite(gpu, interleaved):
    rng = np.random.default_rng(4)
    x = inputs(rng, 8, 2, 1, 16, 8, 20)
    want = [t.cpu().reshape(8, -1, 16) for t in gpu.qk_norm_rope(*call(tensors(gpu, x)), interleaved=interleaved)]
    bad = dict(x)
    bad["pos"] = x["pos"].copy()
    bad["pos"][[1, 2, 3, 4, 5]] = [20, -1, 2.5, np.nan, np.inf]
    got = [t.cpu().reshape(8, -1, 16) for t in gpu.qk_norm_rope(*call(tensors(gpu, bad)), interleaved=interleaved)]
    for g, w in zip(got, want):
        assert np.isnan(g[1:6]).all()
        assert np.array_equal(g[[0, 6, 7]], w[[0, 6, 7]])
    # A head that is not finite leaves every other head as it was.
    bad = dict(x)
    bad["q"] = x["q"].copy()
    bad["q"][3, 1, 15] = np.inf
    got = gpu.qk_norm_rope(*call(tensors(gpu, bad)), interleaved=interleaved)
    g = got[0].cpu().reshape(8, 2, 16)
    assert np.isnan(g[3, 1, 15])
    keep = np.ones((8, 2), dtype=bool)
    keep[3, 1] = False
    assert np.array_equal(g[keep], want[0][keep])
    assert np.array_equal(got[1].cpu().reshape(8, 1, 16), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("at", range(9))
def test_every_operand_needs_values(gpu, at):
    given = [gpu.zeros(s) for s in ([3, 4, 8], [3, 2, 8], [3, 4, 8], [3, 2, 8], [8], [8], [16, 4], [16, 4], [3])]
    given[at] = gpu.placeholder(given[at].shape())
    with pytest.raises(RuntimeError, match="placeholder"):
        gpu.qk_norm_rope_backward(*given)
    if at >= 2:
        with pytest.raises(RuntimeError, match="placeholder"):
            gpu.qk_norm_rope(*given[2:])


@pytest.mark.gpu
def test_no_tokens(gpu):
    rng = np.random.default_rng(4)
    x = inputs(rng, 0, 2, 1, 16, 8, 20)
    m = tensors(gpu, x)
    q, k = gpu.qk_norm_rope(*call(m))
    assert q.shape() == [0, 2, 16] and k.shape() == [0, 1, 16]
    g = gpu.qk_norm_rope_backward(q, k, *call(m))
    assert g[0].shape() == [0, 2, 16] and not g[2].cpu().any() and not g[3].cpu().any()


@pytest.mark.gpu
def test_gradient_is_the_same_every_time(gpu):
    rng = np.random.default_rng(8)
    x = inputs(rng, 500, 6, 3, 64, 64, 50)
    m = tensors(gpu, x)
    dq, dk = (gpu.tensor([500, h, 64], rng.normal(0, 1, (500, h, 64)).astype(np.float32)) for h in (6, 3))
    first = [t.cpu() for t in gpu.qk_norm_rope_backward(dq, dk, *call(m))]
    for _ in range(3):
        again = [t.cpu() for t in gpu.qk_norm_rope_backward(dq, dk, *call(m))]
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
def test_tensors_of_another_thread(gpu):
    import threading

    rng = np.random.default_rng(8)
    x = inputs(rng, 300, 6, 3, 64, 64, 50)
    want = [t.cpu() for t in gpu.qk_norm_rope(*call(tensors(gpu, x)))]
    m = tensors(gpu, x)
    lazy = dict(m)
    lazy["q"], lazy["k"] = gpu.as_tensor(m["q"] * 1.0), gpu.as_tensor(m["k"] * 1.0)
    got = {}

    def work():
        got["out"] = [t.cpu() for t in gpu.qk_norm_rope(*call(lazy))]

    th = threading.Thread(target=work)
    th.start()
    th.join()
    assert all(np.array_equal(a, b) for a, b in zip(got["out"], want))


@pytest.mark.gpu
def test_copies_from_and_to_another_library(gpu):
    torch = pytest.importorskip("torch")
    x = torch.arange(60, device="cuda", dtype=torch.float32).reshape(3, 4, 5)
    t = gpu.tensor_from_device(x)
    x.zero_()
    assert np.array_equal(t.cpu(), np.arange(60, dtype=np.float32).reshape(3, 4, 5))
    view = torch.as_tensor(t, device="cuda")
    assert view.data_ptr() == t.device_data()[0]
    gpu.synchronize()
    assert view.sum().item() == 59 * 30
    with pytest.raises(gpu.InvalidArgument, match="contiguous"):
        gpu.tensor_from_device(x.transpose(0, 1))
    with pytest.raises(gpu.InvalidArgument, match="float32"):
        gpu.tensor_from_device(x.int())
    assert gpu.tensor_from_device(x[:0]).shape() == [0, 4, 5]
