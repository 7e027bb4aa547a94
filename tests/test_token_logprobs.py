"""Log probabilities of given tokens, entropy and alternatives against their
definition in 64 bits, and the gradient against the formula and differences."""

import numpy as np
import pytest

U = 2.0**-24

SIZES = [(1, 1), (3, 2), (5, 31), (2, 33), (7, 500), (1, 4097), (4, 8191), (2, 32768), (1, 100003), (700, 257), (37, 50257),
         (1, 1 << 20)]


def make(rng, rows, vocab):
    x = (rng.normal(0, 1, (rows, vocab)) * rng.uniform(0.2, 6, (rows, 1))).astype(np.float32)
    tokens = rng.integers(0, vocab, rows)
    return x, tokens.astype(np.float32)


def define(x, tokens):
    """(log probabilities, entropies, m, s, p, log p) of finite or masked rows in 64 bits."""
    x = x.astype(np.float64)
    m = x.max(1)
    e = np.exp(x - m[:, None])
    s = e.sum(1)
    logp = x - m[:, None] - np.log(s)[:, None]
    p = e / s[:, None]
    entropy = -np.where(p > 0, p * np.where(p > 0, logp, 0), 0).sum(1)
    t = tokens.astype(int)
    said = np.where(t >= 0, logp[np.arange(len(t)), np.maximum(t, 0)], 0.0)
    return said, entropy, m, s, p, logp


def sum_error(x, m, p):
    """Relative error of a row's sum: an exponential is off by 2^-22 (ex2.approx,
    and units of log2) and by 2 u |x - m|, weighted by p; a thread adds at most
    V / 4096 + 1 groups of 16 in two chains, and up to 11 joins with a
    rescaling of two steps follow."""
    d = np.where(p > 0, np.where(p > 0, m[:, None] - x, 0) * p, 0).sum(1)
    return 2.0**-22 + 3 * U * d + (x.shape[1] / 4096 + 60) * U


def check_forward(x, tokens, got, top=0):
    rows, vocab = x.shape
    said, entropy, m, s, p, logp = define(x, tokens)
    off = sum_error(x.astype(np.float64), m, p)
    got = [g.cpu() for g in got]
    # log p = (x - m) - log s: each step rounded, log s off by off (and an ulp).
    tol = off + 4 * U * (np.abs(said) + np.log(s) + 1e-30)
    assert (np.abs(got[0] - said) <= tol).all()
    # H = log s - w / s, where w's terms are off as the sum's, by 2 u more each.
    mean = np.where(p > 0, p * np.where(p > 0, x - m[:, None], 0), 0).sum(1)
    assert (np.abs(got[1] - entropy) <= off + (3 * off + 8 * U) * np.abs(mean) + 4 * U * np.log(s) + 1e-30).all()
    norm = got[2].reshape(rows, 2)
    assert np.array_equal(norm[:, 0], m.astype(np.float32))
    assert (np.abs(norm[:, 1] - s) <= (off + U) * s).all()
    if top:
        order = np.argsort(-x, axis=1, kind="stable")[:, :top]
        assert np.array_equal(got[4].reshape(rows, top), order)
        want = np.take_along_axis(logp, order, 1)
        near = off[:, None] + 4 * U * (np.abs(want) + np.log(s)[:, None])
        with np.errstate(invalid="ignore"):
            assert ((np.abs(got[3].reshape(rows, top) - want) <= near) | (got[3].reshape(rows, top) == want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_against_the_definition(gpu, rows, vocab):
    rng = np.random.default_rng(rows * 7 + vocab)
    x, tokens = make(rng, rows, vocab)
    if rows > 1:
        tokens[1] = -1
    logits, t = gpu.tensor([rows, vocab], x), gpu.tensor([rows], tokens)
    check_forward(x, tokens, gpu.token_logprobs(logits, t))
    for top in sorted({1, min(7, vocab), min(32, vocab)}):
        check_forward(x, tokens, gpu.token_logprobs(logits, t, top=top), top)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("bonus", [False, True])
def test_gradient_against_the_formula(gpu, rows, vocab, bonus):
    rng = np.random.default_rng(rows * 5 + vocab)
    x, tokens = make(rng, rows, vocab)
    if rows > 2:
        tokens[2] = -1
    g, h = (rng.normal(0, 1, rows).astype(np.float32) for _ in range(2))
    logits, t = gpu.tensor([rows, vocab], x), gpu.tensor([rows], tokens)
    _, entropy, norm = gpu.token_logprobs(logits, t)
    more = dict(d_entropy=gpu.tensor([rows], h), entropy=entropy) if bonus else {}
    got = gpu.token_logprobs_backward(gpu.tensor([rows], g), logits, t, norm, **more).cpu().reshape(rows, vocab)
    _, ent, m, s, p, logp = define(x, tokens)
    off = sum_error(x.astype(np.float64), m, p)[:, None]
    live = (tokens >= 0)[:, None]
    hot = (np.arange(vocab) == tokens[:, None]) & live
    want = np.where(live, g[:, None], 0.0) * (hot - p)
    # p: x - m rounded (u |x - m|), the exponential (2^-22 and 4 u), 1 / s and s.
    p_off = p * (U * np.abs(x - m[:, None]) + 2.0**-22 + 12 * U + off)
    tol = np.abs(g[:, None]) * (p_off + 4 * U * (p + hot)) + 2.0**-126 * (1 + np.abs(g[:, None]))
    if bonus:
        inner = logp + ent[:, None]
        want = want - h[:, None] * p * inner
        mean = (p * np.abs(x - m[:, None])).sum(1)[:, None]
        inner_off = off + (3 * off + 8 * U) * mean + 6 * U * (np.abs(x - m[:, None]) + ent[:, None] + 2 * np.log(s)[:, None] + 1)
        tol = tol + np.abs(h[:, None]) * (p_off * np.abs(inner) + p * inner_off + 4 * U * p * np.abs(inner))
        tol = tol + 2.0**-126 * np.abs(h[:, None]) * (1 + np.abs(inner))
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    rng = np.random.default_rng(5)
    rows, vocab, step = 4, 19, 1e-4
    x, tokens = make(rng, rows, vocab)
    g, h = (rng.normal(0, 1, rows).astype(np.float32) for _ in range(2))
    logits, t = gpu.tensor([rows, vocab], x), gpu.tensor([rows], tokens)
    _, entropy, norm = gpu.token_logprobs(logits, t)
    got = gpu.token_logprobs_backward(gpu.tensor([rows], g), logits, t, norm, gpu.tensor([rows], h), entropy)
    got = got.cpu().reshape(rows, vocab)

    def loss(y):
        said, ent, *_ = define64(y, tokens)
        return (g * said + h * ent).sum()

    def define64(y, tokens):
        m = y.max(1, keepdims=True)
        logp = y - m - np.log(np.exp(y - m).sum(1, keepdims=True))
        return logp[np.arange(rows), tokens.astype(int)], -(np.exp(logp) * logp).sum(1)

    for i in range(rows):
        for j in range(vocab):
            up, down = x.astype(np.float64), x.astype(np.float64)
            up[i, j] += step
            down[i, j] -= step
            d = (loss(up) - loss(down)) / (2 * step)
            # The difference is off by step^2 / 6 of third derivatives, which stay
            # below 8 (|g| + |h| (1 + |log p|)); the kernel by a few units.
            assert abs(got[i, j] - d) <= 1e-6 * (1 + np.abs(g[i]) + np.abs(h[i]) * 40)


@pytest.mark.gpu
def test_equal_logits_and_rows_in_order(gpu):
    vocab = 5000
    rows = np.stack([np.zeros(vocab), np.arange(vocab), -np.arange(vocab), np.arange(vocab) % 7,
                     np.where(np.arange(vocab) == 4321, 0.0, -0.0)]).astype(np.float32)
    tokens = np.array([0, 4999, 0, 6, 3], np.float32)
    got = gpu.token_logprobs(gpu.tensor([5, vocab], rows), gpu.tensor([5], tokens), top=32)
    check_forward(rows, tokens, got, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("low", [-np.inf, np.finfo(np.float32).min])
def test_masked_logits(gpu, low):
    rng = np.random.default_rng(11)
    x, tokens = make(rng, 6, 9001)
    x[0, 1:] = low  # one token left
    tokens[0] = 0
    x[1, 100:] = low
    tokens[1] = 7
    x[2, ::2] = low
    tokens[2] = 8999
    x[3, :9000] = low
    tokens[3] = 9000
    logits, t = gpu.tensor([6, 9001], x), gpu.tensor([6], tokens)
    got = gpu.token_logprobs(logits, t, top=20)
    check_forward(x, tokens, got, 20)
    assert got[0].cpu()[0] == 0 and got[1].cpu()[0] == 0 and got[1].cpu()[3] == 0
    g = gpu.tensor([6], np.ones(6, np.float32))
    d = gpu.token_logprobs_backward(g, logits, t, got[2], g, got[1]).cpu().reshape(6, 9001)
    assert np.isfinite(d).all() and not d[x == low].any()
    # A masked token is said with probability 0.
    said = gpu.token_logprobs(logits, gpu.tensor([6], np.array([5, 200, 0, 1, -1, -1], np.float32)))[0].cpu()
    assert (said[:4] <= -3e38).all() and not said[4:].any()


@pytest.mark.gpu
def test_rows_of_the_lowest_value_are_flat(gpu):
    x = np.full((2, 300), np.finfo(np.float32).min, np.float32)
    tokens = np.array([3, 299], np.float32)
    check_forward(x, tokens, gpu.token_logprobs(gpu.tensor([2, 300], x), gpu.tensor([2], tokens), top=4), 4)


@pytest.mark.gpu
def test_rows_that_are_not_finite_and_bad_tokens_stay_by_themselves(gpu):
    rng = np.random.default_rng(12)
    x, tokens = make(rng, 9, 700)
    want = [r.cpu() for r in gpu.token_logprobs(gpu.tensor([9, 700], x), gpu.tensor([9], tokens), top=3)]
    x[1, 5], x[2, 6], x[3] = np.nan, np.inf, -np.inf
    x[4, :] = np.nan
    tokens[4] = -1
    tokens[5:8] = [700, 2.5, -2]
    logits, t = gpu.tensor([9, 700], x), gpu.tensor([9], tokens)
    out = gpu.token_logprobs(logits, t, top=3)
    got = [r.cpu() for r in out]
    assert np.isnan(got[0][[1, 2, 3, 5, 6, 7]]).all() and got[0][4] == 0
    assert np.isnan(got[1][1:5]).all() and np.isnan(got[2].reshape(9, 2)[1:5, 1]).all()
    assert np.isnan(got[3].reshape(9, 3)[1:5]).all()
    top = got[4].reshape(9, 3)
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x)[:4], axis=1, kind="stable")[:, :3]
    assert np.array_equal(top[:4], order) and np.array_equal(top[4], [0, 1, 2])
    for i in (0, 8):
        assert got[0][i] == want[0][i]
    for i in (0, 5, 6, 7, 8):
        assert got[1][i] == want[1][i]
        assert all(np.array_equal(got[j].reshape(9, -1)[i], want[j].reshape(9, -1)[i]) for j in (2, 3, 4))
    g = gpu.tensor([9], np.ones(9, np.float32))
    d = gpu.token_logprobs_backward(g, logits, t, out[2]).cpu().reshape(9, 700)
    assert np.isnan(d[[1, 2, 3, 5, 6, 7]]).all() and not d[4].any() and np.isfinite(d[[0, 8]]).all()
    # A padded row whose entropy has no gradient gives zeros, too.
    h = gpu.tensor([9], np.zeros(9, np.float32))
    assert not gpu.token_logprobs_backward(g, logits, t, out[2], h, out[1]).cpu().reshape(9, 700)[4].any()


@pytest.mark.gpu
def test_nan_comes_last(gpu):
    x = np.array([[np.nan, -np.inf, 3, np.nan, 2]], np.float32)
    top = gpu.token_logprobs(gpu.tensor([1, 5], x), gpu.tensor([1], np.zeros(1, np.float32)), top=5)[4].cpu().reshape(5)
    assert np.array_equal(top, [2, 4, 1, 0, 3])


@pytest.mark.gpu
def test_views_are_read_in_place(gpu):
    rng = np.random.default_rng(13)
    wide = rng.normal(0, 2, (12, 1003)).astype(np.float32)
    base = gpu.tensor([12, 1003], wide)
    for rows, columns in ((slice(1, 12, 2), slice(3, 900)), (slice(0, 12), slice(1, 1003)), (slice(5, 6), slice(2, 999))):
        x = np.ascontiguousarray(wide[rows, columns])
        n, v = x.shape
        tokens = rng.integers(0, v, n).astype(np.float32)
        view = gpu.materialize(base[rows, columns])
        t = gpu.tensor([n], tokens)
        got = gpu.token_logprobs(view, t, top=5)
        check_forward(x, tokens, got, 5)
        g = gpu.tensor([n], rng.normal(0, 1, n).astype(np.float32))
        a = gpu.token_logprobs_backward(g, view, t, got[2], g, got[1]).cpu()
        b = gpu.token_logprobs_backward(g, gpu.tensor([n, v], x), t, got[2], g, got[1]).cpu()
        assert np.array_equal(a, b)
    # One whose innermost axis is not contiguous is copied first.
    turned = gpu.materialize(gpu.transpose(base))
    tokens = np.zeros(1003, np.float32)
    check_forward(np.ascontiguousarray(wide.T), tokens, gpu.token_logprobs(turned, gpu.tensor([1003], tokens), top=3), 3)


@pytest.mark.gpu
def test_no_rows(gpu):
    x, t = gpu.zeros([0, 50]), gpu.zeros([0])
    out = gpu.token_logprobs(x, t, top=4)
    assert [o.shape() for o in out] == [[0], [0], [0, 2], [0, 4], [0, 4]]
    assert gpu.token_logprobs_backward(t, x, t, out[2]).shape() == [0, 50]


@pytest.mark.gpu
def test_the_same_every_time_and_from_other_threads(gpu):
    import threading

    rng = np.random.default_rng(14)
    x, tokens = make(rng, 3, 70001)
    logits, t = gpu.tensor([3, 70001], x), gpu.tensor([3], tokens)
    want = [r.cpu() for r in gpu.token_logprobs(logits, t, top=32)]
    lazy, wrong = gpu.as_tensor(logits * 1.0), []

    def work():
        for _ in range(5):
            got = [r.cpu() for r in gpu.token_logprobs(lazy, t, top=32)]
            if not all(np.array_equal(a, b) for a, b in zip(got, want)):
                wrong.append(got)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


def test_refusals(api):
    x, t = api.placeholder([4, 50]), api.placeholder([4])
    for logits, tokens, top in ((api.placeholder([4]), t, 0), (x, api.placeholder([5]), 0), (x, api.placeholder([4, 1]), 0),
                                (x, t, 33), (x, t, -1), (api.placeholder([4, 3]), t, 4), (api.placeholder([4, 0]), t, 0),
                                (api.placeholder([4, (1 << 24) + 1]), t, 0)):
        with pytest.raises(api.InvalidArgument, match="token_logprobs"):
            api.token_logprobs(logits, tokens, top=top)
    n = api.placeholder([4, 2])
    for args in ((api.placeholder([5]), x, t, n), (t, x, t, api.placeholder([4, 3])), (t, x, t, n, t), (t, x, t, n, None, t),
                 (t, x, t, n, t, api.placeholder([3])), (t, x, t, n, api.placeholder([3]), t), (t, t, t, n)):
        with pytest.raises(api.InvalidArgument, match="token_logprobs"):
            api.token_logprobs_backward(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("at", range(6))
def test_every_operand_needs_values(gpu, at):
    given = [gpu.zeros(s) for s in ([4], [4, 50], [4], [4, 2], [4], [4])]
    given[at] = gpu.placeholder(given[at].shape())
    with pytest.raises(RuntimeError, match="placeholder"):
        gpu.token_logprobs_backward(*given)
    if at in (1, 2):
        with pytest.raises(RuntimeError, match="placeholder"):
            gpu.token_logprobs(*given[1:3])


@pytest.mark.gpu
def test_gradient_of_many_rows(gpu):
    # As many as take several rounds a block; every row against the formula.
    rng = np.random.default_rng(21)
    rows, vocab = 700, 65539
    x, tokens = make(rng, rows, vocab)
    x[:, 60000:] = -np.inf
    tokens = np.minimum(tokens, 59999)
    tokens[::7] = -1
    g, h = (rng.normal(0, 1, rows).astype(np.float32) for _ in range(2))
    logits, t = gpu.tensor([rows, vocab], x), gpu.tensor([rows], tokens)
    _, entropy, norm = gpu.token_logprobs(logits, t)
    got = gpu.token_logprobs_backward(gpu.tensor([rows], g), logits, t, norm, gpu.tensor([rows], h), entropy)
    got = got.cpu().reshape(rows, vocab)
    for i in range(0, rows, 13):
        y, at = x[i : i + 1].astype(np.float64), tokens[i : i + 1]
        _, ent, m, s, p, logp = define(y, at)
        off = sum_error(y, m, p)
        inner = np.where(p > 0, logp + ent, 0)
        hot = (np.arange(vocab) == at[0]) & (at[0] >= 0)
        want = (g[i] if at[0] >= 0 else 0.0) * (hot - p) - h[i] * p * inner
        gap = np.where(p > 0, m - y, 0)
        p_off = p * (U * gap + 2.0**-22 + 12 * U + off)
        inner_off = off + (3 * off + 8 * U) * (p * gap).sum() + 6 * U * (gap + ent + 2 * np.log(s) + 1)
        tol = np.abs(g[i]) * (p_off + 4 * U * (p + hot)) + np.abs(h[i]) * (p_off * np.abs(inner) + p * inner_off + 4 * U * p * np.abs(inner))
        tol = tol + 2.0**-126 * (1 + np.abs(g[i]) + np.abs(h[i]) * (1 + np.abs(inner)))
        assert (np.abs(got[i] - want[0]) <= tol[0]).all()


@pytest.mark.gpu
def test_more_than_two_to_the_31_logits(gpu):
    rows, vocab = 16400, 131072
    logits = gpu.zeros([rows, vocab])
    tokens = np.arange(rows, dtype=np.float32)
    t = gpu.tensor([rows], tokens)
    said, entropy, norm, _, best = gpu.token_logprobs(logits, t, top=2)
    flat = np.log(np.float64(vocab))
    # Sums of equal terms in a tree with a thread's 32 rounds at its ends: 64 roundings.
    assert np.abs(said.cpu() + flat).max() <= 64 * U + 4 * U * flat and np.abs(entropy.cpu() - flat).max() <= 64 * U + 4 * U * flat
    assert (best.cpu().reshape(rows, 2) == [0, 1]).all()
    d = gpu.token_logprobs_backward(gpu.tensor([rows], np.ones(rows, np.float32)), logits, t, norm)
    for row in (0, 16383, 16384, rows - 1):
        x = gpu.materialize(d[row : row + 1, gpu.all]).cpu().reshape(vocab)
        want = -np.full(vocab, 1.0 / vocab)
        want[row] += 1
        assert np.abs(x - want).max() <= 2.0**-20
        assert np.abs(np.delete(x, row) * vocab + 1).max() <= 2.0**-17
