"""The serving operators together: an 8-bit cache behind a shared prompt, what the
model says, and training its output on that."""

import numpy as np
import pytest

from test_shared_prefix import Shared


@pytest.fixture
def sharing():
    from porch_b200._lib import lib

    assert lib().pb_test_share_prefix(1) == 0
    yield
    assert lib().pb_test_share_prefix(0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "int8"])
def test_sequences_behind_a_shared_prompt_decode_as_each_by_itself(gpu, dtype, sharing):
    from porch_b200.decode_step import Decoder, Model

    model = Model(vocabulary=64, width=64, heads=4, kv_heads=2, head_dim=16, positions=128)
    prompt = np.arange(48) * 5 % 64
    # 20 sequences of 2 query heads a key head: 40 queries read the prompt together.
    decoder = Decoder(model, 20, 40, dtype, page_size=8, prompt=prompt)
    plain = Decoder(model, 20, 100, dtype, page_size=8)
    for token in prompt:
        plain.step(np.full(20, token))
    rng = np.random.default_rng(5)
    for _ in range(12):
        tokens = rng.integers(0, 64, 20)
        got, want = decoder.step(tokens), plain.step(tokens)
        # As in the decoding example's test; an 8-bit cache rounds to codes 1 / 254
        # of a row's largest size apart, which may differ by a float32 rounding, too.
        assert np.abs(got - want).max() <= (1e-4 if dtype == "f32" else 0.02) * want.max()
        best, said, entropy = decoder.step_top(tokens, 5)
        p = plain.step(tokens)
        tol = 1e-3 if dtype == "f32" else 0.1
        assert np.abs(np.exp(said) - np.take_along_axis(p, best, 1)).max() <= tol * p.max()
        assert np.abs(entropy + (p * np.log(p)).sum(1)).max() <= 10 * tol
        assert (np.diff(said, axis=1) <= 0).all()
    assert decoder.length == 24 and decoder.seen == 72


@pytest.mark.gpu
def test_a_step_of_serving_and_of_training_on_it(gpu, sharing):
    # New tokens go behind a shared prefix in 8 bits, are attended to, and their
    # heads' output is trained on the tokens that were said: against 64 bits.
    rng = np.random.default_rng(3)
    n, heads, group, dim, vocab = 18, 2, 4, 64, 500
    lengths = [193 + i for i in range(n)]
    host = Shared(rng, [(n, 192)], lengths, heads, dim, 64, "int8")
    cache, _ = host.build(gpu)
    batch = cache.batch(host.tables, lengths, prefix=host.prefix)
    new = [np.stack([x[-1] for x in y]) for y in (host.k, host.v)]
    batch.append(*(gpu.tensor([n, heads, dim], x) for x in new))
    q = rng.normal(0, 1, (n, heads * group, dim)).astype(np.float32)
    a = gpu.paged_attention(gpu.tensor(list(q.shape), q), batch)
    out, tol, _, _ = host.attend(q, dim**-0.5)
    got = a.cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()
    w = rng.normal(0, 0.05, (heads * group * dim, vocab)).astype(np.float32)
    tw = gpu.tensor(list(w.shape), w)
    flat = gpu.materialize(gpu.reshape(a, [n, heads * group * dim]))
    logits = gpu.materialize(gpu.matmul(flat, tw))
    tokens = rng.integers(0, vocab, n).astype(np.float32)
    tokens[4] = -1
    t = gpu.tensor([n], tokens)
    said, entropy, norm, _, best = gpu.token_logprobs(logits, t, top=3)
    g = gpu.tensor([n], np.where(tokens >= 0, -1.0, 0).astype(np.float32) / n)
    h = gpu.tensor([n], np.full(n, -0.01, np.float32))
    d = gpu.token_logprobs_backward(g, logits, t, norm, h, entropy)
    dw = gpu.materialize(gpu.matmul(gpu.transpose(flat), d)).cpu().reshape(w.shape)
    # From the device's own attention on, in 64 bits; each product of 512 or 18
    # terms within 2^-19 of its terms' sizes (as matmul's tests have it).
    x = got.reshape(n, -1).astype(np.float64)
    y = x @ w
    y -= y.max(1, keepdims=True)
    logp = y - np.log(np.exp(y).sum(1, keepdims=True))
    p = np.exp(logp)
    live = tokens >= 0
    at = np.maximum(tokens.astype(int), 0)
    off = 2.0**-19 * (np.abs(x) @ np.abs(w)).max()
    assert np.abs(said.cpu() - np.where(live, logp[np.arange(n), at], 0)).max() <= 4 * off
    assert np.abs(entropy.cpu() + (p * logp).sum(1)).max() <= 40 * off
    assert np.array_equal(best.cpu().reshape(n, 3)[:, 0], p.argmax(1))
    hot = np.zeros((n, vocab))
    hot[np.arange(n), at] = live
    ent = -(p * logp).sum(1, keepdims=True)
    want_d = np.where(live, -1.0 / n, 0)[:, None] * (hot - p * live[:, None]) + 0.01 * p * (logp + ent)
    want = x.T @ want_d
    size = np.abs(x).T @ (np.abs(want_d) + 40 * off * p)
    assert (np.abs(dw - want) <= 40 * off * size + 1e-6 * np.abs(want).max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("more", [["--dtype", "int8"], ["--prompt", "32", "--top", "3"], ["--top", "2", "--dtype", "f32"]])
def test_the_command_runs(gpu, capsys, more):
    from porch_b200 import decode_step

    decode_step.main(["--steps", "12", "--sequences", "3", "--budget", "8", *more])
    out = capsys.readouterr().out
    assert "sequence 2:" in out and "ms a step" in out
    assert ("entropy" in out) == ("--top" in more)


@pytest.mark.gpu
def test_a_prompt_that_does_not_fit(gpu):
    from porch_b200.decode_step import Decoder, Model

    model = Model(vocabulary=16, width=16, heads=2, kv_heads=1, head_dim=16, positions=64)
    with pytest.raises(ValueError, match="whole pages"):
        Decoder(model, 2, 8, page_size=8, prompt=np.arange(9))
    decoder = Decoder(model, 2, 4, slack=2, page_size=8, prompt=np.arange(8))
    for _ in range(6):
        decoder.step(np.arange(2))
    with pytest.raises(ValueError, match="room for 6 tokens"):
        decoder.step(np.arange(2))
