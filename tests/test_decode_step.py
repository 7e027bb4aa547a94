"""The decoding example against the same model in 64 bits."""

import numpy as np
import pytest

import fake_driver
import paged


def norm(x, w, c, s):
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w
    h = y.shape[-1] // 2
    a, b = y[..., :h], y[..., h:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


class Plain:
    """Decoder's step, sequence by sequence. Which slots are evicted is taken
    over from the device's scores, so that both sides keep the same ones."""

    def __init__(self, model, n, budget, slack, recent, sinks, dtype):
        self.m, self.n, self.budget, self.slack, self.recent, self.sinks = model, n, budget, slack, recent, sinks
        self.rounded = paged.bf16 if dtype == "bf16" else (lambda x: np.float32(x))
        shape = (model.layers, n, model.kv_heads, 0, model.head_dim)
        self.k, self.v = np.zeros(shape), np.zeros(shape)
        self.places, self.seen = [None] * model.layers, 0

    def step(self, tokens, device_scores):
        m, n = self.m, self.n
        x = m.embedding[tokens].astype(np.float64)
        c, s = m.cos[self.seen].astype(np.float64), m.sin[self.seen].astype(np.float64)
        new_k, new_v = [], []
        slots = self.k.shape[3] + 1
        for i, b in enumerate(m.blocks):
            b = {k: v.astype(np.float64) for k, v in b.items()}
            heads = (x @ b["qkv"]).reshape(n, -1, m.head_dim)
            q = norm(heads[:, : m.heads], b["q_norm"], c, s)
            k = norm(heads[:, m.heads : m.heads + m.kv_heads], b["k_norm"], c, s)
            v = heads[:, m.heads + m.kv_heads :]
            k, v = (self.rounded(y.astype(np.float32)).astype(np.float64)[:, :, None] for y in (k, v))
            keys, values = np.concatenate([self.k[i], k], 2), np.concatenate([self.v[i], v], 2)
            logits = np.einsum("nhgd,nhsd->nhgs", q.reshape(n, m.kv_heads, -1, m.head_dim), keys) * m.head_dim**-0.5
            p = np.exp(logits - logits.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            a = np.einsum("nhgs,nhsd->nhgd", p, values).reshape(n, -1)
            x = x + a @ b["out"]
            x = x + np.maximum(x @ b["up"], 0) @ b["down"]
            if slots == self.budget + self.slack:
                source, _, self.places[i] = paged.evict([slots] * n, [self.seen] * n, device_scores(i), self.places[i],
                                                        self.budget, self.recent, self.sinks)
                keys, values = (np.take_along_axis(y, source[..., None], 2) for y in (keys, values))
            new_k.append(keys)
            new_v.append(values)
        self.k, self.v = np.stack(new_k), np.stack(new_v)
        self.seen += 1
        logits = x @ m.head.astype(np.float64)
        p = np.exp(logits - logits.max(1, keepdims=True))
        return p / p.sum(1, keepdims=True)


def test_positions_end_with_the_models_table(api, tmp_path):
    # Over the driver's stand-in: a step past the table is an error, not NaN
    # probabilities, and the command's model has a table for all its steps.
    out, _ = fake_driver.run("""
from porch_b200 import decode_step
d = decode_step.Decoder(decode_step.Model(vocabulary=16, width=16, heads=2, kv_heads=1, head_dim=8, positions=5), 2, 8)
try:
    for step in range(9):
        d.step(np.arange(2))
except ValueError as e:
    print(step, e)
decode_step.Decoder = lambda model, *a: exit(len(model.cos) != 5000)
decode_step.main(["--steps", "5000"])
""", tmp_path)
    assert out.split("\n")[0] == "5 the model has angles for 5 positions"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_example_decodes_as_the_formulas_do(gpu, dtype, monkeypatch):
    from porch_b200.decode_step import Decoder, Model

    model = Model(vocabulary=64, width=64, heads=4, kv_heads=2, head_dim=16, positions=64)
    budget, slack = 12, 4
    decoder = Decoder(model, 3, budget, dtype, slack=slack, recent=4, sinks=1, page_size=8)
    plain = Plain(model, 3, budget, slack, 4, 1, dtype)
    ranked = []
    evict = gpu.cache_evict
    monkeypatch.setattr(gpu, "cache_evict", lambda batch, scores, *a, **k: (
        ranked.append(scores.cpu().reshape(scores.shape())), evict(batch, scores, *a, **k))[1])
    rng = np.random.default_rng(5)
    for step in range(30):
        tokens = rng.integers(0, 64, 3)
        ranked.clear()
        got = decoder.step(tokens)
        want = plain.step(tokens, lambda i: ranked[i])
        # float32 throughout: two layers of products of up to 128 terms and a
        # softmax of logits of at most a few tens, each within 2^-24 of its
        # terms' sizes per operation: 1e-4 is some hundred times that. A
        # bfloat16 cache rounds keys and values that may differ by a float32
        # rounding to neighbouring bfloat16 values, 2^-8 apart.
        assert np.abs(got - want).max() <= (1e-4 if dtype == "f32" else 0.02) * want.max()
        assert abs(got.sum(1) - 1).max() < 1e-5
    assert decoder.length < budget + slack and decoder.seen == 30
    assert plain.k.shape[3] == decoder.length


@pytest.mark.gpu
def test_the_command_runs(gpu, capsys):
    from porch_b200 import decode_step

    decode_step.main(["--steps", "20", "--sequences", "2", "--budget", "8", "--dtype", "f32"])
    out = capsys.readouterr().out
    assert "sequence 1:" in out and "ms a step" in out
