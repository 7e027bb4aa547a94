"""Decoding with a small transformer on one GPU: the framework's matmul,
softmax and views around the decode-step operators (norms and rotation of query
and key heads, a paged cache, its scored attention, and eviction once a sequence
holds more than its budget).

  python -m porch_b200.decode_step [--steps N] [--sequences N] [--budget N] [--dtype f32|bf16]

Weights and prompts are synthetic (seeded). Prints the tokens of each sequence
and the time of a step.
"""

from __future__ import annotations

import argparse
import time

import numpy as np

from . import api


class Model:
    """`layers` blocks of attention and a two-layer MLP over `width` channels,
    without biases, between an embedding and an output matrix."""

    def __init__(self, vocabulary=512, width=256, layers=2, heads=8, kv_heads=2, head_dim=32, positions=4096, seed=1):
        self.vocabulary, self.width, self.layers = vocabulary, width, layers
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        rng = np.random.default_rng(seed)

        def weight(rows, columns):
            return rng.normal(0, rows**-0.5, (rows, columns)).astype(np.float32)

        inner = heads * head_dim
        self.embedding = rng.normal(0, 1, (vocabulary, width)).astype(np.float32)
        self.head = weight(width, vocabulary)
        self.blocks = [
            {
                "qkv": weight(width, inner + 2 * kv_heads * head_dim),
                "q_norm": rng.normal(1, 0.1, head_dim).astype(np.float32),
                "k_norm": rng.normal(1, 0.1, head_dim).astype(np.float32),
                "out": weight(inner, width),
                "up": weight(width, 2 * width),
                "down": weight(2 * width, width),
            }
            for _ in range(layers)
        ]
        angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(head_dim // 2) * 2 / head_dim)
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


class Decoder:
    """The model's weights on a GPU, a cache of each layer and the sequences."""

    def __init__(self, model: Model, sequences: int, budget: int, dtype: str = "bf16", slack: int = 8,
                 recent: int | None = None, sinks: int = 2, page_size: int = 16, device: int = 0):
        self.model, self.n, self.budget, self.slack = model, sequences, budget, slack
        self.recent = budget // 4 if recent is None else recent
        self.sinks, self.device = min(sinks, budget - self.recent), device
        self.blocks = [{k: self._tensor(v) for k, v in b.items()} for b in model.blocks]
        self.cos, self.sin = self._tensor(model.cos), self._tensor(model.sin)
        self.head = self._tensor(model.head)
        # A sequence holds at most budget + slack slots: its pages never change.
        width = -(-(budget + slack) // page_size)
        self.tables = np.arange(sequences * width, dtype=np.int32).reshape(sequences, width)
        self.caches = [api.KVCache(sequences * width, page_size, model.kv_heads, model.head_dim, dtype, device)
                       for _ in range(model.layers)]
        self.scores = [None] * model.layers
        self.positions = [None] * model.layers
        self.length = 0  # slots in use, the same for every sequence
        self.seen = 0  # tokens so far

    def _tensor(self, x: np.ndarray) -> api.Tensor:
        return api.tensor(list(x.shape), x, self.device)

    def step(self, tokens: np.ndarray) -> np.ndarray:
        """Takes one token of each sequence; the next ones' probabilities."""
        m, n = self.model, self.n
        if self.seen >= len(m.cos):  # the operator would turn by NaN
            raise ValueError(f"the model has angles for {len(m.cos)} positions")
        self.length += 1
        batch = self.caches[0].batch(self.tables, [self.length] * n, newest=[self.seen] * n)
        at = api.full([n], float(self.seen), self.device)
        self.seen += 1
        x = self._tensor(m.embedding[tokens])
        inner, kv = m.heads * m.head_dim, m.kv_heads * m.head_dim
        evict = self.length == self.budget + self.slack
        for i, b in enumerate(self.blocks):
            here = batch.on(self.caches[i])
            # A token's queries, keys and values side by side, read in place as heads.
            qkv = api.materialize(api.reshape(api.matmul(x, b["qkv"]), [n, m.heads + 2 * m.kv_heads, m.head_dim]))
            q, k, v = (api.materialize(qkv[api.all, lo // m.head_dim:hi // m.head_dim, api.all])
                       for lo, hi in ((0, inner), (inner, inner + kv), (inner + kv, inner + 2 * kv)))
            q, k = api.qk_norm_rope(q, k, b["q_norm"], b["k_norm"], self.cos, self.sin, at)
            here.append(k, v)
            a, self.scores[i] = api.paged_attention_scored(q, here, self.scores[i])
            if evict:
                self.scores[i], self.positions[i] = api.cache_evict(
                    here, self.scores[i], self.positions[i], budget=self.budget, recent=self.recent, sinks=self.sinks)
            x = api.materialize(x + api.matmul(api.reshape(a, [n, inner]), b["out"]))
            x = api.materialize(x + api.matmul(api.relu(api.matmul(x, b["up"])), b["down"]))
        if evict:
            self.length = self.budget
        return api.materialize(api.softmax(api.matmul(x, self.head), 1)).cpu().reshape(n, m.vocabulary)


def main(argv: list[str] | None = None) -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--sequences", type=int, default=4)
    parser.add_argument("--budget", type=int, default=64)
    parser.add_argument("--dtype", choices=("f32", "bf16"), default="bf16")
    a = parser.parse_args(argv)
    model = Model(positions=max(4096, a.steps))
    decoder = Decoder(model, a.sequences, a.budget, a.dtype)
    tokens = np.arange(a.sequences) % model.vocabulary
    said, times = [tokens], []
    for _ in range(a.steps):
        began = time.perf_counter()
        tokens = decoder.step(tokens).argmax(1)
        times.append(time.perf_counter() - began)
        said.append(tokens)
    for s, row in enumerate(np.stack(said, 1)):
        print(f"sequence {s}: {' '.join(map(str, row[:24]))} ...")
    print(f"{a.steps} steps of {a.sequences} sequences, {decoder.length} slots each at the end: "
          f"{1e3 * float(np.median(times)):.2f} ms a step")


if __name__ == "__main__":
    main()
