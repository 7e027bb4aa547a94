"""Decoding with a small transformer on one GPU: the framework's matmul,
softmax and views around the decode-step operators (norms and rotation of query
and key heads, a paged cache, its scored attention, and eviction once a sequence
holds more than its budget). With a prompt, its slots are shared by all sequences
and worked through once for them (and nothing is evicted). With alternatives, what
comes back to the host are the likeliest tokens with their log probabilities
instead of every token's probability.

  python -m porch_b200.decode_step [--steps N] [--sequences N] [--budget N] [--dtype f32|bf16|int8]
                                   [--prompt N] [--top N]

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
                 recent: int | None = None, sinks: int = 2, page_size: int = 16, device: int = 0,
                 prompt: np.ndarray | None = None):
        self.model, self.n, self.budget, self.slack = model, sequences, budget, slack
        self.recent = budget // 4 if recent is None else recent
        self.sinks, self.device = min(sinks, budget - self.recent), device
        self.blocks = [{k: self._tensor(v) for k, v in b.items()} for b in model.blocks]
        self.cos, self.sin = self._tensor(model.cos), self._tensor(model.sin)
        self.head = self._tensor(model.head)
        # A sequence holds at most budget + slack slots of its own: its pages never
        # change. A prompt's pages come first in each of their tables.
        self.shared = 0 if prompt is None else len(prompt)
        if self.shared % page_size:
            raise ValueError(f"a prompt must be whole pages of {page_size} tokens")
        width, before = -(-(budget + slack) // page_size), self.shared // page_size
        own = before + np.arange(sequences * width, dtype=np.int32).reshape(sequences, width)
        first = np.broadcast_to(np.arange(before, dtype=np.int32), (sequences, before))
        self.tables = np.concatenate([first, own], 1)
        self.caches = [api.KVCache(before + sequences * width, page_size, model.kv_heads, model.head_dim, dtype, device)
                       for _ in range(model.layers)]
        self.scores = [None] * model.layers
        self.positions = [None] * model.layers
        self.length = 0  # own slots in use, the same for every sequence
        self.seen = 0  # tokens so far
        for token in () if prompt is None else prompt:  # once, by one sequence
            self._logits(np.array([token]), 1)
            self.length = 0

    def _tensor(self, x: np.ndarray) -> api.Tensor:
        return api.tensor(list(x.shape), x, self.device)

    def step(self, tokens: np.ndarray) -> np.ndarray:
        """Takes one token of each sequence; the next ones' probabilities."""
        logits = self._logits(tokens, self.n)
        return api.materialize(api.softmax(logits, 1)).cpu().reshape(self.n, self.model.vocabulary)

    def step_top(self, tokens: np.ndarray, top: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """Takes one token of each sequence; the next ones' likeliest tokens,
        their log probabilities, and the entropies."""
        none = api.full([self.n], -1.0, self.device)  # no token's own is asked for
        _, entropy, _, said, best = api.token_logprobs(self._logits(tokens, self.n), none, top=top)
        return best.cpu().reshape(self.n, top).astype(np.int64), said.cpu().reshape(self.n, top), entropy.cpu()

    def _logits(self, tokens: np.ndarray, n: int):
        m = self.model
        if self.seen >= len(m.cos):  # the operator would turn by NaN
            raise ValueError(f"the model has angles for {len(m.cos)} positions")
        self.length += 1
        if self.shared:
            if self.length > self.budget + self.slack:
                raise ValueError(f"a sequence has room for {self.budget + self.slack} tokens behind its prompt")
            prefix = min(self.seen, self.shared)  # while it goes in, itself
            batch = self.caches[0].batch(self.tables[:n], [self.seen + 1] * n,
                                         prefix=[prefix] * n if prefix == self.shared else None)
        else:
            batch = self.caches[0].batch(self.tables, [self.length] * n, newest=[self.seen] * n)
        at = api.full([n], float(self.seen), self.device)
        self.seen += 1
        x = self._tensor(m.embedding[tokens])
        inner, kv = m.heads * m.head_dim, m.kv_heads * m.head_dim
        evict = not self.shared and self.length == self.budget + self.slack
        for i, b in enumerate(self.blocks):
            here = batch.on(self.caches[i])
            # A token's queries, keys and values side by side, read in place as heads.
            qkv = api.materialize(api.reshape(api.matmul(x, b["qkv"]), [n, m.heads + 2 * m.kv_heads, m.head_dim]))
            q, k, v = (api.materialize(qkv[api.all, lo // m.head_dim:hi // m.head_dim, api.all])
                       for lo, hi in ((0, inner), (inner, inner + kv), (inner + kv, inner + 2 * kv)))
            q, k = api.qk_norm_rope(q, k, b["q_norm"], b["k_norm"], self.cos, self.sin, at)
            here.append(k, v)
            if self.shared:
                a = api.paged_attention(q, here)
            else:
                a, self.scores[i] = api.paged_attention_scored(q, here, self.scores[i])
            if evict:
                self.scores[i], self.positions[i] = api.cache_evict(
                    here, self.scores[i], self.positions[i], budget=self.budget, recent=self.recent, sinks=self.sinks)
            x = api.materialize(x + api.matmul(api.reshape(a, [n, inner]), b["out"]))
            x = api.materialize(x + api.matmul(api.relu(api.matmul(x, b["up"])), b["down"]))
        if evict:
            self.length = self.budget
        return api.materialize(api.matmul(x, self.head))


def main(argv: list[str] | None = None) -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--sequences", type=int, default=4)
    parser.add_argument("--budget", type=int, default=64)
    parser.add_argument("--dtype", choices=("f32", "bf16", "int8"), default="bf16")
    parser.add_argument("--prompt", type=int, default=0, help="tokens of a prompt that all sequences share, a multiple of 16")
    parser.add_argument("--top", type=int, default=0, help="alternatives to report for each sequence's last token")
    a = parser.parse_args(argv)
    model = Model(positions=max(4096, a.prompt + a.steps))
    if a.prompt:
        prompt = np.arange(a.prompt) * 7 % model.vocabulary
        decoder = Decoder(model, a.sequences, max(a.budget, a.steps), a.dtype, prompt=prompt)
    else:
        decoder = Decoder(model, a.sequences, a.budget, a.dtype)
    tokens = np.arange(a.sequences) % model.vocabulary
    said, times = [tokens], []
    for _ in range(a.steps):
        began = time.perf_counter()
        if a.top:
            best, likely, entropy = decoder.step_top(tokens, a.top)
            tokens = best[:, 0]
        else:
            tokens = decoder.step(tokens).argmax(1)
        times.append(time.perf_counter() - began)
        said.append(tokens)
    for s, row in enumerate(np.stack(said, 1)):
        print(f"sequence {s}: {' '.join(map(str, row[:24]))} ...")
        if a.top and a.steps:
            print(f"  the last of entropy {entropy[s]:.3f}: "
                  + ", ".join(f"{t} {p:.3f}" for t, p in zip(best[s], likely[s])))
    print(f"{a.steps} steps of {a.sequences} sequences, {decoder.length} slots each at the end: "
          f"{1e3 * float(np.median(times)):.2f} ms a step")


if __name__ == "__main__":
    main()
