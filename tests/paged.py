"""A paged cache in numpy and its operators in 64 bits, for the tests."""

import numpy as np

U = 2.0**-24


def bf16(x):
    """Rounded to nearest even bfloat16, as float32; NaN stays NaN."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), x, r)


class Host:
    """Sequences over pages in random order; k[s], v[s]: [slots, heads, dim]."""

    def __init__(self, rng, lengths, heads, dim, page, dtype, spare=2):
        self.lengths, self.heads, self.dim, self.page, self.dtype = list(lengths), heads, dim, page, dtype
        counts = [-(-n // page) for n in lengths]
        self.pages = sum(counts) + spare
        order = rng.permutation(self.pages)
        self.tables = np.full((len(lengths), max(1, max(counts))), -1, dtype=np.int32)
        at = 0
        for i, c in enumerate(counts):
            self.tables[i, :c] = order[at : at + c]
            at += c
        self.k = [rng.normal(0, 1, (n, heads, dim)).astype(np.float32) for n in lengths]
        self.v = [rng.normal(0, 1, (n, heads, dim)).astype(np.float32) for n in lengths]

    def stored(self, x):
        return bf16(x) if self.dtype == "bf16" else x

    def build(self, api, newest=None):
        """The cache with every slot that no sequence uses NaN, and the batch."""
        cache = api.KVCache(self.pages, self.page, self.heads, self.dim, dtype=self.dtype)
        total = self.pages * self.page
        everything = cache.batch(np.arange(self.pages)[None], [total], appended=[total])
        nan = api.tensor([total, self.heads, self.dim], np.full(total * self.heads * self.dim, np.nan, np.float32))
        everything.append(nan, nan)
        batch = cache.batch(self.tables, self.lengths, appended=self.lengths, newest=newest)
        rows = [sum(self.lengths), self.heads, self.dim]
        batch.append(api.tensor(rows, np.concatenate(self.k)), api.tensor(rows, np.concatenate(self.v)))
        return cache, batch

    def attend(self, q, scale, scores=None):
        """(out, its tolerance, new scores, their tolerance). A logit is a sum
        of dim products, in any order, within (2 dim + 64) u of the sum of
        their sizes; that is an error of each weight's exponent, and so of the
        weights' ratios. The weighted sum of n rows, in any order and with
        each step rounded or cut, is within (2 n + 128) u more, relative to
        the sum of weight x |v|."""
        n, heads, dim = q.shape
        group = heads // self.heads
        longest = max(self.lengths)
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        new, new_tol = np.zeros((n, self.heads, longest)), np.zeros((n, self.heads, longest))
        for s, length in enumerate(self.lengths):
            if length == 0:
                continue
            k, v = (self.stored(x[s]).astype(np.float64) for x in (self.k, self.v))
            for h in range(heads):
                kv = h // group
                x = q[s, h].astype(np.float64)
                logits = k[:, kv] @ x * scale
                off = (2 * dim + 64) * U * (np.abs(k[:, kv]) @ np.abs(x)).max() * abs(scale)
                p = np.exp(logits - logits.max())
                p /= p.sum()
                rel = 2 * off + (2 * length + 128) * U
                out[s, h] = p @ v[:, kv]
                tol[s, h] = rel * (p @ np.abs(v[:, kv])) + 1e-37
                new[s, kv, :length] += p
                new_tol[s, kv, :length] += rel * p + 1e-37
            if scores is not None:
                m = min(length, scores.shape[2])
                new[s, :, :m] += scores[s, :, :m]
                new_tol[s] += 4 * U * np.abs(new[s])
        return out, tol, new, new_tol


def evict(lengths, newest, scores, places, budget, recent, sinks):
    """(source slot of each kept place or -1, scores, positions), by the definition."""
    n, heads, _ = scores.shape
    source = np.full((n, heads, budget), -1)
    out = np.zeros((n, heads, budget), np.float32)
    where = np.full((n, heads, budget), -1.0, np.float32)
    for s, length in enumerate(lengths):
        for h in range(heads):
            place = newest[s] - (length - 1 - np.arange(length))
            if places is not None:
                m = min(length, places.shape[2])
                given = places[s, h, :m]
                place[:m] = np.where(given >= 0, given, place[:m])
            score = np.zeros(length, np.float32)
            m = min(length, scores.shape[2])
            score[:m] = scores[s, h, :m]
            rank = np.where(np.isnan(score), -np.inf, score).astype(np.float64)
            safe = (place > newest[s] - recent) | (place < sinks)
            order = sorted(range(length), key=lambda i: (not safe[i], 0 if safe[i] else -rank[i], i))[:budget]
            kept = np.zeros(length, bool)
            kept[order] = True
            src = np.arange(min(length, budget))
            src[~kept[:budget]] = np.flatnonzero(kept[budget:]) + budget
            source[s, h, : len(src)] = src
            out[s, h, : len(src)] = score[src]
            where[s, h, : len(src)] = place[src]
    return source, out, where
