"""An int8 cache in numpy, for the tests: rows as codes and a scale, and
attention over them in 64 bits with tolerances for what the kernel rounds."""

import numpy as np

import paged

U = paged.U


def quantise(x):
    """(codes, scales) of rows of float32 by the definition: 127 x / top rounded
    to nearest, ties to even, in real arithmetic. 127 x, (n + 1/2) top are exact
    in 64 bits, so the rounding is corrected by comparing them."""
    x = np.asarray(x, np.float32).astype(np.float64)
    top = np.abs(x).max(-1, keepdims=True)
    good = np.isfinite(top) & (top >= 2.0**-96)
    unit = np.where(good, top, 1.0)
    a = 127 * np.where(good, np.abs(x), 0.0)
    n = np.floor(a / unit)
    n -= a < n * unit
    n += a >= (n + 1) * unit
    half = (n + 0.5) * unit
    n += (a > half) | ((a == half) & (n % 2 == 1))
    codes = np.where(good, np.copysign(n, x), 0).astype(np.int8)
    with np.errstate(invalid="ignore", over="ignore"):
        scale = np.where(good, (top.astype(np.float32) / np.float32(127)), np.where(np.isfinite(top), 0, np.nan))
    return codes, scale[..., 0].astype(np.float32)


class Host(paged.Host):
    def __init__(self, rng, lengths, heads, dim, page, dtype="int8", spare=2):
        super().__init__(rng, lengths, heads, dim, page, dtype, spare)

    def stored(self, x):
        if self.dtype != "int8":
            return super().stored(x)
        codes, scale = quantise(x)
        return codes.astype(np.float64) * scale[..., None].astype(np.float64)

    def attend(self, q, scale, scores=None):
        """paged.Host.attend, with what eight bits add. A query is a whole number
        of units of at most 2^-22 of its head's largest size, off by half a unit;
        the sums of integers are exact, and eight roundings follow. A weight
        times its value's scale is a whole number of units of at most 2^-21.99
        of the largest in its 64 slots, off by half a unit and by the
        exponential's error, before it meets codes of up to 127."""
        if self.dtype != "int8":
            return super().attend(q, scale, scores)
        n, heads, dim = q.shape
        group = heads // self.heads
        longest = max(self.lengths)
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        new, new_tol = np.zeros((n, self.heads, longest)), np.zeros((n, self.heads, longest))
        for s, length in enumerate(self.lengths):
            if length == 0:
                continue
            k, v = (self.stored(x[s]) for x in (self.k, self.v))
            unit_v = quantise(self.v[s])[1].astype(np.float64)
            for h in range(heads):
                kv = h // group
                x = q[s, h].astype(np.float64)
                logits = k[:, kv] @ x * scale
                off = abs(scale) * (2.0**-23 * np.abs(x).max() * np.abs(k[:, kv]).sum(1)
                                    + 8 * U * (np.abs(k[:, kv]) @ np.abs(x))).max() + 4 * U * np.abs(logits).max()
                p = np.exp(logits - logits.max())
                p /= p.sum()
                rel = 2 * off + (2 * length + 128) * U
                out[s, h] = p @ v[:, kv]
                w = p * unit_v[:, kv]
                tiles = [w[i : i + 64] for i in range(0, length, 64)]
                whole = sum(127 * 2.0**-22.9 * t.max() * len(t) for t in tiles)
                tol[s, h] = rel * (p @ np.abs(v[:, kv])) + whole + 1e-37
                new[s, kv, :length] += p
                new_tol[s, kv, :length] += rel * p + 1e-37
            if scores is not None:
                m = min(length, scores.shape[2])
                new[s, :, :m] += scores[s, :, :m]
                # A score takes the weights of its `group` heads one after the
                # other: as many roundings of a sum that only grows.
                new_tol[s] += (group + 4) * U * np.abs(new[s])
        return out, tol, new, new_tol
