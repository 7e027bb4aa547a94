"""What the weights of 8-bit attention are rounded to: whole units of a tile's largest
weight x value scale, where a tile has 128 slots up to head size 128 and 64 above,
counted from where a sequence, or a shared prefix, begins."""

import numpy as np
import pytest

import int8_cache

U = 2.0**-24


def bounds(host, q, scale, tile):
    """(result, tolerance): int8_cache.Host.attend's, with the units of whole tiles."""
    out, tol, _, _ = host.attend(q, scale)
    group = q.shape[1] // host.heads
    for s, length in enumerate(host.lengths):
        k, v = (host.stored(x[s]) for x in (host.k, host.v))
        unit = int8_cache.quantise(host.v[s])[1].astype(np.float64)
        for h in range(q.shape[1]):
            x = q[s, h].astype(np.float64)
            logits = k[:, h // group] @ x * scale
            off = abs(scale) * (2.0**-23 * np.abs(x).max() * np.abs(k[:, h // group]).sum(1)
                                + 8 * U * (np.abs(k[:, h // group]) @ np.abs(x))).max() + 4 * U * np.abs(logits).max()
            p = np.exp(logits - logits.max())
            p /= p.sum()
            w = p * unit[:, h // group]
            # Units of at most 2^-21.99 of a tile's largest, each weight off by half a
            # one, and codes of up to 127.
            whole = sum(127 * 2.0**-22.9 * t.max() * len(t) for t in (w[i : i + tile] for i in range(0, length, tile)))
            rel = 2 * off + (2 * length + 128) * U
            tol[s, h] = rel * (p @ np.abs(v[:, h // group])) + whole + 1e-37
    return out, tol


@pytest.mark.gpu
@pytest.mark.parametrize("dim,tile", [(64, 128), (128, 128), (192, 64)])
@pytest.mark.parametrize("lengths", [[128], [127, 300, 64], [1000, 129]])
def test_halves_of_very_different_size(gpu, dim, tile, lengths):
    # In every 128 slots the first 64 have large values in some channels and zeros in
    # the others, and the last 64 small ones in all: what a channel of the second kind
    # gets is a sum of weights that are few units of their tile.
    rng = np.random.default_rng(dim + len(lengths))
    host = int8_cache.Host(rng, lengths, 2, dim, 64)
    for s, n in enumerate(lengths):
        at = np.arange(n) % 128
        host.v[s][at >= 64] *= np.float32(2.0**-16)
        host.v[s][at < 64, :, dim // 2 :] = 0
        host.k[s] *= np.float32(0.1)
    _, batch = host.build(gpu)
    q = rng.normal(0, 1, (len(lengths), 6, dim)).astype(np.float32)
    out, tol = bounds(host, q, dim**-0.5, tile)
    got = gpu.paged_attention(gpu.tensor(list(q.shape), q), batch).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()


@pytest.mark.gpu
def test_channels_below_an_outlier_of_the_query(gpu):
    # A query is whole units of 2^-22 of its largest channel: one channel of 2^12,
    # whose keys are 0, and others of about one, which decide.
    rng = np.random.default_rng(3)
    host = int8_cache.Host(rng, [200, 65], 2, 64, 16)
    for k in host.k:
        k[..., 9] = 0
    q = rng.normal(0, 1, (2, 4, 64)).astype(np.float32)
    q[..., 9] = 4096
    _, batch = host.build(gpu)
    out, tol = bounds(host, q, 1.0, 128)
    got = gpu.paged_attention(gpu.tensor(list(q.shape), q), batch, scale=1.0).cpu().reshape(q.shape)
    assert (np.abs(got - out) <= tol).all()
