"""The attention keeps the 24 bits of its queries and weights, whatever the
cache's type. Worst-case bounds (paged.Host.attend) are far above what an operand
cut to 16 bits loses, so the root mean square over many outputs is bounded here,
in units of u = 2^-24 relative to the sum of weight x |value|.

Five slots, one channel of the query in use, logits of at most 2. What each step
adds, as a root mean square: a logit's products are exact against a bfloat16
cache; its two sums on the tensor core are cut (2 u at most, 1.2 u each), three
more operations round (0.6 u each): 1.9 u of the logit, of size 0.9 on average,
so 1.7 u of a weight. exp2's error is at most 4 u, 2.3 u on average. Weights of
five slots average those to about 0.55 of 2.9 u: 1.6 u. The weighted sum is cut
and rounded, the sum of the weights, its reciprocal and the product round: 2 u.
In all 2.6 u; the bound is 4 u. Two tf32 terms leave up to 8 u of each
operand against a float32 cache, cut toward zero: the bound is 6 u.

That the bounds see a term that is missing is checked on the same arithmetic in
numpy: 12 u and more against a bfloat16 cache, a thousand against a float32 one.
"""

import numpy as np
import pytest

import paged

U = paged.U
BOUND = {"bf16": 4 * U, "f32": 6 * U}
SEQUENCES, HEADS, SLOTS = 64, 2, 5


def inputs(dim, group, dtype, seed):
    rng = np.random.default_rng(seed)
    host = paged.Host(rng, [SLOTS] * SEQUENCES, HEADS, dim, 8, dtype)
    host.k = [rng.uniform(-1, 1, (SLOTS, HEADS, dim)).astype(np.float32) for _ in range(SEQUENCES)]
    q = np.zeros((SEQUENCES, HEADS * group, dim), np.float32)
    q[..., rng.integers(0, dim)] = rng.uniform(1, 2, q.shape[:2])
    return host, q


def rows(host, q):
    """q [R, dim], k and v [R, slots, dim] of every query head, as stored."""
    group = q.shape[1] // HEADS
    k, v = (np.repeat(host.stored(np.stack(x)).transpose(0, 2, 1, 3), group, 1).reshape(-1, SLOTS, host.dim)
            for x in (host.k, host.v))
    return q.reshape(-1, host.dim), k, v


def error(out, q, k, v):
    logits = np.einsum("rd,rnd->rn", q.astype(np.float64), k.astype(np.float64))
    assert np.abs(logits).max() <= 2
    p = np.exp(logits)
    p /= p.sum(1, keepdims=True)
    want, size = (np.einsum("rn,rnd->rd", p, x) for x in (v.astype(np.float64), np.abs(v.astype(np.float64))))
    return np.sqrt((((out - want) / size) ** 2).mean())


def cut(x):
    """To float32, toward zero."""
    y = x.astype(np.float32)
    return np.where(np.abs(y.astype(np.float64)) > np.abs(x), np.nextafter(y, np.float32(0)), y)


def split(x, count, dtype):
    out = []
    for i in range(count):
        if dtype == "bf16":
            h = paged.bf16(x)
        else:  # rounded, then what the tensor core reads of the rest
            h = ((x.view(np.uint32) + np.uint32(0 if i else 0x1000)) & np.uint32(0xFFFFE000)).view(np.float32)
        out.append(h.astype(np.float64))
        x = x - h
    return out


def product(a, b, terms, dtype, spec):
    """a (float32) times b (the cache's type), summed, as the kernel does it."""
    full = 3 if dtype == "bf16" else 2
    a = split(a, terms, dtype) + [np.zeros(a.shape)] * (full - terms)
    b = [b.astype(np.float64)] if dtype == "bf16" else split(b, 2, dtype)
    small = [cut(np.einsum(spec, x, b[0])) for x in a[1:]] + [cut(np.einsum(spec, a[0], y)) for y in b[1:]]
    return sum(small[::-1], np.float32(0)) + cut(np.einsum(spec, a[0], b[0]))


def emulated(q, k, v, dtype, query_terms, weight_terms):
    s = product(q, k, query_terms, dtype, "rd,rnd->rn") * np.float32(1.4426950408889634)
    p = np.exp2((s - s.max(1, keepdims=True)).astype(np.float64)).astype(np.float32)
    return product(p, v, weight_terms, dtype, "rn,rnd->rd") * (np.float32(1) / p.sum(1, dtype=np.float32))[:, None]


@pytest.mark.parametrize("dtype,full", [("bf16", 3), ("f32", 2)])
@pytest.mark.parametrize("dim", [8, 128])
def test_the_bound_sees_a_missing_term(dim, dtype, full):
    q, k, v = rows(*inputs(dim, 4, dtype, dim))
    assert error(emulated(q, k, v, dtype, full, full), q, k, v) <= BOUND[dtype]
    assert error(emulated(q, k, v, dtype, full - 1, full), q, k, v) > 2 * BOUND[dtype]
    assert error(emulated(q, k, v, dtype, full, full - 1), q, k, v) > 2 * BOUND[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,group", [(8, 1), (24, 4), (64, 4), (80, 3), (128, 4), (256, 2), (64, 12), (128, 16), (72, 20)])
def test_every_bit_of_queries_and_weights_counts(gpu, dim, group, dtype):
    host, q = inputs(dim, group, dtype, dim + group)
    _, batch = host.build(gpu)
    t = gpu.tensor(list(q.shape), q)
    for out in (gpu.paged_attention(t, batch, scale=1.0), gpu.paged_attention_scored(t, batch, scale=1.0)[0]):
        assert error(out.cpu().reshape(-1, dim), *rows(host, q)) <= BOUND[dtype]
