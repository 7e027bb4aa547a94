"""Log probabilities of rows that are long for each thread that sums them: additions
that follow each other round the same way where terms are alike, so their number is
what bounds the error."""

import numpy as np
import pytest

from test_token_logprobs import check_forward, make

U = 2.0**-24


class Host:
    """What is on the host already, as a tensor hands it out."""

    def __init__(self, values):
        self.values = values

    def cpu(self):
        return self.values


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(300, 1 << 18), (600, (1 << 18) + 1), (310, 131072), (310, 131069), (4, 1 << 22)])
def test_against_the_definition(gpu, rows, vocab):
    # About one and two blocks of 32 rounds a thread, and one CTA a row or several.
    rng = np.random.default_rng(vocab)
    # Four rows, again and again: a row's place in 16 bytes decides which logits a
    # thread has, and comes again after four rows whatever their length.
    few, tokens = make(rng, 4, vocab)
    at = np.arange(rows) % 4
    x, t = gpu.tensor([rows, vocab], few[at]), gpu.tensor([rows], tokens[at])
    for top in (0, 5):
        got = [g.cpu().reshape(rows, -1) for g in gpu.token_logprobs(x, t, top=top)]
        for g in got:  # alike rows give the same, to the bit
            assert np.array_equal(g, g[at])

        check_forward(few[:rows], tokens[:rows], [Host(g[:4].squeeze()) for g in got], top)


@pytest.mark.gpu
def test_terms_that_are_alike(gpu):
    # Every thread begins with four logits of 0; all others are -0.75, and each round
    # adds 16 e^-0.75. In float32 one after the other, 1024 of them come out 244 u off.
    rows, vocab = 297, 1 << 22  # a CTA of 256 threads for each row
    x = gpu.materialize(gpu.concat(gpu.full([rows, 1024], 0.0), gpu.full([rows, vocab - 1024], -0.75), 1))
    tokens = np.zeros(rows, np.float32)
    tokens[1::2] = vocab - 7
    said, entropy, norm = gpu.token_logprobs(x, gpu.tensor([rows], tokens))
    s = 1024 + (vocab - 1024) * np.exp(-0.75)
    # A term: 2^-22 by ex2 and 2 u by its argument; 9 additions of a round, 32 of a
    # block, 32 blocks, 12 joins of threads, of which each rounds once.
    off = (4 + 2 + 9 + 32 + 32 + 12 + 1) * U
    assert (np.abs(norm.cpu().reshape(rows, 2)[:, 1] / s - 1) <= off).all()
    want = np.where(tokens == 0, 0.0, -0.75) - np.log(s)
    tol = off + 2 * U * np.log(s) + U * np.abs(want)  # the logarithm within 2 u of itself, the difference rounded
    assert (np.abs(said.cpu() - want) <= tol).all()
    mean = 0.75 * (s - 1024) / s
    assert (np.abs(entropy.cpu() - (np.log(s) + mean)) <= tol + 3 * off * mean + 4 * U).all()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [131072, 1 << 18])
def test_rows_that_are_not_finite(gpu, vocab):
    rows = 300
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 1, (rows, vocab)).astype(np.float32)
    x[0, 5], x[1, vocab - 9], x[2, vocab // 2], x[3, 3] = np.nan, np.nan, np.inf, np.inf
    x[4] = -np.inf
    x[5, 1:] = -np.inf
    t = gpu.tensor([rows], np.zeros(rows, np.float32))
    said, entropy, norm = (g.cpu() for g in gpu.token_logprobs(gpu.tensor([rows, vocab], x), t))
    assert np.isnan(said[:5]).all() and np.isnan(entropy[:5]).all() and np.isnan(norm.reshape(rows, 2)[:5, 1]).all()
    assert said[5] == 0 and entropy[5] == 0 and np.isfinite(said[5:]).all() and np.isfinite(entropy[5:]).all()
