"""q4_cuda_route_balance: how many roundings its results have.  Inputs with which every step but the looked-at one is exact."""
import numpy as np
import pytest

from test_balance_gpu import EPS, call, inputs, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 7, 41, 47, 55, 61, 82, 83, 107, 1000, 3001])
def test_equal_logits_give_the_fractions_themselves(dev, n):
    """64 equal logits: probabilities of 1/64, whose sums are exact; all picks on expert 0: f is 1, the mean 1/64, the loss 64 * 1/64, whatever
    n is.  A mean that is a product with 1/n is not, for most of these n."""
    e = 64
    logits, ids = np.zeros((n, e), np.float32), np.zeros((n, 1), np.int32)
    counts, prob, loss, grad = call(dev, logits, ids, None, 1.0)
    assert counts[0] == n and (counts[1:] == 0).all()
    assert (prob == np.float32(1 / 64)).all() and loss == 1.0
    # a gradient has one division, 64 / n, and one product that is not exact: 63/64 or 1/64 of it
    want = plain(logits, ids, None, 1.0)[3]
    assert (np.abs(grad - want) <= 2.01 * EPS * np.abs(want)).all()


@pytest.mark.parametrize("n,k", [(3, 7), (41, 3), (1000, 10), (4099, 6)])
def test_shares_are_quotients(dev, n, k):
    """One expert takes all of the probability: its mean is 1 and the loss e f, rounded once for f = counts / (n k) and then exact (e = 32)."""
    rng = np.random.default_rng(n)
    e = 32
    logits = np.full((n, e), -np.inf, np.float32)
    logits[:, 5] = rng.standard_normal(n)
    ids = rng.integers(0, e, (n, k)).astype(np.int32)
    counts, prob, loss, _ = call(dev, logits, ids, None, 1.0)
    assert prob[5] == 1.0 and (np.delete(prob, 5) == 0).all()
    assert loss == np.float32(e) * (np.float32(counts[5]) / np.float32(n * k))


@pytest.mark.parametrize("t,e,k", [(64, 512, 10), (777, 64, 2), (20000, 96, 3), (20000, 600, 4), (300000, 40, 2), (2 ** 23 - 1, 2, 1)])
def test_means_of_many_tokens(dev, t, e, k):
    """Half steps of a mean: a warp adds up its rows one by one.  A cluster is 8 CTAs of 32 warps (24 of more than 128 experts, 16 of more
    than 512); there are as many as the tokens need, all of up to 8 at least on any B200.  Then come its CTA's other half and 16 warps, 8
    CTAs, 148 / 8 clusters and the division.  A probability: as in test_balance_gpu.check."""
    rng = np.random.default_rng(t)
    logits, ids, valid = inputs(rng, t, e, k)
    counts, prob, loss, grad = call(dev, logits, ids, valid, 0.01, 0.5)
    coef = float(np.float32(0.01))
    want = plain(logits, ids, valid, coef, 0.5)
    warps = 32 if e <= 128 else 24 if e <= 512 else 16
    per_cluster = 8 * warps
    rows = -(-t // (per_cluster * min(-(-t // per_cluster), 8)))
    live = logits[valid != 0].astype(np.float64)
    spread = (live.max(axis=1) - live.min(axis=1)).max()
    per_p = (1.34 * spread + e / 32 + 16) * EPS
    mean = (rows + 1 + 16 + 8 + 19 + 1) * EPS
    assert (counts == want[0]).all()
    assert (np.abs(prob - want[1]) <= (per_p + mean) * want[1]).all()
    assert abs(loss - want[2]) <= (per_p + mean + (e / 32 + 20) * EPS) * want[2]
    size = 0.5 * coef * e / len(live) * want[4] * (want[5] + (want[4] @ want[5])[:, None])
    assert (np.abs(grad - want[3]) <= (2 * per_p + (e / 32 + 16) * EPS) * size + 1e-44).all()
    assert dev.lib.q4_cuda_device_error() == 0
