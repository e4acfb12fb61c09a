"""The device sampler where a mask or a bias of -inf bars tokens: what it draws
at given coins. A coin is reached by its seed: the generator's steps
(xorshift64*, model/sampler.c:44-49) run backwards."""
import numpy as np
import pytest

from conftest import MODEL_CACHE

import krafla_b200 as kb

pytestmark = pytest.mark.gpu

MASK64 = (1 << 64) - 1


def seed_of(coin24):
    """The seed whose first draw is coin24 / 2^24."""
    x = (coin24 << 40 | 0x123456789) * pow(0x2545F4914F6CDD1D, -1, 1 << 64) & MASK64

    def undo(y, shift):
        x = y
        for _ in range(64 // abs(shift) + 1):
            x = y ^ (x >> shift if shift > 0 else (x << -shift) & MASK64)
        return x

    return undo(undo(undo(x, 27), -25), 12)


def draw_of(seed):
    x = seed
    x ^= x >> 12
    x ^= x << 25 & MASK64
    x ^= x >> 27
    return (x * 0x2545F4914F6CDD1D & MASK64) >> 40


def test_seeds():
    for c in (0, 1, 12345, (1 << 24) - 1):
        assert draw_of(seed_of(c)) == c


@pytest.fixture(scope="module")
def state(built):
    kb.device_check()
    return kb.State(kb.Model(kb.ensure_model("cfg0", MODEL_CACHE)))


# One token with 0.9998 of the mass, the others below 2^-25 each: a running sum that has passed the one no longer
# moves by another, while a stretch's own sum does. So every coin beyond 0.9998 ends in a stretch without a hit.
COINS = [0.99983, 0.99988, 0.99993, 0.99998]


def peaked(state, barred):
    lg = state.forward(5, 0).astype(np.float64)
    v = len(lg)
    fav = 7
    rest = np.ones(v, bool)
    rest[[fav, *barred]] = False
    up = float(np.log(0.9998 / 0.0002) + np.log(np.exp(lg[rest] - lg[fav]).sum()))
    p = np.where(rest, np.exp(lg - lg[fav] - up), 0.0)
    p[fav] = 1.0
    p /= p.sum()
    assert 0.9997 < p[fav] < 0.9999 and p[rest].max() < 2.0 ** -25
    return p, fav, up


def near(p, tok, coin):
    """The token's stretch of the vocabulary (a 1024th of it) holds the coin, to the rounding of 1024 sums below 1."""
    c = -(-len(p) // 1024)
    cum = np.concatenate([[0.0], np.cumsum(p)])
    lo = tok // c * c
    return cum[lo] - 2.0 ** -15 <= coin <= cum[min(len(p), lo + c)] + 2.0 ** -15


@pytest.mark.parametrize("coin", COINS)
def test_a_token_biased_to_minus_infinity_is_not_drawn(state, coin):
    v = state.cfg["vocab"]
    barred = [v - 1, v - 2, v - 40]
    p, fav, up = peaked(state, barred)
    s = kb.Sampler(state, temperature=1.0, seed=seed_of(int(coin * 2 ** 24)))
    s.set_bias({fav: up, **{t: float("-inf") for t in barred}})
    state.forward(5, 0)
    tok = s.sample()
    assert tok not in barred and p[tok] > 0 and near(p, tok, coin)


@pytest.mark.parametrize("coin", COINS)
def test_a_masked_draw_keeps_its_place(state, coin):
    """Where the walk ends without a hit the drawn stretch's token is taken, not the likeliest one."""
    v = state.cfg["vocab"]
    barred = [v - 1, v - 2, v - 40]
    p, fav, up = peaked(state, barred)
    allowed = np.ones(v, bool)
    allowed[barred] = False
    s = kb.Sampler(state, temperature=1.0, seed=seed_of(int(coin * 2 ** 24)))
    s.set_bias({fav: up}).set_mask(allowed)
    state.forward(5, 0)
    tok = s.sample()
    assert allowed[tok] and tok != fav and near(p, tok, coin)


def test_the_last_coin_stays_inside(state):
    """The largest coin may lie past the sum of all probabilities."""
    v = state.cfg["vocab"]
    allowed = np.arange(v) < v - 5000
    for k in range(1, 40):
        s = kb.Sampler(state, temperature=1.0, seed=seed_of((1 << 24) - k))
        s.set_mask(allowed)
        state.forward(k, 0)
        assert allowed[s.sample()]


@pytest.mark.parametrize("opts", [dict(temperature=0.0), dict(temperature=1.0), dict(temperature=0.9, topk=20),
                                  dict(temperature=0.7, topp=0.9)])
def test_a_mask_holds_where_every_logit_is_barred(state, opts):
    """All of the allowed tokens biased to -inf: every logit is -inf, the softmax uniform, and what is drawn from it
    nearly always a token that the mask does not allow. The mask holds."""
    v = state.cfg["vocab"]
    allowed = np.zeros(v, bool)
    allowed[[900, 31000, 31001]] = True
    for seed in (1, 2, 3, 4):
        s = kb.Sampler(state, seed=seed, **opts)
        s.set_mask(allowed).set_bias({int(t): float("-inf") for t in np.nonzero(allowed)[0]})
        state.forward(3, 0)
        assert allowed[s.sample()]
