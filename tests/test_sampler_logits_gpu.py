"""The sampler's penalties, biases and mask (kc_sampler_set_*) over a model's own
logits: greedy choices against the restatement of the logits' processing, sampled
ones inside the mask, and the plain sampler where nothing is set."""
import numpy as np
import pytest

from conftest import MODEL_CACHE

import krafla_b200 as kb
import serving_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(built):
    kb.device_check()
    return kb.Model(kb.ensure_model("cfg0", MODEL_CACHE))


def words(allowed):
    return np.packbits(np.pad(allowed, (0, -len(allowed) % 32)), bitorder="little").view(np.uint32)[None]


def test_greedy_follows_the_processed_logits(model):
    v = model.config["vocab"]
    rng = np.random.default_rng(1)
    st = kb.State(model)
    s = kb.Sampler(st, temperature=0.0, repeat_penalty=1.2, repeat_last_n=8)
    ring, tok = [], 5
    allowed = rng.random(v) < 0.3
    bias = [(int(t), float(b)) for t, b in zip(rng.integers(0, v, 40), rng.normal(0, 1, 40))]
    bias += [(bias[0][0], 2.0)]                                # the same token twice: the last counts
    for t in (5, 9, 9, 700):
        s.accept(t)
        ring.append(t)
    for step in range(12):
        if step == 2:
            s.set_penalties(0.3, 0.1)
        if step == 4:
            s.set_bias(bias)
        if step == 6:
            s.set_mask(allowed)
        if step == 10:
            s.set_mask(None).set_bias(None)
        lg = st.forward(tok, step)[None]
        h = np.array([ring[-8:]])
        want = ref.logits(lg, history=h, repeat=[1.2], presence=[0.3] if step >= 2 else None,
                          frequency=[0.1] if step >= 2 else None,
                          bias=[(np.array([t for t, _ in bias]), np.array([b for _, b in bias], np.float32))] if 4 <= step < 10 else None,
                          mask=words(allowed) if 6 <= step < 10 else None)
        got = s.sample()
        assert got == int(want[0].argmax()), step
        assert not 6 <= step < 10 or allowed[got]
        ring.append(got)
        tok = got


@pytest.mark.parametrize("opts", [dict(temperature=1.0), dict(temperature=0.9, topk=20), dict(temperature=0.7, topp=0.9)])
def test_sampled_tokens_stay_inside_the_mask(model, opts):
    v = model.config["vocab"]
    st = kb.State(model)
    s = kb.Sampler(st, seed=3, repeat_penalty=1.1, repeat_last_n=16, **opts)
    allowed = np.zeros(v, bool)
    allowed[[3, 77, 31999, 1000, 1001]] = True                 # fewer than top-k
    s.set_mask(allowed)
    toks = st.generate_sampled(s, 1, 0, 40)
    assert allowed[toks].all() and len(set(toks.tolist())) > 1


def test_set_to_nothing_is_the_plain_sampler(model):
    out = []
    for touch in (False, True):
        st = kb.State(model)
        s = kb.Sampler(st, temperature=0.8, topk=40, repeat_penalty=1.3, repeat_last_n=16, seed=9)
        if touch:
            s.set_penalties(0.0, 0.0).set_bias(None).set_mask(None)
        out.append(st.generate_sampled(s, 1, 0, 30).tolist())
    assert out[0] == out[1]


def test_refusals(model):
    v = model.config["vocab"]
    s = kb.Sampler(kb.State(model), temperature=0.0)
    with pytest.raises(kb.KraflaError, match="no token"):
        s.set_mask(np.zeros(v, bool))
    with pytest.raises(kb.KraflaError, match="vocab"):
        s.set_bias({v: 1.0})
    with pytest.raises(kb.KraflaError):
        s.set_bias({3: float("nan")})
    with pytest.raises(kb.KraflaError, match="finite"):
        s.set_penalties(float("inf"))
    with pytest.raises(kb.KraflaError, match="allowed"):
        s.set_mask(np.ones(v + 1, bool))


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_bias_beyond_numbers_is_refused(model, value):
    s = kb.Sampler(kb.State(model), temperature=0.8)
    with pytest.raises(kb.KraflaError):
        s.set_bias({3: value})
    s.set_bias({3: float("-inf")})                     # a token never to be chosen is a bias
