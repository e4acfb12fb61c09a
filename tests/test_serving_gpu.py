"""The serving operators on the GPU against plain restatements (serving_ref.py).

Attention, tolerance from its roundings. A score is a sum of hd products whose
factors keep 22 bits or more (each side off by at most 2^-22 of itself) and
whose f32 additions each lose at most 2^-23 of the partial sum, all relative to
reach = sum |q k| scale: off by d <= (2^-21 + hd 2^-23 + 2^-22) reach. A weight
exp(s - m) is then off by 2 d (s and m) + 2^-21 (exp2 and its argument's
rounding, |s - m| 2^-23 more, weighted by weights below 1: at most 2^-21 in
sum), the numerator and the denominator of an output by that and by the f32 sum
over the tiles, at most 2^-23 for each of them. Against max|v|:
  tol = 2 (2 d + 2^-20 + tiles 2^-23).
The roundings of different terms are independent, so their 2-norm is far less:
sqrt(hd) takes the place of hd, and the typical score that of the reach. With
d_rms = sqrt(hd) 2^-23 and scores of order 1, the relative 2-norm stays below
4 * sqrt(256) * 2^-23 < 8e-6: held at 4e-6 for hd <= 128 and 8e-6 beyond.
"""
import numpy as np
import pytest

import krafla_b200 as kb
import serving_ref as ref

pytestmark = pytest.mark.gpu

KV = {"f32": kb.F32, "f16": kb.F16, "q8": kb.Q8_0}


@pytest.fixture(scope="module", autouse=True)
def _dev(built):
    kb.device_check()


def make_pool(rng, kv, n_pages, hk, page, hd):
    shape = (n_pages, hk, page, hd)
    if kv == "q8":
        k, v = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
        kd, vd = (rng.uniform(0.002, 0.02, shape[:3]).astype(np.float32) for _ in range(2))
        return k, v, kd, vd
    dt = np.float16 if kv == "f16" else np.float32
    return rng.standard_normal(shape).astype(dt), rng.standard_normal(shape).astype(dt), None, None


def make_table(rng, lens, page, n_pages, width=None):
    need = [-(-n // page) for n in lens]
    ids = rng.permutation(n_pages)
    t = np.full((len(lens), width or max(1, max(need))), -1, np.int32)
    at = 0
    for i, k in enumerate(need):
        t[i, :k] = ids[at:at + k]
        at += k
    return t


def spoil(pools, table, lens, page):
    """NaN (8-bit: NaN scales) in every slot that no position uses."""
    k, v, kd, vd = pools
    used = np.zeros((k.shape[0], page), bool)
    for i, n in enumerate(lens):
        for p in range(n):
            used[table[i, p // page], p % page] = True
    for x in (k, v) if kd is None else (kd, vd):
        x.swapaxes(1, 2)[~used] = np.nan


def handle(pools, table, kv, heads):
    k, v, kd, vd = (None if x is None else kb.DevArray.of(x) for x in pools)
    return kb.PagedKV(k, v, kb.DevArray.of(table), KV[kv], kd=kd, vd=vd, n_heads=heads)


def check(got, want, reach, vmax, hd, n_max, tp=8):
    d = (2.0 ** -21 + hd * 2.0 ** -23 + 2.0 ** -22) * reach[..., None]
    tol = vmax * 2 * (2 * d + 2.0 ** -20 + (n_max / tp + 1) * 2.0 ** -23)
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), (err / tol).max()
    if np.linalg.norm(want):
        assert np.linalg.norm(err) / np.linalg.norm(want) <= (4e-6 if hd <= 128 else 8e-6)


SHAPES = [
    # heads, kv heads, head dim, page, lengths, window, softcap
    (32, 8, 64, 16, [1], 0, 0.0),
    (6, 6, 48, 8, [0, 1, 7, 8, 9, 31, 33, 200], 0, 0.0),
    (14, 2, 64, 32, [700, 1, 64, 65, 0, 129], 0, 30.0),
    (32, 8, 128, 16, [513, 17, 64], 0, 0.0),
    (4, 2, 256, 16, [300, 5], 0, 0.0),
    (12, 1, 128, 64, [400, 3, 128], 0, 0.0),          # 12 heads share a KV head
    (40, 2, 64, 16, [130, 31], 0, 0.0),               # 20 heads share one
    (20, 1, 256, 16, [77], 0, 20.0),
    (2, 2, 16, 1, [5, 40], 0, 0.0),                   # a page of one position
    (4, 4, 80, 5, [23, 64, 101], 0, 0.0),             # a page size that divides nothing
    (8, 2, 112, 128, [1000, 999], 257, 0.0),
    (8, 2, 64, 16, [100, 50, 3], 1, 0.0),             # a window of the last position
    (8, 2, 96, 16, [100, 50, 3, 49], 49, 5.0),
]


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s[:4])) for s in SHAPES])
def test_attend(kv, shape):
    heads, hk, hd, page, lens, window, softcap = shape
    rng = np.random.default_rng(hash(shape[:4]) % 1000)
    need = sum(-(-n // page) for n in lens)
    pools = make_pool(rng, kv, need + 2, hk, page, hd)
    table = make_table(rng, lens, page, need + 2)
    spoil(pools, table, lens, page)
    q = rng.standard_normal((len(lens), heads, hd)).astype(np.float32)
    k, v, kd, vd = pools
    c = handle(pools, table, kv, heads)
    out = kb.DevArray.of(np.full(q.shape, np.nan, np.float32))
    scale = hd ** -0.5
    c.attend(kb.DevArray.of(q), kb.DevArray.of(np.array(lens, np.int32)), out, scale=scale, window=window, softcap=softcap)
    kb._check(kb.lib().kc_dev_sync(), "sync")
    want, reach = ref.attend(q, k, v, table, lens, scale, window, softcap, kd, vd)
    vmax = np.nanmax(np.abs(v.astype(np.float64))) if kd is None else np.nanmax(127 * vd)
    check(out.numpy(), want, reach, vmax, hd, max(lens))
    assert (out.numpy()[np.array(lens) == 0] == 0).all()


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("n,heads,hk,hd,top", [(90, 16, 8, 64, 300), (700, 2, 1, 64, 90), (41, 8, 8, 128, 700), (140, 3, 3, 32, 60)])
def test_attend_many_sequences(kv, n, heads, hk, hd, top):
    """More units (sequences times KV heads) than CTAs, more sequences than threads, ragged and empty ones."""
    rng = np.random.default_rng(n + hd)
    page = 16
    lens = np.where(rng.random(n) < 0.1, 0, rng.integers(1, top, n)).tolist()
    n_pages = sum(-(-m // page) for m in lens)
    pools = make_pool(rng, kv, n_pages, hk, page, hd)
    table = make_table(rng, lens, page, n_pages)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    c = handle(pools, table, kv, heads)
    dq, dl = kb.DevArray.of(q), kb.DevArray.of(np.array(lens, np.int32))
    k, v, kd, vd = pools
    vmax = np.abs(v.astype(np.float64)).max() if kd is None else (127 * vd).max()
    for window in (0, 33):
        out = c.attend(dq, dl, kb.DevArray.of(np.full(q.shape, np.nan, np.float32)), window=window)
        want, reach = ref.attend(q, k, v, table, lens, hd ** -0.5, window, 0.0, kd, vd)
        check(out.numpy(), want, reach, vmax, hd, max(lens))
    kb._check(kb.lib().kc_dev_sync(), "sync")


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
def test_attend_long_is_split_and_repeatable(kv):
    rng = np.random.default_rng(5)
    lens, page, hk, hd, heads = [20011, 4096], 16, 2, 128, 8
    n_pages = sum(-(-n // page) for n in lens)
    pools, table = make_pool(rng, kv, n_pages, hk, page, hd), None
    table = make_table(rng, lens, page, n_pages)
    q = (3 * rng.standard_normal((2, heads, hd))).astype(np.float32)   # peaked scores
    c = handle(pools, table, kv, heads)
    args = kb.DevArray.of(q), kb.DevArray.of(np.array(lens, np.int32))
    a, b = (c.attend(*args, kb.DevArray(q.shape, np.float32)).numpy() for _ in range(2))
    assert np.array_equal(a, b)
    k, v, kd, vd = pools
    want, reach = ref.attend(q, k, v, table, lens, hd ** -0.5, 0, 0.0, kd, vd)
    vmax = np.abs(v.astype(np.float64)).max() if kd is None else (127 * vd).max()
    check(a, want, reach, vmax, hd, max(lens))


def test_attend_small_and_large_values():
    """Queries and values far from 1, and a flat tail under one large weight."""
    rng = np.random.default_rng(6)
    page, hk, hd, n = 16, 1, 64, 3000
    for qs, ks in ((1e-20, 1.0), (1e6, 1e-3), (1.0, 60.0)):
        k = (ks * rng.standard_normal((200, hk, page, hd))).astype(np.float16)
        v = (1 + rng.standard_normal(k.shape)).astype(np.float16)
        table = make_table(rng, [n], page, 200)
        q = (qs * rng.standard_normal((1, 4, hd))).astype(np.float32)
        scale = 0.05 / (qs * ks)
        c = handle((k, v, None, None), table, "f16", 4)
        out = c.attend(kb.DevArray.of(q), kb.DevArray.of(np.array([n], np.int32)), kb.DevArray(q.shape, np.float32), scale=scale)
        want, reach = ref.attend(q, k, v, table, [n], scale)
        check(out.numpy(), want, reach, np.abs(v.astype(float)).max(), hd, n)
    # one position's weight is e^18 of every other's: the 2999 others still count
    k[:] = 0
    k[table[0, 0], 0, 0] = 1.0
    q = np.full((1, 4, hd), 18.0 / hd, np.float32)
    c = handle((k, v, None, None), table, "f16", 4)
    out = c.attend(kb.DevArray.of(q), kb.DevArray.of(np.array([n], np.int32)), kb.DevArray(q.shape, np.float32), scale=1.0)
    want, reach = ref.attend(q, k, v, table, [n], 1.0)
    check(out.numpy(), want, reach, np.abs(v.astype(float)).max(), hd, n)


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("softcap", [0.0, 4.0])
def test_attend_signs_of_the_scale(kv, softcap):
    """A negative scale, one of zero (the mean of V), and a query head of zeros."""
    rng = np.random.default_rng(9)
    lens, page, hk, hd, heads = [70, 33], 16, 2, 64, 6
    pools = make_pool(rng, kv, 12, hk, page, hd)
    table = make_table(rng, lens, page, 12)
    q = rng.standard_normal((2, heads, hd)).astype(np.float32)
    q[0, 2] = 0.0
    c = handle(pools, table, kv, heads)
    k, v, kd, vd = pools
    vmax = np.abs(v.astype(np.float64)).max() if kd is None else (127 * vd).max()
    for scale in (-0.2, 0.0, 0.1):
        out = c.attend(kb.DevArray.of(q), kb.DevArray.of(np.array(lens, np.int32)), kb.DevArray(q.shape, np.float32),
                       scale=scale, softcap=softcap)
        want, reach = ref.attend(q, k, v, table, lens, scale, 0, softcap, kd, vd)
        check(out.numpy(), want, reach, vmax, hd, 70)


def test_attend_one_bad_head_stays_alone():
    """A NaN in one sequence's KV head reaches that head's queries only."""
    rng = np.random.default_rng(10)
    lens, page, hk, hd, heads = [50, 40], 16, 2, 64, 4
    pools = make_pool(rng, "f16", 12, hk, page, hd)
    table = make_table(rng, lens, page, 12)
    q = rng.standard_normal((2, heads, hd)).astype(np.float32)
    k, v = pools[:2]
    want, reach = ref.attend(q, k, v, table, lens, hd ** -0.5)
    k[table[0, 1], 1, 3] = np.nan
    out = handle(pools, table, "f16", heads).attend(kb.DevArray.of(q), kb.DevArray.of(np.array(lens, np.int32)),
                                                    kb.DevArray(q.shape, np.float32)).numpy()
    assert np.isnan(out[0, 2:]).all()
    out[0, 2:] = want[0, 2:]
    check(out, want, reach, 6, hd, 50)


def test_attend_strides_and_rows_behind():
    """Query and output rows inside wider ones; fewer sequences than the cache has."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(7)
    lens, page, hk, hd, heads = [40, 3, 90], 16, 2, 64, 4
    pools = make_pool(rng, "f16", 12, hk, page, hd)
    table = make_table(rng, lens, page, 12)
    c = handle(pools, table, "f16", heads)
    wide = torch.randn(3, heads * hd + 36, device="cuda")
    out = torch.full((3, heads * hd + 12), 7.0, device="cuda")
    dl = kb.DevArray.of(np.array(lens[:2], np.int32))
    c.attend(wide[:2, :heads * hd], dl, out[:2, :heads * hd])
    torch.cuda.synchronize()
    q = wide[:2, :heads * hd].cpu().numpy().reshape(2, heads, hd)
    want, reach = ref.attend(q, pools[0], pools[1], table, lens[:2], hd ** -0.5)
    got = out.cpu().numpy()
    check(got[:2, :heads * hd].reshape(2, heads, hd), want, reach, np.abs(pools[1].astype(float)).max(), hd, 90)
    assert (got[2] == 7).all() and (got[:, heads * hd:] == 7).all()


def test_attend_bad_pages_and_lengths_are_skipped_and_told():
    rng = np.random.default_rng(8)
    page, hk, hd, heads, lens = 16, 2, 64, 4, [40, 48, 33]
    pools = make_pool(rng, "f32", 9, hk, page, hd)
    table = make_table(rng, lens, page, 9)
    q = rng.standard_normal((3, heads, hd)).astype(np.float32)
    dq = kb.DevArray.of(q)

    def run(t, n):
        c = handle(pools, t, "f32", heads)
        return c.attend(dq, kb.DevArray.of(np.array(n, np.int32)), kb.DevArray(q.shape, np.float32))

    bad = table.copy()
    bad[1, 1] = 9
    bad[2, 0] = -7
    out = run(bad, lens)
    with pytest.raises(kb.KraflaError, match="page number"):
        kb._check(kb.lib().kc_dev_sync(), "sync")
    kb._check(kb.lib().kc_dev_sync(), "sync")                  # told once
    want, reach = ref.attend(q, pools[0], pools[1], table, lens, hd ** -0.5)
    check(out.numpy()[:1], want[:1], reach[:1], 6, hd, 48)
    # the bad page's positions count as not there
    keep = [p for p in range(48) if p // page != 1]
    k, v = (ref.gather(x, table, page, 1, keep).astype(float) for x in pools[:2])
    s = np.einsum("pgd,ghd->ghp", k, q[1].reshape(hk, -1, hd).astype(float)) * hd ** -0.5
    w = np.exp(s - s.max(-1, keepdims=True))
    w1 = np.einsum("ghp,pgd->ghd", w / w.sum(-1, keepdims=True), v).reshape(heads, hd)
    assert np.abs(out.numpy()[1] - w1).max() < 1e-4
    out = run(table, [40, -3, 4000])                           # -3: as 0; 4000: as the table's 48
    with pytest.raises(kb.KraflaError, match="sequence length"):
        kb._check(kb.lib().kc_dev_sync(), "sync")
    check(out.numpy()[:1], want[:1], reach[:1], 6, hd, 48)
    assert (out.numpy()[1] == 0).all()


ROPE = dict(rope_theta=5e5)


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("heads,hk,hd,page,norm,split", [
    (32, 8, 128, 16, True, False), (14, 2, 64, 32, False, False), (6, 6, 48, 8, True, True), (3, 1, 16, 1, True, False),
    (4, 2, 256, 7, True, False), (8, 4, 80, 16, True, True), (2, 2, 32, 64, False, False)])
def test_append(kv, heads, hk, hd, page, norm, split):
    """Rows of three sequences with padding between them; 8-bit and f32 rows as the rule gives them."""
    rng = np.random.default_rng(heads * hd + page)
    n = 61
    seqs = np.array([0] * 20 + [-1] * 3 + [2] * 30 + [-5] * 2 + [1] * 6, np.int32)
    pos = np.array([*range(20), 0, 0, 9, *range(11, 41), 1, 2, *range(50, 56)], np.int32)
    lens = [20, 56, 41]
    n_pages = sum(-(-m // page) for m in lens) + 1
    pools = make_pool(rng, kv, n_pages, hk, page, hd)
    table = make_table(rng, lens, page, n_pages)
    x = rng.standard_normal((n, (heads + 2 * hk) * hd)).astype(np.float32)
    x[5] = 0.0
    wq, wk = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    cos, sin = kb.rope_tables(dict(ROPE, head_dim=hd), 64)
    c = handle(pools, table, kv, heads)
    qo = kb.DevArray.of(np.full((n, heads, hd), 3.0, np.float32))
    dx = kb.DevArray.of(x)
    if split:
        dx = tuple(kb.DevArray.of(np.ascontiguousarray(t)) for t in np.split(x, [heads * hd, (heads + hk) * hd], axis=1))
    args = dict(q_norm=kb.DevArray.of(wq), k_norm=kb.DevArray.of(wk), eps=1e-6) if norm else {}
    c.append(dx, kb.DevArray.of(pos), kb.DevArray.of(cos), kb.DevArray.of(sin), qo, seqs=kb.DevArray.of(seqs), **args)
    kb._check(kb.lib().kc_dev_sync(), "sync")
    h = x.reshape(n, heads + 2 * hk, hd)
    q = ref.norm_rope(h[:, :heads], cos[pos], sin[pos], wq if norm else None, 1e-6)
    k = ref.norm_rope(h[:, heads:heads + hk], cos[pos], sin[pos], wk if norm else None, 1e-6)
    v = h[:, heads + hk:].astype(np.float64)
    live = seqs >= 0
    got = qo.numpy()
    assert (got[~live] == 3.0).all()
    # norm: the sum of hd squares (hd / 2 halvings of 2^-24 at most), a division and a root; product
    # and rotation: a few roundings of values at most sqrt(2) times the pair's larger one
    tol = (hd / 2 + 16) * 2.0 ** -24 * np.abs(q[live]).max(-1, keepdims=True) * 1.5
    assert (np.abs(got[live] - q[live]) <= tol).all()
    arrays = [None if a is None else a.numpy() for a in c._keep[:4]]
    for new, pool, scale, before, before_d in ((k, arrays[0], arrays[2], pools[0], pools[2]),
                                               (v, arrays[1], arrays[3], pools[1], pools[3])):
        want, want_d = before.copy(), None if before_d is None else before_d.copy()
        for i in np.nonzero(live)[0]:
            at = table[seqs[i], pos[i] // page], slice(None), pos[i] % page
            if scale is not None:
                want[at], d = ref.quant_rows(new[i])
                want_d[at] = d[..., 0]
            else:
                want[at] = new[i].astype(before.dtype)
        if scale is not None:
            assert np.array_equal(pool, want) and np.array_equal(scale, want_d)
        else:
            # as for the queries, and a last rounding of the type's half step
            step = np.finfo(before.dtype).eps / 2
            t = 1.5 * (hd / 2 + 16) * 2.0 ** -24 * np.abs(want.astype(float)).max() + 2 * step * np.abs(want.astype(float))
            assert (np.abs(pool.astype(float) - want.astype(float)) <= t).all()


def test_append_in_place_without_seqs_and_bad_rows():
    rng = np.random.default_rng(2)
    heads, hk, hd, page = 4, 2, 64, 16
    table = np.array([[0, 1], [2, 99], [3, 4]], np.int32)
    pools = make_pool(rng, "f16", 5, hk, page, hd)
    c = handle(pools, table, "f16", heads)
    cos, sin = kb.rope_tables(dict(ROPE, head_dim=hd), 32)
    x = rng.standard_normal((3, (heads + 2 * hk) * hd)).astype(np.float32)
    q, k, v = (kb.DevArray.of(np.ascontiguousarray(t)) for t in np.split(x, [heads * hd, (heads + hk) * hd], axis=1))
    dc, ds = kb.DevArray.of(cos), kb.DevArray.of(sin)
    for pos in ([31, 20, 5], [31, 5, 32], [31, -1, 5]):        # a bad page, a position past the tables, one below 0
        c.append((q, k, v), kb.DevArray.of(np.array(pos, np.int32)), dc, ds, kb.DevArray((3, heads, hd), np.float32))
        with pytest.raises(kb.KraflaError, match="new row"):
            kb._check(kb.lib().kc_dev_sync(), "sync")
    before = [a.numpy() for a in c._keep[:2]]
    c.append((q, k, v), kb.DevArray.of(np.array([31, 7, 5], np.int32)), dc, ds, q)   # queries in place
    kb._check(kb.lib().kc_dev_sync(), "sync")
    want = ref.norm_rope(x[:, :heads * hd].reshape(3, heads, hd), cos[[31, 7, 5]], sin[[31, 7, 5]])
    assert np.abs(q.numpy().reshape(want.shape) - want).max() < 1e-5
    after = [a.numpy() for a in c._keep[:2]]
    changed = np.argwhere((before[0] != after[0]).any((1, 3)))
    assert {tuple(t) for t in changed} <= {(1, 15), (2, 7), (3, 5)} and (2, 7) in {tuple(t) for t in changed}


def rand_logits_case(rng, n, v, hist, bias, mask, inf=False):
    z = (4 * rng.standard_normal((n, v))).astype(np.float32)
    if inf:
        z.reshape(-1)[rng.integers(0, n * v, 40)] = np.inf
        z.reshape(-1)[rng.integers(0, n * v, 40)] = -np.inf
        z.reshape(-1)[rng.integers(0, n * v, 40)] = np.nan
    kw, dev = {}, {}
    if hist is not None:
        h = rng.integers(-2, min(v + 3, 200), (n, hist)).astype(np.int32)
        kw.update(history=h, history_len=rng.integers(0, hist + 1, n).astype(np.int32),
                  repeat=rng.uniform(0.8, 2, n).astype(np.float32), presence=rng.normal(0, 1, n).astype(np.float32),
                  frequency=rng.normal(0, 1, n).astype(np.float32))
    dev = {k: kb.DevArray.of(x) for k, x in kw.items()}
    if bias:
        kw["bias"] = [(rng.integers(-1, min(v + 2, 100), m).astype(np.int32), rng.normal(0, 5, m).astype(np.float32))
                      for m in rng.integers(0, bias + 1, n)]
        off = np.concatenate([[0], np.cumsum([len(i) for i, _ in kw["bias"]])]).astype(np.int32)
        dev.update(bias_off=kb.DevArray.of(off), bias_ids=kb.DevArray.of(np.concatenate([i for i, _ in kw["bias"]])),
                   bias_vals=kb.DevArray.of(np.concatenate([b for _, b in kw["bias"]])))
    if mask:
        kw["mask"] = rng.integers(0, 2 ** 32, (n, (v + 31) // 32 + mask - 1), dtype=np.uint64).astype(np.uint32)
        kw["mask"][0] = 0                                      # a row that allows nothing
        dev["mask"] = kb.DevArray.of(kw["mask"])
    return z, kw, dev


@pytest.mark.parametrize("n,v,hist,bias,mask", [
    (1, 32000, 64, 0, 0), (3, 4097, 300, 50, 1), (2, 1, 3, 2, 1), (5, 31, None, 5, 1), (4, 151937, 2000, 0, 2),
    (2, 8192, None, 0, 1), (3, 8191, 0, 300, 0), (70000, 5, 2, 0, 0), (2, 300, 70001, 10, 1), (2, 12289, 9, 70000, 1)])
def test_logits(n, v, hist, bias, mask):
    """Bit for bit: every operation is a single IEEE one, on NaN and infinite logits too."""
    rng = np.random.default_rng(n + v)
    z, kw, dev = rand_logits_case(rng, n, v, hist, bias, mask, inf=v > 100)
    dz = kb.DevArray.of(z)
    out = kb.process_logits(kb.DevArray.of(np.full_like(z, 9.0)), dz, **dev)
    kb._check(kb.lib().kc_dev_sync(), "sync")
    want = ref.logits(z, **kw)
    assert np.array_equal(out.numpy(), want, equal_nan=True)
    kb.process_logits(dz, dz, **dev)                           # in place
    kb._check(kb.lib().kc_dev_sync(), "sync")
    assert np.array_equal(dz.numpy(), want, equal_nan=True)


def test_logits_unaligned_views():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(4)
    z, kw, dev = rand_logits_case(rng, 4, 9001, 20, 5, 1)
    for a, b in ((1, 1), (2, 3), (0, 1), (3, 0)):
        src, dst = torch.zeros(4, 9010, device="cuda"), torch.full((4, 9012), 5.0, device="cuda")
        src[:, a:a + 9001] = torch.from_numpy(z).cuda()
        torch.cuda.synchronize()
        kb.process_logits(dst[:, b:b + 9001], src[:, a:a + 9001], **dev)
        torch.cuda.synchronize()
        got = dst.cpu().numpy()
        assert np.array_equal(got[:, b:b + 9001], ref.logits(z, **kw))
        assert (got[:, :b] == 5).all() and (got[:, b + 9001:] == 5).all()


def test_logits_bad_offsets_and_lengths():
    z = np.ones((2, 50), np.float32)
    ids, vals = kb.DevArray.of(np.array([3, 4], np.int32)), kb.DevArray.of(np.array([1, 2], np.float32))
    out = kb.process_logits(kb.DevArray((2, 50), np.float32), kb.DevArray.of(z), bias_ids=ids, bias_vals=vals,
                            bias_off=kb.DevArray.of(np.array([0, 2, 900], np.int32)))
    with pytest.raises(kb.KraflaError, match="bias offsets"):
        kb._check(kb.lib().kc_dev_sync(), "sync")
    assert out.numpy()[0, 4] == 3 and (out.numpy()[1] == 1).all()
    kb.process_logits(out, out, history=kb.DevArray.of(np.zeros((2, 1), np.int32)),
                      history_len=kb.DevArray.of(np.array([1, 77], np.int32)),
                      presence=kb.DevArray.of(np.ones(2, np.float32)))
    with pytest.raises(kb.KraflaError, match="history length"):
        kb._check(kb.lib().kc_dev_sync(), "sync")
    assert (out.numpy()[:, 0] == 0).all()


def test_refused_pointers():
    """Host memory and wrong types never reach a kernel."""
    a = np.zeros((2, 64), np.float32)
    x = dict({n: 0 for n in kb._LOGITS.names}, out=a.ctypes.data, ld_in=64, ld_out=64, rows=2, vocab=64)
    x["in"] = a.ctypes.data
    assert kb.lib().kc_logits_process_dev(kb._LOGITS.pack(*x.values()), None) == kb.E_SHAPE
    assert "not device memory" in kb.what_detail()
    with pytest.raises(kb.KraflaError, match="float32"):
        kb.process_logits(kb.DevArray((2, 64), np.float32), kb.DevArray((2, 64), np.float16))
    rng = np.random.default_rng(0)
    pools = make_pool(rng, "f16", 2, 1, 16, 64)
    c = handle(pools, np.zeros((1, 1), np.int32), "f16", 4)
    q = kb.DevArray((1, 4, 64), np.float32)
    with pytest.raises(kb.KraflaError, match="lens"):
        c.attend(q, kb.DevArray((2,), np.int32), q)
    with pytest.raises(kb.KraflaError, match="workspace"):
        c.attend(q, kb.DevArray((1,), np.int32), q, ws=kb.DevBuf(64))


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
def test_decode_steps_together(kv):
    """A prompt and then steps of three sequences: append, attend, logits, the least of them masked away."""
    rng = np.random.default_rng(11)
    heads, hk, hd, page, vocab, steps = 14, 2, 64, 16, 1003, 6
    prompt = [37, 1, 16]
    cap = -(-(max(prompt) + steps) // page)
    n_pages = 3 * cap
    shape = (n_pages, hk, page, hd)
    dt = {"f32": np.float32, "f16": np.float16, "q8": np.int8}[kv]
    k, v = kb.DevArray(shape, dt), kb.DevArray(shape, dt)
    kd, vd = (kb.DevArray(shape[:3], np.float32) for _ in range(2)) if kv == "q8" else (None, None)
    table = rng.permutation(n_pages).reshape(3, cap).astype(np.int32)
    c = kb.PagedKV(k, v, kb.DevArray.of(table), KV[kv], kd=kd, vd=vd, n_heads=heads)
    cfg = dict(head_dim=hd, rope_theta=1e6)
    cos, sin = kb.rope_tables(cfg, 64)
    dc, ds = kb.DevArray.of(cos), kb.DevArray.of(sin)
    w = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    dw = [kb.DevArray.of(t) for t in w]
    head = rng.standard_normal((heads * hd, vocab)).astype(np.float32)
    keys, vals = [[] for _ in prompt], [[] for _ in prompt]

    def rows(x, seqs, pos):
        h = x.reshape(len(x), heads + 2 * hk, hd)
        kk = ref.norm_rope(h[:, heads:heads + hk], cos[pos], sin[pos], w[1], 1e-5)
        for i, s in enumerate(seqs):
            for store, t in ((keys, kk[i]), (vals, h[i, heads + hk:])):
                if kv == "q8":
                    qq, d = ref.quant_rows(t)
                    t = qq.astype(float) * d
                store[s].append(t.astype(dt).astype(float) if kv != "q8" else t)

    seqs = np.repeat(np.arange(3), prompt).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in prompt]).astype(np.int32)
    x = rng.standard_normal((len(pos), (heads + 2 * hk) * hd)).astype(np.float32)
    c.append(kb.DevArray.of(x), kb.DevArray.of(pos), dc, ds, kb.DevArray((len(pos), heads, hd), np.float32),
             seqs=kb.DevArray.of(seqs), q_norm=dw[0], k_norm=dw[1])
    rows(x, seqs, pos)
    hist = np.full((3, steps), -1, np.int32)
    for t in range(steps):
        pos = np.array(prompt, np.int32) + t
        x = rng.standard_normal((3, (heads + 2 * hk) * hd)).astype(np.float32)
        q = c.append(kb.DevArray.of(x), kb.DevArray.of(pos), dc, ds, kb.DevArray((3, heads, hd), np.float32),
                     q_norm=dw[0], k_norm=dw[1])
        o = c.attend(q, kb.DevArray.of(pos + 1), kb.DevArray((3, heads, hd), np.float32)).numpy()
        rows(x, range(3), pos)
        qn = q.numpy()
        if kv == "q8":
            qi, qd = ref.quant_rows(qn)
            qn = qi.astype(float) * qd
        for i in range(3):
            kk, vv = np.stack(keys[i]), np.stack(vals[i])
            s = np.einsum("pgd,ghd->ghp", kk, qn[i].reshape(hk, -1, hd).astype(float)) * hd ** -0.5
            e = np.exp(s - s.max(-1, keepdims=True))
            want = np.einsum("ghp,pgd->ghd", e / e.sum(-1, keepdims=True), vv).reshape(heads, hd)
            # the stored f16 rows are off by half a step of the kernel's f32 ones at most where both round
            # apart: 2^-11 of a value in a rare element; f32 and 8-bit rows agree to 2^-22
            assert np.linalg.norm(o[i] - want) <= (2e-4 if kv == "f16" else 1e-5) * np.linalg.norm(want)
        z = (o.reshape(3, -1) @ head).astype(np.float32)
        mask = np.full((3, (vocab + 31) // 32), 0xffffffff, np.uint32)
        mask[1, 1:] = 0                                        # the second sequence may say 0..31 only
        got = kb.process_logits(kb.DevArray(z.shape, np.float32), kb.DevArray.of(z), history=kb.DevArray.of(hist),
                                repeat=kb.DevArray.of(np.full(3, 1.3, np.float32)),
                                presence=kb.DevArray.of(np.full(3, 1e9, np.float32)), mask=kb.DevArray.of(mask)).numpy()
        assert np.array_equal(got, ref.logits(z, history=hist, repeat=[1.3] * 3, presence=[1e9] * 3, mask=mask))
        tok = got.argmax(1)
        assert tok[1] < 32 and all(tok[i] not in hist[i] for i in range(3))   # no token twice
        hist[:, t] = tok
    kb._check(kb.lib().kc_dev_sync(), "sync")


def test_streams_graphs_and_far_offsets():
    """A pool beyond 2^32 bytes, filled and read on another stream, then captured and replayed with
    other lengths; two graphs with a workspace each, replayed at once."""
    torch = pytest.importorskip("torch")
    heads, hk, hd, page, n_pages = 8, 2, 256, 64, 36000        # 36000 * 2 * 64 * 256 * 4 = 4.7e9 bytes
    k, v = (torch.empty(n_pages, hk, page, hd, device="cuda") for _ in range(2))
    assert k.numel() * 4 > 2 ** 32
    ids = torch.tensor([[35999, 7, 35990], [35998, 35997, 0]], dtype=torch.int32, device="cuda")
    c = kb.PagedKV(k, v, ids, kb.F32, n_heads=heads)
    cos, sin = kb.rope_tables(dict(head_dim=hd, rope_theta=1e4), 192)
    dc, ds = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(300, (heads + 2 * hk) * hd, generator=g)
    pos = torch.tensor([*range(150)] * 2, dtype=torch.int32, device="cuda")
    seqs = torch.tensor([0] * 150 + [1] * 150, dtype=torch.int32, device="cuda")
    q = torch.randn(2, heads, hd, generator=g).cuda()
    lens = torch.tensor([150, 70], dtype=torch.int32, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    outs = [torch.zeros(2, heads, hd, device="cuda") for _ in range(3)]
    ws = c.workspace()
    with torch.cuda.stream(st):
        dx = x.cuda()
        qo = torch.empty(300, heads, hd, device="cuda")
        c.append(dx, pos, dc, ds, qo, seqs=seqs, stream=st.cuda_stream)
        c.attend(q, lens, outs[0], stream=st.cuda_stream)
        graphs = []
        for o, w in ((outs[1], None), (outs[2], ws)):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=st):
                c.attend(q, lens, o, stream=st.cuda_stream, ws=w)
            graphs.append(gr)
    torch.cuda.synchronize()
    h = x.numpy().reshape(300, heads + 2 * hk, hd)
    kk = ref.norm_rope(h[:, heads:heads + hk], cos[pos.cpu()], sin[pos.cpu()]).reshape(2, 150, hk, hd)
    vv = h[:, heads + hk:].reshape(2, 150, hk, hd).astype(float)

    def close(o, n):
        for i in range(2):
            s = np.einsum("pgd,ghd->ghp", kk[i, :n[i]], q[i].cpu().numpy().reshape(hk, -1, hd).astype(float)) * hd ** -0.5
            e = np.exp(s - s.max(-1, keepdims=True))
            want = np.einsum("ghp,pgd->ghd", e / e.sum(-1, keepdims=True), vv[i, :n[i]]).reshape(heads, hd)
            assert np.linalg.norm(o[i].cpu().numpy() - want) <= 2e-5 * np.linalg.norm(want)

    close(outs[0], (150, 70))
    other = torch.cuda.Stream()
    for n in ((150, 70), (1, 149), (65, 0)):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[1], outs[2])
        if n[1]:
            close(outs[1], n)
        else:
            assert (outs[1][1] == 0).all()
    del graphs


def test_logits_negative_history_length_is_told():
    out = kb.process_logits(kb.DevArray((2, 50), np.float32), kb.DevArray.of(np.ones((2, 50), np.float32)),
                            history=kb.DevArray.of(np.zeros((2, 3), np.int32)),
                            history_len=kb.DevArray.of(np.array([-5, 3], np.int32)),
                            frequency=kb.DevArray.of(np.ones(2, np.float32)))
    with pytest.raises(kb.KraflaError, match="history length"):
        kb._check(kb.lib().kc_dev_sync(), "sync")
    assert (out.numpy()[0] == 1).all() and out.numpy()[1, 0] == -2


def test_two_streams_in_one_graph():
    """A graph whose two branches append to and read a cache each, join, and are followed by the logits of both:
    every launch has a kernel or an event of another stream before it. Replays give what calls in a row give."""
    torch = pytest.importorskip("torch")
    heads, hk, hd, page, n = 4, 2, 64, 16, 3
    g = torch.Generator().manual_seed(3)
    cos, sin = (torch.from_numpy(t).cuda() for t in kb.rope_tables(dict(head_dim=hd, rope_theta=1e4), 64))
    table = torch.arange(n * 4, dtype=torch.int32).reshape(n, 4).cuda()
    caches, xs, qs = [], [], []
    for _ in range(2):
        k, v = (torch.randn(n * 4, hk, page, hd, generator=g).half().cuda() for _ in range(2))
        caches.append(kb.PagedKV(k, v, table, kb.F16, n_heads=heads))
        xs.append(torch.randn(n, (heads + 2 * hk) * hd, generator=g).cuda())
        qs.append(torch.empty(n, heads, hd, device="cuda"))
    pos = torch.tensor([40, 3, 63], dtype=torch.int32, device="cuda")
    lens = pos + 1
    both, last = torch.empty(2 * n, heads * hd, device="cuda"), torch.empty(2 * n, heads * hd, device="cuda")
    hist = torch.randint(0, heads * hd, (2 * n, 9), generator=g, dtype=torch.int32).cuda()
    rep = torch.full((2 * n,), 1.3, device="cuda")

    def half(i, st):
        caches[i].append(xs[i], pos, cos, sin, qs[i], stream=st)
        caches[i].attend(qs[i], lens, both[i * n:(i + 1) * n], stream=st)

    def end(st):
        kb.process_logits(last, both, history=hist, repeat=rep, stream=st)

    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(2):
        half(i, main.cuda_stream)
    end(main.cuda_stream)
    torch.cuda.synchronize()
    want = last.clone()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=main):
        side.wait_stream(main)
        half(1, side.cuda_stream)
        half(0, main.cuda_stream)
        main.wait_stream(side)
        end(main.cuda_stream)
    for _ in range(3):
        both.zero_()
        last.zero_()
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(last, want)
    del gr


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("heads,hk,hd", [(8, 2, 256), (12, 1, 192), (2, 2, 144)])
def test_attend_wide_heads_few_and_many(kv, heads, hk, hd):
    """Calls of one sequence and of many, which wide heads take in different shapes, in turn in one workspace."""
    rng = np.random.default_rng(heads + hd)
    lens, page = [2500, 0, 1, 700, 64, 8, 33, 1500, 15, 2049], 16
    n_pages = sum(-(-m // page) for m in lens)
    pools = make_pool(rng, kv, n_pages, hk, page, hd)
    table = make_table(rng, lens, page, n_pages)
    q = rng.standard_normal((len(lens), heads, hd)).astype(np.float32)
    c = handle(pools, table, kv, heads)
    k, v, kd, vd = pools
    vmax = np.abs(v.astype(np.float64)).max() if kd is None else (127 * vd).max()
    want, reach = ref.attend(q, k, v, table, lens, hd ** -0.5, 0, 20.0, kd, vd)
    for n in (1, len(lens), 2, 1, 5, len(lens)):
        out = kb.DevArray.of(np.full((n, heads, hd), np.nan, np.float32))
        c.attend(kb.DevArray.of(q[:n]), kb.DevArray.of(np.array(lens[:n], np.int32)), out, softcap=20.0)
        check(out.numpy(), want[:n], reach[:n], vmax, hd, max(lens))
    kb._check(kb.lib().kc_dev_sync(), "sync")
