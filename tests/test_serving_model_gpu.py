"""The paged operators against the model path: the q|k|v rows that a model's own
decode steps made, through append into a paged cache, and attention over the
rows that the model's cache holds, against the attention output of its step
kernel."""
import ctypes as C

import numpy as np
import pytest

from conftest import MODEL_CACHE

import krafla_b200 as kb
import serving_ref as ref

pytestmark = pytest.mark.gpu

KV = {"f32": kb.F32, "f16": kb.F16, "q8": kb.Q8_0}
DT = {"f32": np.float32, "f16": np.float16, "q8": np.int8}


@pytest.fixture(scope="module")
def model(built):
    kb.device_check()
    return kb.Model(kb.ensure_model("cfg0", MODEL_CACHE))


def debug(st, which, dtype, n):
    out = np.empty(n, dtype)
    kb._check(kb.lib().kc_debug_copy(st._h, which, out.ctypes.data_as(C.c_void_p), out.nbytes), "debug copy")
    return out


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
def test_rows_and_attention_of_the_model(model, kv):
    c = model.config
    heads, hk, hd, layers, top = c["n_heads"], c["n_kv_heads"], c["head_dim"], c["n_layers"], c["max_seq"]
    steps, page = 41, 16
    st = kb.State(model, kv_type=KV[kv])
    tok, rows = 3, []
    for t in range(steps):
        tok = int(np.argmax(st.forward(tok, t)))
        rows.append(debug(st, 1, np.float32, (heads + 2 * hk) * hd))
    x = np.stack(rows)                                         # the last layer's q|k|v of every step
    model_out = debug(st, 2, np.float32, heads * hd)           # and its attention output at the last one, in 8 bits
    mk, mv = (debug(st, w, DT[kv], layers * top * hk * hd).reshape(layers, top, hk, hd)[-1, :steps] for w in (4, 5))
    ms = [debug(st, w, np.float32, layers * top * hk).reshape(layers, top, hk)[-1, :steps] for w in (6, 7)] if kv == "q8" else None
    n_pages = -(-steps // page)
    table = np.arange(n_pages, dtype=np.int32)[None, ::-1].copy()

    def paged(a):
        """[steps, hk, ...] into the pool's [page][hk][slot]."""
        p = np.zeros((n_pages, hk, page, *a.shape[2:]), a.dtype)
        for t in range(steps):
            p[table[0, t // page], :, t % page] = a[t]
        return p

    cos, sin = kb.rope_tables(c, steps)
    pools = [kb.DevArray.of(np.zeros_like(paged(a))) for a in (mk, mv, *(ms or []))]
    cache = kb.PagedKV(pools[0], pools[1], kb.DevArray.of(table), KV[kv], *pools[2:], n_heads=heads)
    pos = np.arange(steps, dtype=np.int32)
    q = cache.append(kb.DevArray.of(x), kb.DevArray.of(pos), kb.DevArray.of(cos), kb.DevArray.of(sin),
                     kb.DevArray((steps, heads, hd), np.float32), seqs=kb.DevArray.of(np.zeros(steps, np.int32)))
    kb._check(kb.lib().kc_dev_sync(), "sync")
    got = [p.numpy() for p in pools]
    want = [paged(a) for a in (mk, mv, *(ms or []))]
    # V is not rotated: the same bits. A rotated value is two products and their sum on both sides, each within
    # 3 half steps of 32 bits of the pair's size; then a rounding to the cache's type, which may fall on either side.
    assert np.array_equal(got[1], want[1])
    size = np.abs(x).max() * np.sqrt(2)
    err = 6 * 2.0 ** -24 * size
    if kv == "q8":
        assert np.array_equal(got[3], want[3])
        assert (np.abs(got[2] - want[2]) <= err / 127 + 2.0 ** -23 * want[2]).all()
        assert (np.abs(got[0].astype(int) - want[0]) <= 1).all() and (got[0] != want[0]).mean() < 1e-3
    else:
        step = np.finfo(DT[kv]).eps * np.abs(want[0].astype(float)) if kv == "f16" else 0
        assert (np.abs(got[0].astype(float) - want[0]) <= err + step).all()
    # attention over the model's own rows; both sides within the bound of test_serving_gpu, then the model's 8 bits a
    # value (one scale for 32 of them)
    dev = [kb.DevArray.of(a) for a in want]
    cache = kb.PagedKV(dev[0], dev[1], kb.DevArray.of(table), KV[kv], *dev[2:], n_heads=heads)
    last = np.ascontiguousarray(q.numpy()[-1:])
    o = cache.attend(kb.DevArray.of(last), kb.DevArray.of(np.array([steps], np.int32)), kb.DevArray((1, heads, hd), np.float32)).numpy()
    k, v, kd, vd = (want + [None, None])[:4]
    _, reach = ref.attend(last, k, v, table, [steps], hd ** -0.5, 0, 0.0, kd, vd)
    vmax = np.abs(v.astype(float)).max() if kd is None else (127 * vd).max()
    d = (2.0 ** -21 + hd * 2.0 ** -23 + 2.0 ** -22) * reach.max()
    tol = 2 * vmax * 2 * (2 * d + 2.0 ** -20 + (steps / 8 + 1) * 2.0 ** -23)
    blocks, mo = o.reshape(-1, 32), model_out.reshape(-1, 32)
    half = (np.abs(blocks).max(-1, keepdims=True) + tol) / 127 / 2
    assert (np.abs(blocks - mo) <= half * (1 + 2.0 ** -20) + tol).all()
