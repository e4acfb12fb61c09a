"""The serving operators' refusals and host parts, without a GPU: sizes and
types that the C entries and the Python wrappers turn down before any launch."""
import ctypes as C

import numpy as np
import pytest

import krafla_b200 as kb
import serving_ref as ref


@pytest.fixture(scope="module", autouse=True)
def _built(built):
    return built


P = 4096   # an address that no check before the device's reads


def cache(**kw):
    d = dict(k=P, v=P, kd=None, vd=None, table=P, n_seqs=4, ld_table=8, n_pages=32, page_size=16, n_kv_heads=2,
             head_dim=64, kv_type=kb.F16)
    d.update(kw)
    return kb._PagedKV(*[d[n] for n, _ in kb._PagedKV._fields_])


def refused(fn, *structs):
    st = fn(*[s if isinstance(s, bytes) else C.byref(s) for s in structs], None)
    return st == kb.E_SHAPE and kb.what_detail()


@pytest.mark.parametrize("kw,word", [
    (dict(kv_type=kb.Q4_0), "kv_type"), (dict(head_dim=24), "head_dim"), (dict(head_dim=272), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(n_pages=0), "n_pages"), (dict(page_size=-1), "page_size"),
    (dict(n_pages=1 << 26, page_size=64), "2^32"), (dict(ld_table=1 << 28), "2^31"), (dict(n_seqs=0), "n_seqs")])
def test_cache_sizes_are_refused(kw, word):
    L = kb.lib()
    for fn, a in ((L.kc_paged_append_dev, bytes(256)), (L.kc_paged_attend_dev, bytes(256))):
        assert word in refused(fn, cache(**kw), a)
    n = C.c_size_t()
    assert L.kc_paged_attend_ws(C.byref(cache(**kw)), 4, C.byref(n)) == kb.E_SHAPE


def attend_args(**kw):
    d = dict(q=P, out=P, ldq=256, ldo=256, lens=P, n_seqs=4, n_heads=4, window=0, scale=0.1, softcap=0.0, ws=P, ws_bytes=0)
    d.update(kw)
    return kb._ATTEND.pack(*[d[n] for n in kb._ATTEND.names])


@pytest.mark.parametrize("kw,word", [
    (dict(n_heads=3), "n_heads"), (dict(n_heads=0), "n_heads"), (dict(n_seqs=5), "n_seqs"), (dict(n_seqs=-1), "n_seqs"),
    (dict(ldq=254), "multiples of 4"), (dict(ldo=128), "shorter"), (dict(window=-1), "window"),
    (dict(scale=float("nan")), "scale"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap")])
def test_attend_is_refused(kw, word):
    assert word in refused(kb.lib().kc_paged_attend_dev, cache(), attend_args(**kw))


def append_args(**kw):
    d = dict(q=P, k=P, v=P, q_out=P, ldq=512, ldk=512, ldv=512, ldo=256, cos=P, sin=P, q_norm=0, k_norm=0, seqs=P,
             pos=P, rows=9, n_heads=4, n_pos=100, eps=1e-5)
    d.update(kw)
    return kb._APPEND.pack(*[d[n] for n in kb._APPEND.names])


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "rows"), (dict(n_heads=0), "n_heads"), (dict(n_pos=0), "n_pos"), (dict(ldk=130), "multiples of 4"),
    (dict(ldv=64), "shorter"), (dict(q_norm=P), "together"), (dict(eps=float("nan")), "eps"), (dict(eps=-1.0), "eps"),
    (dict(seqs=0), "more rows"), (dict(rows=1 << 30), "too many")])
def test_append_is_refused(kw, word):
    assert word in refused(kb.lib().kc_paged_append_dev, cache(), append_args(**kw))


def test_append_in_place_needs_one_stride():
    assert "in place" in refused(kb.lib().kc_paged_append_dev, cache(), append_args())


def logits_args(**kw):
    d = dict({n: 0 for n in kb._LOGITS.names}, out=P, ld_in=100, ld_out=100, rows=3, vocab=100)
    d["in"] = P
    d.update(kw)
    return kb._LOGITS.pack(*[d[n] for n in kb._LOGITS.names])


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 27) + 1), "vocab"), (dict(ld_in=99), "shorter"),
    (dict(history=P, history_cap=9, ld_history=8), "history_cap"), (dict(history_cap=2), "history"),
    (dict(bias_off=P, n_bias=3), "biases"), (dict(bias_ids=P, n_bias=3), "biases"), (dict(bias_off=P, n_bias=-1), "biases"),
    (dict(mask=P, ld_mask=3), "mask"), (dict(ld_out=104), "in place")])
def test_logits_are_refused(kw, word):
    assert word in refused(kb.lib().kc_logits_process_dev, logits_args(**kw))


class Fake:
    """An array with a type and strides and no memory."""

    def __init__(self, shape, dtype, stride=None):
        self.shape, self.dtype = tuple(shape), np.dtype(dtype)
        self._s = stride or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))

    def stride(self):
        return self._s

    def data_ptr(self):
        return P


@pytest.mark.parametrize("kw,word", [
    (dict(logits=Fake((2, 50), "float64")), "float64"), (dict(logits=Fake((50,), "float32")), "rows, vocab"),
    (dict(out=Fake((3, 50), "float32")), "out"), (dict(logits=Fake((2, 50), "float32", (100, 2))), "contiguous"),
    (dict(history=Fake((3, 5), "int32")), "history"), (dict(repeat=Fake((2,), "float32")), "history"),
    (dict(history=Fake((2, 5), "int32"), repeat=Fake((3,), "float32")), "repeat"),
    (dict(bias_off=Fake((2,), "int32")), "bias_off"), (dict(mask=Fake((2, 1), "int32")), "mask"),
    (dict(mask=Fake((2, 2), "float32")), "mask")])
def test_python_logits_refusals(kw, word):
    d = dict(out=Fake((2, 50), "float32"), logits=Fake((2, 50), "float32"))
    d.update(kw)
    with pytest.raises(kb.KraflaError, match=word) as e:
        kb.process_logits(**d)
    assert e.value.status == kb.E_SHAPE


@pytest.mark.parametrize("kw,word", [
    (dict(k=Fake((8, 2, 16, 64), "float32")), "float32"), (dict(k=Fake((8, 2, 64), "float16")), "n_pages"),
    (dict(v=Fake((8, 2, 16, 32), "float16")), "v is"), (dict(kd=Fake((8, 2, 16), "float32")), "scales"),
    (dict(table=Fake((4,), "int32")), "table"), (dict(table=Fake((4, 3), "int64")), "int64"),
    (dict(kv_type=kb.Q8_0, k=Fake((8, 2, 16, 64), "int8")), "scales"), (dict(kv_type=7), "kv_type"),
    (dict(k=Fake((8, 2, 16, 64), "float16", (2048, 64, 128, 1))), "contiguous")])
def test_python_cache_refusals(kw, word):
    d = dict(k=Fake((8, 2, 16, 64), "float16"), v=Fake((8, 2, 16, 64), "float16"), table=Fake((4, 3), "int32"), kv_type=kb.F16)
    d.update(kw)
    with pytest.raises(kb.KraflaError, match=word):
        kb.PagedKV(d.pop("k"), d.pop("v"), d.pop("table"), d.pop("kv_type"), **d)


def test_rope_tables():
    cfg = dict(head_dim=64, rope_theta=5e5)
    cos, sin = kb.rope_tables(cfg, 300)
    ang = np.arange(300)[:, None] * 5e5 ** (-np.arange(0, 64, 2) / 64)
    # float's half step, and the angle's own (a few of 2^-53 times 299)
    assert np.abs(cos - np.cos(ang)).max() <= 2.0 ** -24 and np.abs(sin - np.sin(ang)).max() <= 2.0 ** -24
    lin, _ = kb.rope_tables(dict(cfg, rope_type=2, rope_factor=4.0), 300)
    assert np.abs(lin - np.cos(ang / 4)).max() <= 2.0 ** -24
    loc, _ = kb.rope_tables(dict(cfg, rope_type=2, rope_factor=4.0, rope_local_theta=1e4), 300, local=True)
    assert np.abs(loc - np.cos(np.arange(300)[:, None] * 1e4 ** (-np.arange(0, 64, 2) / 64))).max() <= 2.0 ** -24
    for bad in (dict(head_dim=63, rope_theta=1e4), dict(head_dim=64), dict(rope_theta=1e4)):
        with pytest.raises(kb.KraflaError):
            kb.rope_tables(bad, 4)


def test_reference_rows():
    """The restatement's own rules at values where they can go wrong."""
    q, d = ref.quant_rows(np.array([[127, 0.5, -0.5, 1.5, -2.5], [1e-31, 0, 0, 0, 0]], np.float32))
    assert q.tolist() == [[127, 1, -1, 2, -3], [0] * 5] and d[:, 0].tolist() == [1, 0]
    z = ref.logits(np.array([[2.0, -2.0, 1.0]], np.float32), history=np.array([[0, 1, 1, -1, 9]]), repeat=[2.0],
                   frequency=[1.0], presence=[0.5], bias=[(np.array([2, 2]), np.array([5.0, 7.0]))])
    assert z.tolist() == [[1 - 1 - 0.5, -4 - 2 - 0.5, 8]]
