"""Serving operators on the GPU at edges that the tests beside this one leave
out. Tolerances of attention: test_serving_gpu's."""
import numpy as np
import pytest

import krafla_b200 as kb
import serving_ref as ref
from test_serving_gpu import check, handle, make_pool, make_table, spoil

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _dev(built):
    kb.device_check()


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("heads,hk,hd", [(12, 3, 256), (9, 1, 192), (4, 4, 144)])
def test_attend_wide_heads_tile_by_tile(kv, heads, hk, hd):
    """Wide heads of more than 8 units keep one tile a warp at a time: what a tile holds (its unit, its mask, whether
    it is the last) is another in every pass. Lengths of every remainder of a quantum, so that masks differ between
    warps and between passes, units that begin and end in the middle of a share, and warps without a tile; the same
    call many times gives the same bits."""
    rng = np.random.default_rng(heads + hd)
    page = 8
    lens = [*range(1, 70, 3), *rng.integers(1, 600, 90).tolist(), 0, 0, *rng.integers(200, 900, 30).tolist()]
    n_pages = sum(-(-m // page) for m in lens)
    pools = make_pool(rng, kv, n_pages, hk, page, hd)
    table = make_table(rng, lens, page, n_pages)
    spoil(pools, table, lens, page)
    q = rng.standard_normal((len(lens), heads, hd)).astype(np.float32)
    c = handle(pools, table, kv, heads)
    dq, dl = kb.DevArray.of(q), kb.DevArray.of(np.array(lens, np.int32))
    k, v, kd, vd = pools
    vmax = np.nanmax(np.abs(v.astype(np.float64))) if kd is None else np.nanmax(127 * vd)
    first = None
    for _ in range(20):
        out = c.attend(dq, dl, kb.DevArray.of(np.full(q.shape, np.nan, np.float32))).numpy()
        first = out if first is None else first
        assert np.array_equal(out, first)
    kb._check(kb.lib().kc_dev_sync(), "sync")
    want, reach = ref.attend(q, k, v, table, lens, hd ** -0.5, 0, 0.0, kd, vd)
    check(first, want, reach, vmax, hd, max(lens))


def test_attend_8bit_weights_do_not_lose_bits_to_small_scales():
    """Rows whose scales are near 1e-30: half of the positions have V = v and score 0, half -v and a score x / log2 e
    with x = 3.7e-6, so the output is v (w_0 - w_x) / (w_0 + w_x) = -v 1.28e-6. A weight keeps its 22 bits whatever V's
    scale is. Errors against v, of two weights near 1, half of each: 2^-22 each for exp2 and for the two halves of 11
    bits, 2^-24 for the product with the scale; 2^-22 for the sums, which stay small since the signs alternate. In all
    below 2^-20. (Weights rounded at the size of a lift of 2^114 would come out equal, and the output 0.)"""
    hd, page, n, x = 64, 16, 512, 3.7e-6
    k = np.zeros((n // page, 1, page, hd), np.int8)
    k[..., 0] = 1
    v = np.full(k.shape, 127, np.int8)
    v[:, :, 1::2] = -127
    kd = np.zeros(k.shape[:3], np.float32)
    kd[:, :, 1::2] = 1.0
    vd = np.full(k.shape[:3], 2.0 ** -100, np.float32)
    q = np.zeros((1, 1, hd), np.float32)
    q[0, 0, 0] = 1.0
    table = np.arange(n // page, dtype=np.int32)[None]
    c = handle((k, v, kd, vd), table, "q8", 1)
    scale = x * np.log(2.0)
    out = c.attend(kb.DevArray.of(q), kb.DevArray.of(np.array([n], np.int32)), kb.DevArray(q.shape, np.float32), scale=scale)
    want, _ = ref.attend(q, k, v, table, [n], float(np.float32(scale)), 0, 0.0, kd, vd)
    top = 127 * 2.0 ** -100
    assert np.allclose(want / top, -1.28e-6, rtol=0.01)
    assert (np.abs(out.numpy() - want) <= 2.0 ** -20 * top).all()


FIRST_USE = """
import sys, threading
sys.path[:0] = {paths!r}
import numpy as np
import krafla_b200 as kb
kb.lib()
n, heads, hk, hd, page = 3, 8, 2, 64, 16
rng = np.random.default_rng(0)
k, v = (kb.DevArray.of(rng.standard_normal((6, hk, page, hd)).astype(np.float16)) for _ in range(2))
table = kb.DevArray.of(np.arange(6, dtype=np.int32).reshape(n, 2))
q, lens = kb.DevArray.of(rng.standard_normal((n, heads, hd)).astype(np.float32)), kb.DevArray.of(np.array([5, 32, 17], np.int32))
go, outs, errors = threading.Barrier(24), [None] * 24, []

def first(i):
    out = kb.DevArray(q.shape, np.float32)
    go.wait()
    try:
        outs[i] = kb.PagedKV(k, v, table, kb.F16, n_heads=heads).attend(q, lens, out)
    except Exception as e:
        errors.append(e)

ts = [threading.Thread(target=first, args=(i,)) for i in range(24)]
[t.start() for t in ts]
[t.join() for t in ts]
kb._check(kb.lib().kc_dev_sync(), "sync")
assert not errors, errors
assert all(np.array_equal(o.numpy(), outs[0].numpy()) for o in outs)
print("same")
"""


def test_first_use_by_many_threads():
    """24 threads make a process's first calls at once, each with a handle of its own."""
    import subprocess
    import sys
    for _ in range(3):
        r = subprocess.run([sys.executable, "-c", FIRST_USE.format(paths=sys.path)], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


FIRST_IN_A_GRAPH = """
import sys
sys.path[:0] = {paths!r}
import torch
import krafla_b200 as kb
n, heads, hk, hd, page, vocab = 3, 8, 2, 64, 16, 5000
g = torch.Generator().manual_seed(0)
k, v = (torch.randn(6, hk, page, hd, generator=g).half().cuda() for _ in range(2))
table = torch.arange(6, dtype=torch.int32).reshape(n, 2).cuda()
c = kb.PagedKV(k, v, table, kb.F16, n_heads=heads)
cos, sin = (torch.from_numpy(t).cuda() for t in kb.rope_tables(dict(head_dim=hd, rope_theta=1e4), 32))
x = torch.randn(n, (heads + 2 * hk) * hd, generator=g).cuda()
pos = torch.tensor([5, 31, 16], dtype=torch.int32).cuda()
lens = pos + 1
q, o = torch.zeros(n, heads, hd).cuda(), torch.zeros(n, heads, hd).cuda()
z = torch.randn(n, vocab, generator=g).cuda()
y, w = torch.zeros_like(z), torch.zeros_like(z)
mask = torch.randint(0, 2 ** 31, (n, (vocab + 31) // 32), generator=g, dtype=torch.int32).cuda()
hist, rep = torch.randint(0, vocab, (n, 40), generator=g, dtype=torch.int32).cuda(), torch.full((n,), 1.5).cuda()
kb.process_logits(w, z)                                       # a first call, of the plainest kind
st = torch.cuda.Stream()

def step():
    c.append(x, pos, cos, sin, q, stream=st.cuda_stream)
    c.attend(q, lens, o, stream=st.cuda_stream)
    kb.process_logits(y, z, history=hist, repeat=rep, mask=mask, stream=st.cuda_stream)

torch.cuda.synchronize()
gr = torch.cuda.CUDAGraph()
with torch.cuda.graph(gr, stream=st):
    step()
assert not q.any() and not o.any() and not y.any()
gr.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (q, o, y)]
step()
torch.cuda.synchronize()
kb._check(kb.lib().kc_dev_sync(), "sync")
assert all(torch.equal(a, b) for a, b in zip(got, (q, o, y))) and q.any() and o.any() and y.any()
del gr
print("same")
"""


def test_first_calls_inside_a_capture():
    """A process that has made a PagedKV and one plain call of process_logits captures the rest unseen."""
    pytest.importorskip("torch")
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_GRAPH.format(paths=sys.path)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]
