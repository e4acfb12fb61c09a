"""Cases of the serving operators over several sequences: the paged KV cache
(norm, rotation and append of new rows; attention of one new token per
sequence) and the processing of logits before a token is chosen.

With `own` false, run() computes an operator in its plain form from elementary
torch operations; with `own` true it calls krafla_b200. Head layouts, vocabulary
sizes and lengths are those of this repository's model configurations
(isa-lm_b200/krafla_models.py) or generic ones.

A case of `attend`: n_seqs sequences whose lengths are spread evenly from len_lo
to len_hi (their order comes from the seed), each with its own pages of a shared
pool. A case of `append`: `rows` new rows, either one each for `n_seqs`
sequences or stretches of consecutive positions, some of them padding. A case of
`logits`: `rows` rows of logits with their own histories, penalties, biases and
allowed tokens.
"""
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "isa-lm_b200")
_NEG = float("-inf")
_BYTES = {"f32": 4, "f16": 2, "q8": 1}


def _kb():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import krafla_b200
    return krafla_b200


# ------------------------------------------------------------------ the cases

def _attend(name, kv, heads, kv_heads, hd, page, n_seqs, len_lo, len_hi, window=0, softcap=0.0):
    c = dict(op="attend", kv=kv, heads=heads, kv_heads=kv_heads, hd=hd, page=page, n_seqs=n_seqs, len_lo=len_lo,
             len_hi=len_hi, window=window, softcap=softcap)
    return dict(c, name=name) if name else c


def _append(name, kv, heads, kv_heads, hd, page, rows, n_seqs, norm, pad):
    c = dict(op="append", kv=kv, heads=heads, kv_heads=kv_heads, hd=hd, page=page, rows=rows, n_seqs=n_seqs, norm=norm,
             pad=pad)
    return dict(c, name=name) if name else c


def _logits(name, rows, vocab, hist, bias, mask, count):
    c = dict(op="logits", rows=rows, vocab=vocab, hist=hist, bias=bias, mask=mask, count=count)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one conversation at the shortest context the decode benchmark quotes: latency only
        _attend("attend_one_short", "f32", 32, 8, 64, 16, 1, 128, 128),
        # one conversation at the same model's longest context
        _attend("attend_one_full", "f32", 32, 8, 64, 16, 1, 4096, 4096),
        # two very long documents, the whole machine on two sequences
        _attend("attend_long_f16", "f16", 32, 8, 128, 64, 2, 120001, 131072),
        # a busy server: 64 conversations of mixed length on the 8B shape
        _attend("attend_batch_f16", "f16", 32, 8, 128, 16, 64, 2048, 8192),
        # many short and middling conversations, 8-bit cache, seven heads to a KV head
        _attend("attend_batch_q8", "q8", 14, 2, 64, 32, 96, 1, 4097),
        # a sliding-window layer with soft-capped scores, heads without sharing, a head of 48
        _attend("attend_window_f32", "f32", 6, 6, 48, 8, 13, 100, 2011, window=257, softcap=50.0),
        # a decode step's new rows, one for each of 64 sequences
        _append("append_step_f16", "f16", 14, 2, 64, 32, 64, 64, False, 0),
        # prompts: four full prefill chunks of the 8B shape
        _append("append_prompt_f16", "f16", 32, 8, 128, 16, 4096, 3, False, 0),
        # a padded batch of prompts into an 8-bit cache, heads normed
        _append("append_ragged_q8", "q8", 32, 8, 128, 64, 1531, 5, True, 77),
        # one row, the penalty of the device sampler alone: latency only
        _logits("logits_one", 1, 32000, 64, 0, False, False),
        # a batch where every request has a history, biases and a grammar
        _logits("logits_batch", 64, 128256, 2048, 100, True, True),
        # a few rows, a vocabulary that no vector width divides, a grammar only
        _logits("logits_odd", 9, 151937, 0, 0, True, False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "logits"])
    kv = rng.choice(["f32", "f16", "q8"])
    heads, kv_heads = rng.choice([(32, 8), (14, 2), (6, 6), (32, 4), (16, 1), (24, 8), (40, 2)])
    hd = rng.choice([48, 64, 64, 80, 128, 128, 256])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if op == "attend":
        n_seqs = _log_int(rng, 1, 200)
        per = 2 * kv_heads * hd * _BYTES[kv]
        top = max(16, min(131072, int(6e8 / (per * n_seqs)), int(2.0e8 / (kv_heads * hd * n_seqs))))
        hi = _log_int(rng, 16, top) + rng.randrange(2)
        lo = rng.choice([hi, max(1, hi // 3), 1])
        window = rng.choice([0, 0, 0, _log_int(rng, 1, 2 * hi)])
        return _attend(None, kv, heads, kv_heads, hd, page, n_seqs, lo, hi, window, rng.choice([0.0, 0.0, 30.0]))
    if op == "append":
        top = max(2, min(4096, int(4096 * 6144 / ((heads + 2 * kv_heads) * hd))))
        rows = _log_int(rng, 1, top)
        step = rng.random() < 0.4
        rows = min(rows, 256) if step else rows
        return _append(None, kv, heads, kv_heads, hd, page, rows, rows if step else rng.randrange(1, min(rows, 9) + 1),
                       rng.random() < 0.5, rng.choice([0, rows // 20]))
    vocab = _log_int(rng, 500, 200000) | rng.randrange(2)
    rows = _log_int(rng, 1, max(1, min(128, int(64 * 128256 / vocab))))
    hist, bias = rng.choice([0, _log_int(rng, 1, 4000)]), rng.choice([0, _log_int(rng, 1, 300)])
    return _logits(None, rows, vocab, hist, bias, rng.random() < 0.5 or not (hist or bias), hist > 0 and rng.random() < 0.6)


# ------------------------------------------------------------------ the inputs

def _lens(c):
    return np.rint(np.linspace(c["len_lo"], c["len_hi"], c["n_seqs"])).astype(np.int64)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _pool(c, n_pages, g):
    """K and V of a pool [page][kv head][slot][head dim], Q8 with a scale for each row of a head."""
    shape = (n_pages, c["kv_heads"], c["page"], c["hd"])
    if c["kv"] == "q8":
        kv = [torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8) for _ in range(2)]
        sc = [(0.01 + 0.01 * torch.rand(shape[:3], generator=g, device="cuda")) for _ in range(2)]
        return kv + sc
    dt = torch.float16 if c["kv"] == "f16" else torch.float32
    return [_randn(shape, g, dt), _randn(shape, g, dt), None, None]


def _table(need, page, n_pages, rng):
    """Pages of each sequence in a random order of the pool's pages 1.. (page 0 is nobody's); -1 where it has none."""
    pages = -(-need // page)
    ids = 1 + rng.permutation(n_pages - 1)
    t = np.full((len(need), int(pages.max())), -1, np.int32)
    at = 0
    for i, k in enumerate(pages):
        t[i, :k] = ids[at:at + k]
        at += k
    return torch.from_numpy(t).cuda()


def prepare(case, seed):
    c, g, rng = case, _gen(seed), np.random.default_rng(seed)
    s = {"case": c}
    if c["op"] == "logits":
        n, v = c["rows"], c["vocab"]
        s["logits"] = 4 * _randn((n, v), g)
        s["out"] = torch.empty_like(s["logits"])
        if c["hist"]:
            # half of a history repeats a few tokens, as text does; -1 pads
            h = rng.integers(0, v, (n, c["hist"]))
            h = np.where(rng.random(h.shape) < 0.5, h[:, :1] // 2 + h % min(v - v // 2, 50), h)
            ln = rng.integers(c["hist"] // 2, c["hist"] + 1, n)
            h[np.arange(c["hist"])[None] >= ln[:, None]] = -1
            s["history"] = torch.from_numpy(h.astype(np.int32)).cuda()
            s["history_len"] = torch.from_numpy(ln.astype(np.int32)).cuda()
            s["repeat"] = torch.from_numpy(rng.uniform(1.0, 1.5, n).astype(np.float32)).cuda()
            if c["count"]:
                s["presence"] = torch.from_numpy(rng.uniform(-0.5, 1.0, n).astype(np.float32)).cuda()
                s["frequency"] = torch.from_numpy(rng.uniform(0.0, 0.5, n).astype(np.float32)).cuda()
        if c["bias"]:
            k = rng.integers(0, c["bias"] + 1, n)
            k[0] = c["bias"]
            s["bias_off"] = torch.from_numpy(np.concatenate([[0], np.cumsum(k)]).astype(np.int32)).cuda()
            s["bias_ids"] = torch.from_numpy(rng.integers(0, v, int(k.sum())).astype(np.int32)).cuda()
            s["bias_vals"] = torch.from_numpy(rng.normal(0, 5, int(k.sum())).astype(np.float32)).cuda()
        if c["mask"]:
            # a grammar allows few tokens in some rows and most in others
            share = rng.choice([0.001, 0.3, 0.95], n)
            words = -(-v // 32)
            bits = torch.rand((n, words * 32), generator=g, device="cuda") < torch.from_numpy(share).cuda()[:, None]
            two = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], dtype=torch.int64, device="cuda")
            s["mask"] = (bits.view(n, words, 32) * two).sum(2).to(torch.int32)
        return s
    hd, hk, page = c["hd"], c["kv_heads"], c["page"]
    if c["op"] == "attend":
        lens = rng.permutation(_lens(c))
        n_pages = 1 + int((-(-lens // page)).sum())
        s["k"], s["v"], s["kd"], s["vd"] = _pool(c, n_pages, g)
        s["table"] = _table(lens, page, n_pages, rng)
        s["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        s["q"] = _randn((c["n_seqs"], c["heads"], hd), g)
        s["scale"] = hd ** -0.5
        s["out"] = torch.empty_like(s["q"])
    else:
        n, b = c["rows"], c["n_seqs"]
        where = np.random.default_rng(n + 10007 * b)   # the positions are the case's, so that the pool's size is too
        if b == n:   # a decode step: one row each, somewhere in its sequence
            seqs, pos = np.arange(n), where.integers(0, max(2, min(700, 16384 // n)), n)
        else:        # stretches of prompts, each from a position of its own
            cut = np.sort(where.choice(np.arange(1, n), b - 1, replace=False)) if b > 1 else np.zeros(0, np.int64)
            seqs = np.searchsorted(cut, np.arange(n), side="right")
            begin = np.concatenate([[0], cut])
            pos = where.integers(0, 100, b)[seqs] + np.arange(n) - begin[seqs]
        need = np.zeros(b, np.int64)
        np.maximum.at(need, seqs, pos + 1)
        if c["pad"]:
            seqs = seqs.copy()
            seqs[n - c["pad"]:] = -1
        n_pages = 1 + int((-(-need // page)).sum())
        s["k"], s["v"], s["kd"], s["vd"] = _pool(c, n_pages, g)
        s["table"] = _table(need, page, n_pages, rng)
        s["seqs"] = torch.from_numpy(seqs.astype(np.int32)).cuda()
        s["pos"] = torch.from_numpy(pos.astype(np.int32)).cuda()
        s["qkv"] = _randn((n, (c["heads"] + 2 * hk) * hd), g)
        s["q_out"] = torch.zeros((n, c["heads"], hd), device="cuda")
        s["q_norm"] = 1 + 0.1 * _randn((hd,), g) if c["norm"] else None
        s["k_norm"] = 1 + 0.1 * _randn((hd,), g) if c["norm"] else None
        ang = torch.arange(int(pos.max()) + 1, device="cuda", dtype=torch.float64)[:, None] * (
            5e5 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd))
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["eps"] = 1e-5
    if own:   # the handle a program keeps beside its pool: pointers and sizes, no data
        kb = _kb()
        s["cache"] = kb.PagedKV(s["k"], s["v"], s["table"], {"f32": kb.F32, "f16": kb.F16, "q8": kb.Q8_0}[c["kv"]],
                                kd=s["kd"], vd=s["vd"], n_heads=c["heads"])
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    op = s["case"]["op"]
    if op == "logits":
        return _logits_own(s) if own else _logits_plain(s)
    if op == "attend":
        return _attend_own(s) if own else _attend_plain(s)
    if own:
        q = _append_own(s)
    else:
        q = _append_plain(s)
    if s["kd"] is None:
        return q, s["k"], s["v"]
    return q, s["k"] * s["kd"][..., None], s["v"] * s["vd"][..., None]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _attend_own(s):
    s["cache"].attend(s["q"], s["lens"], s["out"], scale=s["scale"], window=s["case"]["window"],
                      softcap=s["case"]["softcap"], stream=_stream())
    return s["out"]


def _append_own(s):
    s["cache"].append(s["qkv"], s["pos"], s["cos"], s["sin"], s["q_out"], seqs=s["seqs"], q_norm=s["q_norm"],
                      k_norm=s["k_norm"], eps=s["eps"], stream=_stream())
    return s["q_out"]


def _logits_own(s):
    _kb().process_logits(s["out"], s["logits"], history=s.get("history"), history_len=s.get("history_len"),
                         repeat=s.get("repeat"), presence=s.get("presence"), frequency=s.get("frequency"),
                         bias_off=s.get("bias_off"), bias_ids=s.get("bias_ids"), bias_vals=s.get("bias_vals"),
                         mask=s.get("mask"), stream=_stream())
    return s["out"]


def _quant_rows(x):
    """The 8-bit rule of a cache row in 32 bits: d = max|x| / 127, q = x * (127 / max|x|) rounded half away from zero."""
    amax = x.abs().amax(-1, keepdim=True)
    some = amax >= 1e-30
    top = torch.full_like(amax, 127.0)   # a tensor: a division by a number would multiply by its rounded inverse
    r = x * torch.where(some, top / amax, 0.0)
    q = torch.trunc(r + torch.copysign(torch.full_like(r, 0.5), x)).clamp(-127, 127)
    return torch.where(some, q, 0.0), torch.where(some, amax / top, 0.0)


def _attend_plain(s):
    c = s["case"]
    b, h, hd = s["q"].shape
    hk = c["kv_heads"]
    idx = s["table"].clamp(min=0).long()
    flat = lambda t: t[idx].transpose(1, 2).flatten(2, 3)   # noqa: E731  [B][kv head][position](...)
    k, v = flat(s["k"]).float(), flat(s["v"]).float()
    length = s["lens"].long()[:, None]
    at = torch.arange(k.shape[2], device="cuda")[None]
    seen = at < length
    if c["window"]:
        seen = seen & (at >= length - c["window"])
    q = s["q"].view(b, hk, h // hk, hd)
    if s["kd"] is not None:
        q, qd = _quant_rows(q)
        score = (q @ k.transpose(2, 3)) * (qd * s["scale"]) * flat(s["kd"])[:, :, None]
        v = v * flat(s["vd"])[..., None]
    else:
        score = (q @ k.transpose(2, 3)) * s["scale"]
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    score = score.masked_fill(~seen[:, None, None], _NEG)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == _NEG, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill(~seen[:, None, :, None], 0.0)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    return out.reshape(b, h, hd)


def _rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _append_plain(s):
    c = s["case"]
    n, h, hk, hd = c["rows"], c["heads"], c["kv_heads"], c["hd"]
    q, k, v = s["qkv"].view(n, h + 2 * hk, hd).split([h, hk, hk], 1)
    if c["kv"] == "q8":
        k = k.double()   # an 8-bit rounding follows: values next to a border
    if s["q_norm"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + s["eps"]) * s["q_norm"]
        k = k * (1.0 / torch.sqrt((k * k).mean(-1, keepdim=True) + s["eps"])) * s["k_norm"]
    pos, live = s["pos"].long(), s["seqs"] >= 0
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    q = torch.where(live[:, None, None], q, s["q_out"])
    page = s["table"][s["seqs"].long().clamp(min=0), pos // c["page"]].long()
    page = torch.where(live, page, 0)          # padding writes back what page 0, nobody's, holds
    slot = torch.where(live, pos % c["page"], 0)
    keep = live[:, None, None]
    for x, pool, scale in ((k, s["k"], s["kd"]), (v, s["v"], s["vd"])):
        x = x.float()
        if scale is not None:
            x, d = _quant_rows(x)
            scale[page, :, slot] = torch.where(keep[..., 0], d[..., 0], scale[0, :, 0])
        pool[page, :, slot] = torch.where(keep, x.to(pool.dtype), pool[0, :, 0])
    return q


def _logits_plain(s):
    z = s["logits"]
    n, v = z.shape
    if "history" in s:
        h = s["history"].long()
        used = (torch.arange(h.shape[1], device="cuda")[None] < s["history_len"][:, None]) & (h >= 0)
        count = torch.zeros((n, v + 1), device="cuda").scatter_add_(1, torch.where(used, h, v), torch.ones_like(h, dtype=torch.float32))[:, :v]
        r = s["repeat"][:, None]
        z = torch.where(count > 0, torch.where(z > 0, z / r, z * r), z)
        if "presence" in s:
            z = z - s["frequency"][:, None] * count
            z = z - torch.where(count > 0, s["presence"][:, None], 0.0)
    if "bias_off" in s:
        off = s["bias_off"].long()
        m = s["bias_ids"].numel()
        row = torch.repeat_interleave(torch.arange(n, device="cuda"), off[1:] - off[:-1], output_size=m)
        entry = torch.arange(m, device="cuda")
        last = torch.full((n * v,), -1, device="cuda").scatter_reduce_(0, row * v + s["bias_ids"].long(), entry, "amax").view(n, v)
        z = torch.where(last >= 0, z + s["bias_vals"][last.clamp(min=0)], z)
    if "mask" in s:
        at = torch.arange(v, device="cuda")
        z = z.masked_fill((s["mask"][:, at // 32] >> (at % 32)) & 1 == 0, _NEG)
    return z


# ------------------------------------------------------------------ what a pass cannot do without

def work(c):
    if c["op"] == "logits":
        n, v = c["rows"], c["vocab"]
        b = 8 * n * v + 4 * n * c["hist"] + 8 * n * c["bias"] / 2 + (n * v / 8 if c["mask"] else 0)
        return {"bytes": b, "flops": 4 * n * v}
    h, hk, hd, e = c["heads"], c["kv_heads"], c["hd"], _BYTES[c["kv"]]
    row = hk * (hd * e + (4 if c["kv"] == "q8" else 0))
    if c["op"] == "attend":
        lens = _lens(c)
        if c["window"]:
            lens = np.minimum(lens, c["window"])
        total = int(lens.sum())
        return {"bytes": 2 * total * row + 8 * c["n_seqs"] * h * hd + 4 * total // c["page"], "flops": 4 * total * h * hd}
    n = c["rows"] - c["pad"]
    b = n * (4 * (h + 2 * hk) * hd + 4 * h * hd + 2 * row) + 4 * min(n, 4096) * hd
    return {"bytes": b, "flops": n * (h + hk) * hd * 6}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "logits":
        return _logits_exact(s)
    return _attend_exact(s) if c["op"] == "attend" else _append_exact(s)


def _np(t):
    return t.cpu().numpy()


def _quant_np(x):
    """The cache's 8-bit rule is a rule on 32-bit numbers; its values as 64-bit ones."""
    x = x.astype(np.float32)
    amax = np.abs(x).max(-1, keepdims=True)
    tiny = amax < np.float32(1e-30)
    safe = np.where(tiny, np.float32(1), amax)
    q = np.clip(np.trunc(x * (np.float32(127) / safe) + np.copysign(np.float32(0.5), x)), -127, 127)
    return np.where(tiny, 0, q).astype(np.float64), np.where(tiny, 0, safe / np.float32(127)).astype(np.float64)


def _attend_exact(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    lens, table = _np(s["lens"]), _np(s["table"])
    q = _np(s["q"])
    qs = q.astype(np.float64) * s["scale"]
    if s["kd"] is not None:
        qi, qd = _quant_np(q)
        qs = qi * qd * s["scale"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n == 0:
            continue
        first = max(0, int(n) - c["window"]) if c["window"] else 0
        rows = np.arange(first, n)
        page = torch.from_numpy(table[i, rows // c["page"]].astype(np.int64)).cuda()
        slot = torch.from_numpy(rows % c["page"]).cuda()
        for j in range(c["kv_heads"]):
            kk, vv = s["k"][page, j, slot].double(), s["v"][page, j, slot].double()
            if s["kd"] is not None:
                kk = kk * s["kd"][page, j, slot].double()[:, None]
                vv = vv * s["vd"][page, j, slot].double()[:, None]
            x = kk @ torch.from_numpy(qs[i, j * group:(j + 1) * group].T.copy()).cuda()
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            w = torch.exp(x - x.max(0).values)
            out[i, j * group:(j + 1) * group] = (w / w.sum(0)).T @ vv
    return out


def _append_exact(s):
    c = s["case"]
    n, h, hk, hd, page = c["rows"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    x = _np(s["qkv"]).astype(np.float64).reshape(n, h + 2 * hk, hd)
    seqs, pos, table = _np(s["seqs"]), _np(s["pos"]), _np(s["table"])
    qk, v = x[:, :h + hk].copy(), x[:, h + hk:]
    if s["q_norm"] is not None:
        qk /= np.sqrt((qk ** 2).sum(-1, keepdims=True) / hd + s["eps"])
        qk[:, :h] *= _np(s["q_norm"]).astype(np.float64)
        qk[:, h:] *= _np(s["k_norm"]).astype(np.float64)
    turn = _np(s["cos"]).astype(np.float64) + 1j * _np(s["sin"]).astype(np.float64)
    z = (qk[..., 0::2] + 1j * qk[..., 1::2]) * turn[pos][:, None]
    qk[..., 0::2], qk[..., 1::2] = z.real, z.imag
    live = np.nonzero(seqs >= 0)[0]
    q = _np(s["q_out"]).astype(np.float64)
    q[live] = qk[live, :h]
    pools = []
    for y, pool, scale in ((qk[:, h:], s["k"], s["kd"]), (v, s["v"], s["vd"])):
        p = _np(pool).astype(np.float64)
        if scale is not None:
            p = p * _np(scale).astype(np.float64)[..., None]
            yq, yd = _quant_np(y)
            y = yq * yd
        for i in live:
            p[table[seqs[i], pos[i] // page], :, pos[i] % page] = y[i]
        pools.append(p)
    return [q] + pools


def _logits_exact(s):
    z = _np(s["logits"]).astype(np.float64)
    n, v = z.shape
    for i in range(n):
        if "history" in s:
            used = _np(s["history"][i])[:int(s["history_len"][i])]
            ids, count = np.unique(used[used >= 0], return_counts=True)
            r = float(s["repeat"][i])
            x = z[i, ids]
            x = np.where(x > 0, x / r, x * r)
            if "presence" in s:
                x = x - float(s["frequency"][i]) * count - float(s["presence"][i])
            z[i, ids] = x
        if "bias_off" in s:
            a, b = (int(t) for t in s["bias_off"][i:i + 2])
            last = dict(zip(_np(s["bias_ids"][a:b]).tolist(), _np(s["bias_vals"][a:b]).tolist()))
            z[i, list(last)] += np.array(list(last.values()), np.float64)
        if "mask" in s:
            bits = np.unpackbits(_np(s["mask"][i]).view(np.uint8), bitorder="little")[:v]
            z[i, bits == 0] = -np.inf
    return z
