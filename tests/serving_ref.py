"""Plain 64-bit (attention, append) and exact 32-bit (8-bit rows, logits)
restatements of the serving operators, for their tests. No library code."""
import numpy as np


def quant_rows(x):
    """The 8-bit cache's row rule on float32 rows: int8 values and float32 scales [..., 1]."""
    x = np.asarray(x, np.float32)
    amax = np.abs(x).max(-1, keepdims=True)
    tiny = amax < np.float32(1e-30)
    safe = np.where(tiny, np.float32(1), amax)
    q = np.clip(np.trunc(x * (np.float32(127) / safe) + np.copysign(np.float32(0.5), x)), -127, 127)
    return np.where(tiny, 0, q).astype(np.int8), np.where(tiny, np.float32(0), safe / np.float32(127))


def gather(pool, table, page, seq, pos):
    """Rows [len(pos), n_kv, ...] of a sequence's positions."""
    return np.stack([pool[table[seq, p // page], :, p % page] for p in pos])


def attend(q, k, v, table, lens, scale, window=0, softcap=0.0, kd=None, vd=None):
    """q [n, heads, hd]; k, v pools. Returns (out, reach): reach = per row, the largest sum of
    |q_d k_d| * scale over its positions, which the score's rounding is relative to."""
    n, heads, hd = q.shape
    hk, page = k.shape[1], k.shape[2]
    group = heads // hk
    out, reach = np.zeros(q.shape), np.zeros((n, heads))
    if kd is not None:
        qi, qd = quant_rows(q)
        qf = qi.astype(np.float64) * qd
    else:
        qf = q.astype(np.float64)
    for i in range(n):
        pos = range(max(0, lens[i] - window) if window else 0, lens[i])
        if not len(pos):
            continue
        kk, vv = gather(k, table, page, i, pos).astype(np.float64), gather(v, table, page, i, pos).astype(np.float64)
        if kd is not None:
            kk = kk * gather(kd, table, page, i, pos)[..., None]
            vv = vv * gather(vd, table, page, i, pos)[..., None]
        for h in range(heads):
            g = h // group
            s = kk[:, g] @ qf[i, h] * scale
            reach[i, h] = (np.abs(kk[:, g]) @ np.abs(qf[i, h])).max() * abs(scale)
            if softcap:
                s = softcap * np.tanh(s / softcap)
            w = np.exp(s - s.max())
            out[i, h] = (w / w.sum()) @ vv[:, g]
    return out, reach


def norm_rope(x, cos, sin, w=None, eps=0.0):
    """x [n, heads, hd] in 64 bits: norm of each head, rotation of adjacent pairs by cos, sin [n, hd/2]."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
    y = np.empty_like(x)
    y[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    y[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return y


def logits(z, history=None, history_len=None, repeat=None, presence=None, frequency=None, bias=None, mask=None):
    """Row by row, token by token, in float32. bias: a list of (ids, vals) per row; mask [n, words] uint32."""
    z = np.array(z, np.float32)
    n, v = z.shape
    f = np.float32
    with np.errstate(all="ignore"):
        for i in range(n):
            if history is not None:
                h = history[i][:history_len[i]] if history_len is not None else history[i]
                ids, cnt = np.unique(h[(h >= 0) & (h < v)], return_counts=True)
                for t, c in zip(ids, cnt):
                    x = z[i, t]
                    if repeat is not None:
                        x = x / f(repeat[i]) if x > 0 else x * f(repeat[i])
                    if frequency is not None:
                        x = x - f(frequency[i]) * f(c)
                    if presence is not None:
                        x = x - f(presence[i])
                    z[i, t] = x
            if bias is not None:
                for t, b in dict(zip(*[a.tolist() for a in bias[i]])).items():
                    if 0 <= t < v:
                        z[i, t] = z[i, t] + f(b)
            if mask is not None:
                bits = np.unpackbits(np.ascontiguousarray(mask[i]).view(np.uint8), bitorder="little")[:v]
                z[i, bits == 0] = -np.inf
    return z
