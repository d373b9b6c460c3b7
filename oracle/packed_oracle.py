"""Attention over packed sequences, quantised rows and attention over a cache, restated in float64 (numpy), with bounds on what a
computation in 16-bit operands and fp32 sums may be off.

Bounds.  ``unit`` is half a step of the 16-bit type relative to the value.  With exact 16-bit inputs a score is a sum of D exact
products in fp32: off by at most ``e = (D + 4) 2^-23 scale sum |q_d k_d|`` (two units a step, so that the order and the
rounding of a matrix instruction's inner sums do not matter), a probability by ``2 e`` of itself plus its own rounding of one
``unit``.  Results are sums over these, rounded once more.
"""
import numpy as np

F32 = 2.0 ** -23
UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float16": 2.0 ** -25, "bfloat16": 0.0}       # half a step of the smallest values: fp16 ones below 2^-14 have fewer bits


def _softmax(s, visible):
    s = np.where(visible, s, -np.inf)
    top = s.max(-1, keepdims=True) if s.shape[-1] else np.zeros(s.shape[:-1] + (1,))
    e = np.where(visible, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
    total = e.sum(-1, keepdims=True)
    return np.where(total > 0, e / np.where(total > 0, total, 1.0), 0.0)


def rows(q, k, v, visible, scale, kind, dout=None, weight_tiny=0.0, lifted=False):
    """One head: ``q [n, d]``, ``k``, ``v [m, d]``, ``visible [n, m]``.  Returns ``{name: (value, bound)}``.

    ``lifted``: dS is rounded times a power of two that brings the largest of its query (for dq) or key (for dk) to 2^3 or more, so that
    half the smallest step is 2^-3 ``TINY`` of that largest one; otherwise as it is."""
    unit, tiny = UNIT[kind], TINY[kind]
    d = q.shape[1]
    s = scale * (q @ k.T)
    e = (d + 4) * F32 * abs(scale) * (np.abs(q) @ np.abs(k).T) + 8 * F32 * (1 + np.abs(s))
    e = np.where(visible, e, 0.0).max(-1, keepdims=True) if s.shape[1] else np.zeros((len(q), 1))
    p = _softmax(s, visible)
    m = max(1, s.shape[1])
    off = p * (unit + 2 * e + 2 * m * F32) + weight_tiny + tiny * (p > 0)
    out = p @ v
    out_off = off @ np.abs(v) + unit * np.abs(out) + tiny
    found = {"out": (out, out_off)}
    if dout is not None:
        dp = dout @ v.T
        delta = (dout * out).sum(-1, keepdims=True)
        ds = scale * p * (dp - delta)
        dp_off = (d + 4) * F32 * (np.abs(dout) @ np.abs(v).T)
        delta_off = (np.abs(dout) * (out_off + (d + 4) * F32 * np.abs(out))).sum(-1, keepdims=True)
        ds_off = np.abs(ds) * (unit + 2 * e + 2 * m * F32 + 8 * F32) + abs(scale) * p * (dp_off + delta_off)
        largest = lambda axis: np.abs(ds).max(axis, keepdims=True) / 8 if lifted else max(1.0, abs(scale))
        ds_off, ds_off_k = (ds_off + tiny * (p > 0) * largest(axis) for axis in (1, 0))
        dq, dk, dv = ds @ k, ds.T @ q, p.T @ dout
        found["dq"] = (dq, ds_off @ np.abs(k) + unit * np.abs(dq) + tiny)
        found["dk"] = (dk, ds_off_k.T @ np.abs(q) + unit * np.abs(dk) + tiny)
        found["dv"] = (dv, off.T @ np.abs(dout) + unit * np.abs(dv) + tiny)
    return found


def packed(q, k, v, offsets, scale, causal, kind, dout=None):
    """``q [T, Hq, D]``, ``k``, ``v [T, Hk, D]``: ``{name: (value, bound)}``; tokens outside every sequence have zeros."""
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    shapes = {"out": q.shape}
    if dout is not None:
        shapes.update(dq=q.shape, dk=k.shape, dv=k.shape)
    found = {name: (np.zeros(shape), np.zeros(shape)) for name, shape in shapes.items()}
    for a, b in zip(offsets[:-1], offsets[1:]):
        n = b - a
        if n <= 0:
            continue
        visible = np.tril(np.ones((n, n), dtype=bool)) if causal else np.ones((n, n), dtype=bool)
        for h in range(heads):
            one = rows(q[a:b, h], k[a:b, h // group], v[a:b, h // group], visible, scale, kind,
                       None if dout is None else dout[a:b, h])
            for name, (value, off) in one.items():
                at = h if name in ("out", "dq") else h // group
                found[name][0][a:b, at] += value
                found[name][1][a:b, at] += off
    return found


def e4m3(x):
    """Nearest e4m3 value, ties to even: eight steps to a power of two, 2^-9 apart below 2^-6."""
    exponent = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -20))), -6)
    step = 2.0 ** (exponent - 3)
    return np.rint(x / step) * step


def quantise(x, kind):
    """Rows ``[..., D]`` -> (held values, scales ``[...]``), both float64; ``kind`` 'int8' or 'e4m3'."""
    bound = 127.0 if kind == "int8" else 448.0
    top = np.abs(x).max(-1)
    with np.errstate(invalid="ignore", divide="ignore"):
        y = np.where(top[..., None] > 0, x * bound / top[..., None], 0.0)
    y = np.rint(y) if kind == "int8" else e4m3(y)
    fine = np.isfinite(top)
    return np.where(fine[..., None], y, 0.0), np.where(fine, top / bound, np.nan)


def cached(q, k, v, held_keys, held_values, value_scales, lengths, tree, scale, kind, by_weight=False):
    """``q [B, n, Hq, D]``, new ``k``, ``v [B, n, Hk, D]``, ``held_* [b] -> [Hk, length, D]`` (dequantised), ``value_scales [b] ->
    [Hk, length]`` (None: a 16-bit cache), ``tree [B, n, n]``.

    Bound of a quantised cache.  The weight of value row j is p_j t_j / top before it is rounded, p_j relative to a reference point at
    which the sum of all p is at least 1, t_j the row's scale (1 of a new token) and top at most twice the largest of them.  Where that
    is below the smallest normal fp16 value the rounding is off by up to half the smallest step, ``TINY``, whatever the weight: by
    TINY top / t_j of p_j, and of the normalised probability no more, the sum being at least 1.  With ``by_weight`` top is what the
    largest p_j t_j of the cached rows is, less a factor of 2^4 (for a new token, whose row comes as it is, of all that the token
    sees): a row that weighs nothing is no measure for the others."""
    batch, n, heads, _ = q.shape
    group = heads // k.shape[2]
    value, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(batch):
        for h in range(heads):
            g = h // group
            keys = np.concatenate([held_keys[b][g], k[b, :, g]])
            values = np.concatenate([held_values[b][g], v[b, :, g]])
            visible = np.concatenate([np.ones((n, lengths[b]), dtype=bool), tree[b]], 1)
            tiny = 0.0
            if value_scales is not None:
                t = np.concatenate([value_scales[b][g], np.ones(n)])
                tiny = np.where(t > 0, TINY[kind] * 2 * t.max() / np.where(t > 0, t, 1.0), 0.0)
                if by_weight:
                    w = _softmax(scale * (q[b, :, h] @ keys.T), visible) * t
                    n_held = lengths[b]
                    top = np.concatenate([np.broadcast_to(w[:, :n_held].max(-1, keepdims=True), (n, n_held)) if n_held else np.zeros((n, 0)),
                                          np.broadcast_to(w.max(-1, keepdims=True), (n, n))], 1)
                    tiny = np.where(t > 0, TINY[kind] * 2.0 ** -4 * top / np.where(t > 0, t, 1.0), 0.0)
            value[b, :, h], bound[b, :, h] = rows(q[b, :, h], keys, values, visible, scale, kind, weight_tiny=tiny)["out"]
    return value, bound
