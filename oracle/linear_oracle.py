"""Linear attention with a decay for each key head, restated in float64 (numpy) token by token, with bounds on what a computation in 16-bit
operands and fp32 sums may be off.

    S_t = exp(log_decay) S_(t-1) + k_t v_t^T,      o_t = scale q_t S_t

Bounds.  ``unit`` is half a step of the 16-bit type relative to the value.  Every product ``scale l^(t-s) (q_t . k_s) v_s`` is rounded once to
16 bits on its way (the weight ``P_ts``, or the state it is a part of), besides fp32 sums of ``D`` and of ``n`` terms and decays within
a few fp32 steps; what enters a state travels in parts whose rest is at most ``unit^2`` of it.  With ``A`` the same sum over magnitudes a
result is off by at most ``A (unit + unit^2 + (D + n + 64) 2^-22) + unit |o|`` and half a step of the type's smallest value.  A state that is
returned has one more part where ``unit^2`` is not fp32's own step: off by ``A (2^-22 + (n + 64) 2^-22)``.
"""
import numpy as np

F32 = 2.0 ** -22                                      # two fp32 steps: the order and inner rounding of a matrix instruction do not matter
UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float16": 2.0 ** -25, "bfloat16": 0.0}


def _head(q, k, v, decay, scale, first, dout, dlast):
    """``q [g, n, d]``: the query heads of a key head; results likewise."""
    n, d = k.shape
    s = np.zeros((d, d)) if first is None else first.copy()
    out, dq = np.zeros(q.shape), np.zeros(q.shape)
    for t in range(n):
        s = decay * s + np.outer(k[t], v[t])
        out[:, t] = scale * q[:, t] @ s
        if dout is not None:
            dq[:, t] = scale * dout[:, t] @ s.T
    found = {"out": out, "last": s}
    if dout is not None:
        r = np.zeros((d, d)) if dlast is None else dlast.copy()
        dk, dv = np.zeros(k.shape), np.zeros(v.shape)
        for t in range(n - 1, -1, -1):
            r = r + scale * q[:, t].T @ dout[:, t]
            dk[t], dv[t] = r @ v[t], k[t] @ r
            r = decay * r
        found.update(dq=dq, dk=dk, dv=dv, dfirst=r)
    return found


def packed(q, k, v, log_decay, offsets, scale, first=None, dout=None, dlast=None):
    """``q [T, Hq, D]``, ``k``, ``v [T, Hk, D]``, ``first [B, Hk, D, D]``: a dict of results; tokens outside every sequence have zeros."""
    key_heads, dim = k.shape[1:]
    group, count = q.shape[1] // key_heads, len(offsets) - 1
    states = np.zeros((count, key_heads, dim, dim))
    found = {"out": np.zeros(q.shape), "last": states.copy()}
    if dout is not None:
        found.update(dq=np.zeros(q.shape), dk=np.zeros(k.shape), dv=np.zeros(v.shape), dfirst=states.copy())
    for b in range(count):
        at = slice(max(0, offsets[b]), max(0, offsets[b + 1]))
        for h in range(key_heads):
            mine = slice(h * group, (h + 1) * group)
            one = _head(q[at, mine].transpose(1, 0, 2), k[at, h], v[at, h], np.exp(log_decay[h]), scale, None if first is None else first[b, h],
                        None if dout is None else dout[at, mine].transpose(1, 0, 2), None if dlast is None else dlast[b, h])
            for name, x in one.items():
                if name in ("out", "dq"):
                    found[name][at, mine] = x.transpose(1, 0, 2)
                elif name in ("dk", "dv"):
                    found[name][at, h] = x
                else:
                    found[name][b, h] = x
    return found


def bounds(q, k, v, log_decay, offsets, scale, kind, first=None, dout=None, dlast=None):
    """``{name: (value, bound)}``."""
    exact = packed(q, k, v, log_decay, offsets, scale, first, dout, dlast)
    mag = lambda x: None if x is None else np.abs(x)
    sums = packed(mag(q), mag(k), mag(v), log_decay, offsets, abs(scale), mag(first), mag(dout), mag(dlast))
    n, unit, found = max(1, int(np.max(np.diff(offsets)))) if len(offsets) > 1 else 1, UNIT[kind], {}
    steps = (k.shape[2] + n * q.shape[1] // k.shape[1] + 64) * F32
    for name, x in exact.items():
        if name in ("last", "dfirst"):
            found[name] = (x, sums[name] * (F32 + steps))
        else:
            found[name] = (x, sums[name] * (unit + unit ** 2 + steps) + unit * np.abs(x) + TINY[kind])
    return found


def step(q, k, v, log_decay, states, slots, scale):
    """``(out, states)`` of one token of every sequence."""
    out, states, group = np.zeros(q.shape), states.copy(), q.shape[1] // k.shape[1]
    for b, slot in enumerate(slots):
        if 0 <= slot < len(states):
            for h in range(k.shape[1]):
                states[slot, h] = np.exp(log_decay[h]) * states[slot, h] + np.outer(k[b, h], v[b, h])
                out[b, h * group:(h + 1) * group] = scale * q[b, h * group:(h + 1) * group] @ states[slot, h]
    return out, states
