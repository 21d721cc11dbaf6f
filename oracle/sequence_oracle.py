"""Checker for the sequence operators (test infrastructure, like everything under oracle/): the gated recurrence and its
gradients row by row, and counter-based dropout, in float64 with numpy on the CPU, from their definitions.  The reference
has no counterpart.

The recurrence also returns first-order bounds of what 32-bit arithmetic may change, from the same loops run on magnitudes:
with u = 2^-24, every product and sum adds at most u times the magnitude of what is summed, however the rows are grouped,
because each row's share passes through at most one rounding per row between it and the result plus a few of the grouping.
"""
import numpy as np

U = 2.0 ** -24
# Roundings a row adds, in units of u, relative to its product f h and to its input i.  A logit's gate: the exponential 5
# (2 ulp = 4 u, its argument's correction 1), the sum 1 + e 1, the reciprocal 2 (1 ulp), the product e f of 1 - f 1: 9.  The
# input's product 1, the fused multiply-add 1, the two of the grouping's products: 13.
# 16-bit logits are not corrected: 1.22 |g| more.  The 3 that are left cover |g| <= 2.4; callers double the bound, which covers
# |g| <= 15.  Beyond that the gates by themselves are what to compare.
ROW = 16.0


def row_order(rows, begin, count, reverse):
    """For every sequence its rows in the order of the recurrence."""
    out = []
    for b, c in zip(begin, count):
        r = np.arange(b, b + c)
        out.append(r[::-1] if reverse else r)
    return out


def recurrence(x, gate, state, begin, count, form, coupled, reverse, v_h=None, v_last=None):
    """x [N, D], gate [N, H], state [S, D]; sequence s holds rows begin[s] .. begin[s] + count[s].  Returns a dict of
    (value, bound) pairs: h, last, and with gradients of the outputs given also dx, dgate, dstate."""
    x, gate, state = (np.asarray(t, np.float64) for t in (x, gate, state))
    n, d = x.shape
    heads = gate.shape[1]
    with np.errstate(over="ignore", invalid="ignore"):
        f1 = 1.0 / (1.0 + np.exp(-gate)) if form == "logit" else gate
        k1 = 1.0 / (1.0 + np.exp(gate)) if form == "logit" else 1.0 - gate
    f, k = np.repeat(f1, d // heads, 1), np.repeat(k1, d // heads, 1)
    i = k * x if coupled else x
    zero = lambda *s: np.zeros(s)  # noqa: E731
    h, eh, last, elast = zero(n, d), zero(n, d), state.copy(), zero(*state.shape)
    hp, ehp, mag = zero(n, d), zero(n, d), zero(n, d)          # h_{t-1}, its bound, and its magnitude
    orders = row_order(n, begin, count, reverse)
    for s, rows in enumerate(orders):
        a, e, m = state[s].copy(), zero(d), np.abs(state[s])
        for r in rows:
            hp[r], ehp[r], mag[r] = a, e, m
            e = np.abs(f[r]) * e + ROW * U * (np.abs(f[r]) * m + np.abs(i[r]))
            m = np.abs(f[r]) * m + np.abs(i[r])
            a = f[r] * a + i[r]
            h[r], eh[r] = a, e
        last[s], elast[s] = a, e
    out = dict(h=(h, eh), last=(last, elast))
    if v_h is None and v_last is None:
        return out
    v_h = zero(n, d) if v_h is None else np.asarray(v_h, np.float64)
    v_last = zero(*state.shape) if v_last is None else np.asarray(v_last, np.float64)
    dx, edx, df, edf = zero(n, d), zero(n, d), zero(n, d), zero(n, d)
    dstate, edstate = v_last.copy(), zero(*state.shape)
    for s, rows in enumerate(orders):
        q, e, m = v_last[s].copy(), zero(d), np.abs(v_last[s])
        for r in rows[::-1]:
            g, mg = v_h[r] + q, np.abs(v_h[r]) + m
            eg = e + 2 * U * mg
            dx[r] = k[r] * g if coupled else g
            edx[r] = (np.abs(k[r]) * (eg + ROW * U * mg)) if coupled else eg
            w = hp[r] - x[r] if coupled else hp[r]
            ew = ehp[r] + 2 * U * (mag[r] + (np.abs(x[r]) if coupled else 0.0))
            slope = f[r] * k[r] if form == "logit" else np.ones(d)
            df[r] = g * w * slope
            edf[r] = np.abs(slope) * (eg * np.abs(w) + mg * ew + 2 * ROW * U * mg * np.abs(w))
            q = f[r] * g
            e = np.abs(f[r]) * eg + ROW * U * np.abs(f[r]) * mg
            m = np.abs(f[r]) * mg
        dstate[s], edstate[s] = q, e
    per_head = d // heads
    terms = np.abs(df).reshape(n, heads, per_head).sum(-1)
    dgate = df.reshape(n, heads, per_head).sum(-1)
    edgate = edf.reshape(n, heads, per_head).sum(-1) + (0 if per_head == 1 else (per_head + 8) * U) * terms
    out.update(dx=(dx, edx), dgate=(dgate, edgate), dstate=(dstate, edstate))
    return out


def philox_words(count, seed, step, first=0):
    """Words first .. first + count - 1 of Philox4x32-10 (Salmon et al., SC'11): block w // 4 has the counter (w // 4, step)
    and the key seed.  ``first`` a multiple of four."""
    u = np.uint64
    low, half = u(0xFFFFFFFF), u(32)
    block = np.arange(first // 4, first // 4 + -(-count // 4), dtype=u)
    c = [block & low, block >> half, np.full_like(block, u(step & 0xFFFFFFFF)), np.full_like(block, u(step >> 32))]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(p1 >> half) ^ c[1] ^ u(k[0]), p1 & low, (p0 >> half) ^ c[3] ^ u(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:count]


def dropout(x, p, seed, step, residual=None):
    """(value, kept) of x (any shape) in row-major order."""
    x = np.asarray(x, np.float64)
    keep = (philox_words(x.size, seed, step) >= round(p * 2 ** 32)).reshape(x.shape)
    with np.errstate(invalid="ignore", over="ignore"):
        out = np.where(keep, x / (1.0 - p) if p < 1 else 0.0, 0.0)
    return (out if residual is None else out + np.asarray(residual, np.float64)), keep
