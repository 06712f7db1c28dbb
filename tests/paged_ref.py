"""Plain float64 forms of the paged cache's operators (tests only), on numpy arrays."""
import numpy as np


def page_tables(page, old, add, free, table, nslots):
    """(table, q_start, kv_len, slots, used): request after request, as a program would write it."""
    table = table.copy()
    most = table.shape[1]
    q_start, kv_len, slots = [0], [], []
    base = used = 0
    for i, (o, a) in enumerate(zip(old, add)):
        o, a = max(int(o), 0), max(int(a), 0)
        have, need = -(-o // page), -(-(o + a) // page)
        grow = need - have if need <= most else 0
        fits = need <= most and (grow == 0 or base + grow <= len(free))
        if fits:
            table[i, have:need] = free[base:base + grow]
            used = max(used, base + grow)
            slots += [int(table[i, p // page]) * page + p % page for p in range(o, o + a)]
        else:
            slots += [-1] * a
        base += grow
        q_start.append(q_start[-1] + a)
        kv_len.append(o + a if fits else o)
    slots = (slots + [-1] * nslots)[:nslots]
    return table, np.array(q_start), np.array(kv_len), np.array(slots), used


def rows_of(plane, table, n, page):
    """Keys 0 .. n - 1 of a request from a plane [pages, heads, page, dim]: [n, heads, dim]."""
    j = np.arange(n)
    return plane[np.asarray(table)[j // page], :, j % page].astype(np.float64) if n else np.zeros((0,) + (plane.shape[1], plane.shape[3]))


def visible(p, j, window, sinks):
    return j <= p and (window == 0 or p - window < j or j < sinks)


def attend(q, k, v, first, scale, window=0, sinks=0, lead=0):
    """One request: q [new, heads, dim] at places first ..., k and v [n, kv heads, dim]; `lead` keys in front are seen by all.
    Returns (out, spread): spread = sum_j e_j |v_j| / sum_j e_j, and reach = max_j sum_d |q_d k_jd| scale, which the
    rounding errors are proportional to. Keys a token does not see do not enter (0 times a hidden NaN is not taken)."""
    new, heads, dim = q.shape
    n, g = k.shape[0], heads // max(k.shape[1], 1)
    out, spread, reach = (np.zeros((new, heads, dim)) for _ in range(3))
    for t in range(new):
        see = np.array([j < lead or visible(first + t, j - lead, window, sinks) for j in range(n)], bool)
        if not see.any():
            continue
        for a in range(heads):
            kk, vv, qq = k[see, a // g], v[see, a // g], q[t, a].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = scale * (kk @ qq)
                e = np.exp(s - s.max())
                out[t, a] = (e @ vv) / e.sum()
                spread[t, a] = (e @ np.abs(vv)) / e.sum()
                reach[t, a] = scale * (np.abs(kk) @ np.abs(qq)).max()
    return out, spread, reach


def bound(dtype, dim, n, out, spread, reach):
    """How far an fp32 computation over 16-bit inputs may be from the float64 one: the output's rounding (u, half a unit), the
    weights' rounding to 16 bits (u), fp32 sums of dim products in each score (dim 2^-24 of their absolute sum, entering
    numerator and denominator through e) and of n weights (n 2^-24), 2^-20 for exp2 and the divide, and what a
    weight loses below the smallest f16 (2^-25 of the largest weight, n times)."""
    u = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
    weights = u + 2 * dim * 2.0 ** -24 * reach + 2 * n * 2.0 ** -24 + 2.0 ** -20
    floor = n * 2.0 ** -25 if dtype == "f16" else 0.0
    return u * np.abs(out) + (1 + u) * (weights + floor) * spread + (2.0 ** -25 if dtype == "f16" else 1e-38)
