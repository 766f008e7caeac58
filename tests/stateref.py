"""Plain numpy (64-bit) forms of the operators over kept states, with bounds on what 32 bits may be off by."""
import numpy as np

U = 2.0 ** -24  # half a step of 32 bits, relative


def conv(x, w, bias, silu, before):
    """One sequence: x [n, C], w [C, taps], before [taps - 1, C] -> (out, bound on its error before it is rounded, the last inputs)."""
    taps = w.shape[1]
    line = np.concatenate([before.astype(np.float64), x.astype(np.float64)])
    n = len(x)
    parts = np.stack([line[j:j + n] * w[:, j] for j in range(taps)]) if n else np.zeros((taps, 0, x.shape[1]))
    b = 0.0 if bias is None else bias.astype(np.float64)
    y = parts.sum(0) + b
    # a rounding for each product added, of what is there by then
    off = taps * U * (np.abs(parts).sum(0) + np.abs(b))
    if silu:
        s = 1 / (1 + np.exp(-y))
        # |slope| <= 1.1; exp: its argument's rounding (half a step of |y| log2 e, times ln 2) and a step of its own, which reach
        # the result through 1 - s; the sum, the quotient
        off = 1.1 * off + np.abs(y * s) * ((np.abs(y) + 3) * U * (1 - s) + 2 * U) + 1e-37
        y = y * s
    return y, off, line[n:]


def gates(decay, beta, a_log, dt_bias):
    """-> (log decay, beta, bounds on the errors of both)."""
    g, b = decay.astype(np.float64), beta.astype(np.float64)
    if a_log is None:
        return g, b, np.zeros(g.shape), np.zeros(g.shape)
    x = g + dt_bias
    g = -np.exp(a_log.astype(np.float64)) * (np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x))))
    b = 1 / (1 + np.exp(-b))
    # the sum's rounding, by a slope of at most s / softplus <= 1 relative to max(1, |x|); exp, log1p, exp of a_log and the product,
    # each a step or two: 16 half steps in all, and |x| + |a_log| of them for the exponents' own rounding
    return g, b, np.abs(g) * (16 + np.abs(x) + np.abs(a_log)) * U, b * 8 * U


def delta(q, k, v, g, beta, state, scale, unit_eps, g_off, b_off):
    """One sequence and head: q, k [n, dk], v [n, dv], g, beta [n], state [dk, dv] -> (out, bound, state, bound).

    An error of a column of the state goes from a token to the next through exp(g) (I - beta k k^T), whose norm is no more than
    max(1, |1 - beta k.k|) exp(g): so the bounds are 2-norms of columns, added up token by token. What a token adds, relative to
    the sizes that go in (column s of S', its correction d): products and sums over the key's elements, in any order and with up to
    three parts of 8 bits a number, less than `c` half steps; the decay's; the key's own division by its norm."""
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    if unit_eps:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + np.float64(np.float32(unit_eps))) for x in (q, k))
    scale = np.float64(np.float32(scale))
    S = state.astype(np.float64).copy()
    e = np.zeros(S.shape[1])
    out, off = np.zeros(v.shape), np.zeros(v.shape)
    c = 2 * k.shape[1] + 32
    for t in range(len(v)):
        f = np.exp(g[t])
        S = S * f
        s, kk = np.sqrt((S * S).sum(0)), float(k[t] @ k[t])
        d = beta[t] * (v[t] - k[t] @ S)
        local = (c * U + b_off[t] / max(beta[t], 1e-30)) * (np.abs(beta[t]) * kk * s + np.sqrt(kk) * np.abs(d) + np.abs(beta[t]) * np.sqrt(kk) * np.abs(v[t]))
        local += s * ((abs(g[t]) if np.isfinite(g[t]) else 0) * U + 8 * U + g_off[t])
        e = e * f * max(1.0, abs(1 - beta[t] * kk)) + local
        S = S + np.outer(k[t], d)
        out[t] = scale * (q[t] @ S)
        nq = np.sqrt(q[t] @ q[t])
        off[t] = abs(scale) * nq * (e + c * U * (np.sqrt((S * S).sum(0)) + s + np.sqrt(kk) * np.abs(d)))
    return out, off, S, e
