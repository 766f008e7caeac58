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


def parts_of(x, n):
    """x (32 bits) as n numbers of 8 bits, the largest first, each rounded to nearest even."""
    out, x = [], np.asarray(x, np.float32)
    for _ in range(n):
        b = x.view(np.uint32).astype(np.uint64)
        out.append((((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint32) << 16).view(np.float32))
        x = x - out[-1]
    return out


# The 2-norm of a head's state, relative to it, may be off by so much where decays let it live for a while: eight half steps of 32 bits.
# About eight roundings meet a state's number on its way through a chunk (sums of K S over four parts, V - K S, three sums of V', of the
# new state), each 2^-24 / sqrt(3) in the mean square of partial sums up to twice the result's size: sqrt(8) * 2 / sqrt(3) = 3.3 half
# steps; the rest is left for the decays' powers. A number in two parts of 8 bits instead of three is off by 2^-17 at most, 2^-17.8 in the mean
# square: 74 half steps.
STATE_NORM = 8 * U
STATE_VALUES, STATE_DECAY = 0.1, 0.005  # of the values and the log decays: what the state was counts for as much as what is added


def chunked(k, v, g, beta, state, exact=True, parts=(3, 3, 3, 3), skip=()):
    """The state after chunks of 64 tokens, the products of parts of 8 bits in 32-bit sums. parts: how many of the state, of V - K S, of
    the inverse, of the corrections; skip: products (part of the inverse, part of V - K S) left out; exact: keys are one part, else two."""
    f32, S = np.float32, np.asarray(state, np.float32).copy()

    def product(a, b, skip=()):
        return sum((a[p] @ b[z] for p in reversed(range(len(a))) for z in reversed(range(len(b))) if p + z < 3 and (p, z) not in skip),
                   np.zeros((a[0].shape[0], b[0].shape[1]), f32))

    for c in range(0, len(k), 64):
        K, G, b = k[c:c + 64].astype(f32), np.cumsum(np.asarray(g[c:c + 64], np.float64)), beta[c:c + 64].astype(f32)
        keys = [K] if exact else parts_of(K, 2)
        A = np.tril((K @ K.T) * np.exp(np.minimum(G[:, None] - G, 0)).astype(f32) * b[:, None], -1)
        T = (np.linalg.inv(np.eye(len(K)) + A.astype(np.float64)).astype(f32)) * b
        R = v[c:c + 64].astype(f32) - np.exp(G).astype(f32)[:, None] * product(keys, parts_of(S, parts[0]))
        V = product(parts_of(T, parts[2]), parts_of(R, parts[1]), skip)
        S = S * f32(np.exp(G[-1])) + product([x.T for x in keys], parts_of(V * np.exp(G[-1] - G).astype(f32)[:, None], parts[3]))
    return S


def state_norm_error(got, want):
    return float(np.sqrt(((got - want) ** 2).sum() / (want ** 2).sum()))
