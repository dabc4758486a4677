"""Float64 references of the gated delta layers' operators (include/hq_serve.h) with bounds of each output's error.

Errors of the recurrence, by the 2-norm of a column of S, e: a step S' = (I - beta k k^T) a S + beta k v^T with |k| <= 1, 0 <= beta <= 1
and a <= 1 is a contraction, so errors add up and never grow: e <- a e + c. A token's own error c: the product k^T S is a 32-bit sum
over k_dim products, (k_dim + 8) 2^-24 of |k| |S| at most; operands that are held as two fp16 terms are off by 2^-22 of their
column's largest; a chunked form has sums over up to 64 tokens beside them. c = 4 (k_dim + 80) 2^-24 (|a S| + |v|) covers both.

Outputs are the state's products with a query of norm 1, so their error is e |q|, and end in fp16; with the norm, those of chunks are
rounded to it before the norm too. (Products of the chunked form besides the state's are of operands of two terms as well, 2^-22 of
the largest of up to 64 tokens' magnitudes: within what c has for each of these tokens.)"""
import numpy as np

U16, U32 = 2.0 ** -11, 2.0 ** -24


def silu(x):
    with np.errstate(over="ignore"):
        return x / (1 + np.exp(-x))


def append(x, old, w, a, b, a_log, dt, n_new, hk, hv, dk, dv, eps):
    """x [tokens, channels], old: each sequence's inputs before its tokens [taps - 1, channels], w [channels, taps]. Returns qkv and
    its bound, decay and its bound, beta and its bound, each sequence's last inputs."""
    taps, T, ch = w.shape[1], x.shape[0], x.shape[1]
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    s, mag, keep, t = np.zeros((T, ch)), np.zeros((T, ch)), [], 0
    for o, n in zip(old, n_new):
        rows = np.concatenate([o.astype(np.float64), x64[t:t + n]])
        for j in range(taps):
            s[t:t + n] += rows[j:j + n] * w64[:, j]
            mag[t:t + n] += np.abs(rows[j:j + n] * w64[:, j])
        keep.append(rows[n:].astype(np.float32))
        t += n
    y = silu(s)
    dy = 1.1 * (taps + 1) * U32 * mag + 8 * U32 * np.abs(y)  # (the slope of silu is below 1.1)
    c = 2 * hk * dk
    q = y[:, :c].reshape(T, 2 * hk, dk)
    d = dy[:, :c].reshape(T, 2 * hk, dk)
    ss = (q * q).sum(-1, keepdims=True) + eps
    n = q / np.sqrt(ss)
    dn = d / np.sqrt(ss) + np.abs(n) * ((np.abs(q) * d).sum(-1, keepdims=True) / ss + (dk / 2 + 8) * U32)
    out, bound = np.concatenate([n.reshape(T, c), y[:, c:]], 1), np.concatenate([dn.reshape(T, c), dy[:, c:]], 1)
    bound = bound + U16 * np.abs(out) + 2.0 ** -25
    z = a.astype(np.float64) + dt.astype(np.float64)
    g = -np.exp(a_log.astype(np.float64)) * np.logaddexp(0, z)
    dg = np.exp(a_log.astype(np.float64)) * 2 * U32 * (np.abs(a) + np.abs(dt)) + 16 * U32 * np.abs(g) + 2.0 ** -140
    with np.errstate(over="ignore"):
        beta = 1 / (1 + np.exp(-b.astype(np.float64)))
    return out, bound, g, dg, beta, 8 * U32 * beta + 2.0 ** -126, keep


def delta(q, k, v, decay, beta, states, n_new, scale, norm=None, gate=None, eps=0.0):
    """q, k [tokens, hk, dk], v [tokens, hv, dv], states [sequences][hv, dk, dv]. Returns out [tokens, hv, dv] and its bound, the
    states behind and their bounds [sequences][hv, 1, dv] (of a column's 2-norm, so of each element too)."""
    T, hv, dv = v.shape
    dk, rep = q.shape[2], hv // q.shape[1]
    q, k = (np.repeat(x.astype(np.float64), rep, 1) for x in (q, k))
    v = v.astype(np.float64)
    out, bound, after, e_after, t = np.zeros((T, hv, dv)), np.zeros((T, hv, dv)), [], [], 0
    for s0, n in zip(states, n_new):
        S, e = s0.astype(np.float64), np.zeros((hv, 1, dv))
        for i in range(n):
            keep = np.exp(decay[t].astype(np.float64))[:, None, None]
            # (a decay's exponential is off by 2^-22 of itself: its argument's sums and the function)
            S = S * keep
            size = np.sqrt((S * S).sum(1, keepdims=True))
            e = e * keep + 4 * (dk + 80) * U32 * (size + np.abs(v[t])[:, None])
            u = (v[t] - (k[t][:, :, None] * S).sum(1)) * beta[t].astype(np.float64)[:, None]
            S = S + k[t][:, :, None] * u[:, None]
            o = scale * (S * q[t][:, :, None]).sum(1)
            b = abs(scale) * e[:, 0] * np.linalg.norm(q[t], axis=-1)[:, None]
            if norm is not None:
                z = silu(gate[t].astype(np.float64)) * norm.astype(np.float64)
                ms = (o * o).mean(-1, keepdims=True) + eps
                # (with the norm, chunks round o to fp16 before it)
                b = b + U16 * np.abs(o) + 2.0 ** -25
                rel = (np.abs(o) * b).mean(-1, keepdims=True) / ms + (dv + 16) * U32
                # (second order: the norm itself moves by at most rel)
                b = (b + np.abs(o) * rel) / np.sqrt(ms) * np.abs(z) * (1 + 2 * rel)
                o = o / np.sqrt(ms) * z
            out[t], bound[t] = o, b + U16 * np.abs(o) + 2.0 ** -25
            t += 1
        after.append(S), e_after.append(e)
    return out, bound, after, e_after
