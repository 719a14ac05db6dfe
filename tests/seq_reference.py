"""Plain 64-bit forms of the sequence operators, for their tests.

Everything is float64 numpy, one position at a time, from the definitions;
gradients are the formulas', which tests/test_seq_host.py holds against central
differences.  No code is shared with the library."""

from __future__ import annotations

import numpy as np


def f64(*arrays):
    out = [None if a is None else np.asarray(a, np.float64) for a in arrays]
    return out[0] if len(out) == 1 else out


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


# ------------------------------------------------------------------- norm
def rms_norm(x, w, residual, eps):
    x, w, residual = f64(x, w, residual)
    s = x if residual is None else x + residual
    return s / np.sqrt((s * s).mean(axis=-1, keepdims=True) + eps) * w, s


def rms_norm_bwd(s, w, dy, dsum, eps):
    s, w, dy, dsum = f64(s, w, dy, dsum)
    rstd = 1.0 / np.sqrt((s * s).mean(axis=-1, keepdims=True) + eps)
    xh = s * rstd
    dx = rstd * (w * dy - xh * (w * dy * xh).mean(axis=-1, keepdims=True))
    if dsum is not None:
        dx = dx + dsum
    return dx, (dy * xh).reshape(-1, s.shape[-1]).sum(axis=0)


def e4m3_values():
    """The 127 finite values >= 0 of e4m3: 3 fraction bits, exponents -6..8,
    subnormals below 2^-6, 448 the largest (the code after it is NaN)."""
    vals = [m / 8 * 2.0 ** -6 for m in range(8)]
    vals += [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)]
    return np.array(vals[:-1])


# ------------------------------------------------------------------- conv
def causal_conv(x, w, bias, state, lengths, silu):
    """(y, state_out), rows past a sequence's end zero in y."""
    x, w, bias, state = f64(x, w, bias, state)
    B, L, D = x.shape
    W = w.shape[1]
    y = np.zeros((B, L, D))
    last = np.zeros((B, W - 1, D))
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        ext = np.concatenate([state[b] if state is not None else np.zeros((W - 1, D)), x[b, :n]])
        for t in range(n):
            p = (ext[t:t + W].T * w).sum(axis=1) + (bias if bias is not None else 0.0)
            y[b, t] = p * sigmoid(p) if silu else p
        last[b] = ext[n:]
    return y, last


def causal_conv_bwd(x, w, bias, state, lengths, silu, dy, dlast):
    x, w, bias, state, dy, dlast = f64(x, w, bias, state, dy, dlast)
    B, L, D = x.shape
    W = w.shape[1]
    dx, dw, db, dstate = np.zeros((B, L, D)), np.zeros(w.shape), np.zeros(D), np.zeros((B, W - 1, D))
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        ext = np.concatenate([state[b] if state is not None else np.zeros((W - 1, D)), x[b, :n]])
        dext = np.zeros_like(ext)
        if dlast is not None:
            dext[n:] += dlast[b]
        for t in range(n):
            p = (ext[t:t + W].T * w).sum(axis=1) + (bias if bias is not None else 0.0)
            g = dy[b, t].copy()
            if silu:
                s = sigmoid(p)
                g = g * (s * (1 + p * (1 - s)))
            dext[t:t + W] += (g[:, None] * w).T
            dw += (g * ext[t:t + W]).T
            db += g
        dx[b, :n] = dext[W - 1:]
        dstate[b] = dext[:W - 1]
    return dx, dw, db, dstate


# ------------------------------------------------------------------- scan
def _step(delta, bias, softplus):
    raw = delta + (bias if bias is not None else 0.0)
    return (np.logaddexp(raw, 0.0), sigmoid(raw)) if softplus else (raw, np.ones_like(raw))


def _spread(v, D):
    """[G, N] rows as every channel of the group sees them: [D, N]."""
    return np.repeat(v, D // v.shape[0], axis=0)


def selective_scan(u, delta, A, B, C, D, z, bias, softplus, h0, lengths, absolute=False):
    """(y, h_last).  With absolute, every addend counts by its magnitude: what
    a rounding error is relative to."""
    u, delta, A, B, C, D, z, bias, h0 = f64(u, delta, A, B, C, D, z, bias, h0)
    mag = np.abs if absolute else lambda v: v
    nb, L, nd = u.shape
    y = np.zeros((nb, L, nd))
    last = np.zeros((nb, nd, A.shape[1]))
    for b in range(nb):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        h = mag(h0[b]) if h0 is not None else np.zeros((nd, A.shape[1]))
        for t in range(n):
            s, _ = _step(delta[b, t], bias, softplus)
            h = np.exp(s[:, None] * A) * h + mag((s * u[b, t])[:, None] * _spread(B[b, t], nd))
            p = (h * mag(_spread(C[b, t], nd))).sum(axis=1) + (mag(D * u[b, t]) if D is not None else 0.0)
            y[b, t] = p if z is None else p * mag(z[b, t] * sigmoid(z[b, t]))
        last[b] = h
    return y, last


def selective_scan_bwd(u, delta, A, B, C, D, z, bias, softplus, h0, lengths, dy, dlast, absolute=False):
    """dict of gradients, rows past a sequence's end zero; absolute as above."""
    u, delta, A, B, C, D, z, bias, h0, dy, dlast = f64(u, delta, A, B, C, D, z, bias, h0, dy, dlast)
    mag = np.abs if absolute else lambda v: v
    nb, L, nd = u.shape
    N, G = A.shape[1], B.shape[2]
    out = dict(du=np.zeros_like(u), ddelta=np.zeros_like(u), dA=np.zeros_like(A), dB=np.zeros_like(B),
               dC=np.zeros_like(C), dD=np.zeros(nd), dz=np.zeros_like(u), ddelta_bias=np.zeros(nd),
               dh0=np.zeros((nb, nd, N)))
    for b in range(nb):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        h = mag(h0[b]) if h0 is not None else np.zeros((nd, N))
        hs = [h]
        for t in range(n):
            s, _ = _step(delta[b, t], bias, softplus)
            h = np.exp(s[:, None] * A) * h + mag((s * u[b, t])[:, None] * _spread(B[b, t], nd))
            hs.append(h)
        g = mag(dlast[b]) if dlast is not None else np.zeros((nd, N))
        for t in reversed(range(n)):
            s, ds = _step(delta[b, t], bias, softplus)
            Bt, Ct, ut = mag(_spread(B[b, t], nd)), mag(_spread(C[b, t], nd)), mag(u[b, t])
            p = (hs[t + 1] * Ct).sum(axis=1) + (mag(D) * ut if D is not None else 0.0)
            dp = mag(dy[b, t])
            if z is not None:
                sz = sigmoid(z[b, t])
                # silu' = sz (1 + z (1 - sz)) has a zero at z = -1.28, where its two
                # addends cancel: their rounding is relative to each of them
                out["dz"][b, t] = dp * p * sz * (1 + mag(z[b, t]) * (1 - sz))
                dp = dp * mag(z[b, t] * sz)
            g = g + Ct * dp[:, None]
            decay = np.exp(s[:, None] * A)
            geh = g * decay * hs[t]
            gb = (g * Bt).sum(axis=1)
            step = mag(s)
            out["dC"][b, t] = (dp[:, None] * hs[t + 1]).reshape(G, -1, N).sum(axis=1)
            out["dB"][b, t] = (g * (step * ut)[:, None]).reshape(G, -1, N).sum(axis=1)
            out["dA"] += geh * step[:, None]
            out["du"][b, t] = step * gb + (mag(D) * dp if D is not None else 0.0)
            out["ddelta"][b, t] = ((geh * mag(A)).sum(axis=1) + ut * gb) * mag(ds)
            out["dD"] += dp * ut
            out["ddelta_bias"] += out["ddelta"][b, t]
            g = g * decay
        out["dh0"][b] = g
    return out
