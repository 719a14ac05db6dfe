"""Sequence operators on the GPU against their 64-bit definitions
(tests/seq_reference.py).

Tolerances come from counting roundings (half a unit in the last place, E =
2^-24 of the value, each), relative to the sum of the magnitudes that went in:
* norm: a sum of D squares in parts of at most D / 32 + 64 additions, half of
  its error in the reciprocal root, and 8 roundings after it;
* conv: W + 3 roundings of the sum; silu adds the 2 + 1.2 |p| units (2 E) of
  its exponential and has slope at most 1.1;
* scan: each of at most L decays is off by 2^-22 (ex2.approx) and each state
  update by two roundings, so (4 + 2) L E, and 64 E for the step, the gate and
  the sum over states; a decay exp(s A) also carries the error of s A, whose
  effect s A exp(s A) on a weight is at most 1/e times the relative error of
  s: within the 64 E.  Gradients multiply a forward and an adjoint state, twice
  that, and sums over B L positions or D channels add one rounding per term."""

from __future__ import annotations

import numpy as np
import pytest

import seq_reference as ref
from conftest import to_host
from remora_b200 import ops
from remora_b200.errors import RemoraB200Error, RemoraShapeError, RemoraUnsupportedError

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TINY = 1e-30


def dev(a, cuda):
    import torch

    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(cuda)


def rnd(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float32)


def within(got, want, bound, what=""):
    got = got if isinstance(got, np.ndarray) else to_host(got)
    err = np.abs(got.astype(np.float64) - want)
    worst = (err / (bound + TINY)).max() if err.size else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound (largest error {err.max():.3g})"


# ------------------------------------------------------------------- norm
def norm_tol(D):
    return (D / 32 + 64) / 2 * E + 8 * E


SHAPES = [(1, 1), (5, 3), (3, 31), (7, 128), (700, 33), (2, 1000), (600, 1000), (9, 2048), (1, 8192), (3, 8193),
          (2, 16384), (2, 16388), (2, 20001), (1300, 64), (9000, 37), (4001, 1003)]


@pytest.mark.parametrize("rows,D", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_forward(cuda, rows, D, residual):
    rng = np.random.default_rng(rows * 31 + D)
    x, w = rnd(rng, rows, D), rnd(rng, D)
    r = rnd(rng, rows, D, scale=3) if residual else None
    got = ops.rms_norm_fwd(dev(x, cuda), dev(w, cuda), residual=dev(r, cuda), eps=1e-5)
    y, s = ref.rms_norm(x, w, r, 1e-5)
    if residual:
        got, total = got
        np.testing.assert_array_equal(to_host(total), x + r)  # one f32 addition
        # y from the rounded sum: its error is half a unit of s at most
    within(got, y, np.abs(y) * norm_tol(D) + np.abs(w) * np.abs(y / np.where(w == 0, 1, w)) * E, "y")


@pytest.mark.parametrize("rows,D", SHAPES)
@pytest.mark.parametrize("through", [False, True])
def test_norm_backward(cuda, rows, D, through):
    rng = np.random.default_rng(rows * 37 + D)
    s, w, dy = rnd(rng, rows, D), rnd(rng, D), rnd(rng, rows, D)
    ds = rnd(rng, rows, D) if through else None
    dx, dw = ops.rms_norm_bwd(dev(s, cuda), dev(w, cuda), dev(dy, cuda), dsum=dev(ds, cuda), eps=1e-5)
    rx, rw = ref.rms_norm_bwd(s, w, dy, ds, 1e-5)
    s6 = s.astype(np.float64)
    rstd = 1 / np.sqrt((s6 * s6).mean(axis=1, keepdims=True) + 1e-5)
    mean = np.abs(s6 * rstd * w * dy).mean(axis=1, keepdims=True)
    mag = rstd * (np.abs(w * dy) + np.abs(s6 * rstd) * mean) + (np.abs(ds) if through else 0)
    within(dx, rx, mag * 4 * norm_tol(D), "dx")
    within(dw, rw, np.abs(dy * s6 * rstd).sum(axis=0) * (norm_tol(D) + rows * E + 8 * E), "dw")


@pytest.mark.parametrize("D", [64, 2048, 3001])
def test_norm_in_place_and_strided(cuda, D):
    import torch

    rng = np.random.default_rng(D)
    B, T = 3, 5
    base = dev(rnd(rng, T, B, 2 * D + 3), cuda)
    x = base.transpose(0, 1)[:, :, 3:3 + D]  # two leading axes that do not collapse, unaligned
    r = dev(rnd(rng, B, T, D), cuda)
    w = dev(rnd(rng, 2 * D), cuda)[::2]
    xh, rh, wh = to_host(x), to_host(r), to_host(w)
    y, s = ref.rms_norm(xh, wh, rh, 1e-6)
    tol = np.abs(y) * norm_tol(D) + np.abs(y) * E
    got = ops.rms_norm_fwd(x, w, residual=r, out=x, sum_out=r)
    assert got[0] is x and got[1] is r
    within(x, y, tol, "y over x")
    np.testing.assert_array_equal(to_host(r), xh + rh)
    dy = dev(rnd(rng, D, B, T), cuda).permute(1, 2, 0)  # last axis not the fastest
    want, wdw = ref.rms_norm_bwd(to_host(r), wh, to_host(dy), None, 1e-6)
    dx, dw = ops.rms_norm_bwd(r, w, dy, out=dy)
    assert dx is dy
    dx2, dw2 = ops.rms_norm_bwd(r, w, dev(to_host(dy) * 0, cuda))
    assert torch.count_nonzero(dx2) == 0 and torch.count_nonzero(dw2) == 0
    np.testing.assert_allclose(to_host(dx), want, rtol=0, atol=4 * norm_tol(D) * 40)
    np.testing.assert_allclose(to_host(dw), wdw, rtol=0, atol=4 * norm_tol(D) * 100)
    flat = ops.rms_norm_fwd(r[0, 0], w)
    np.testing.assert_array_equal(to_host(flat), to_host(ops.rms_norm_fwd(r, w))[0, 0])


@pytest.mark.parametrize("rows,D,group", [(3, 64, 0), (1, 2048, 0), (800, 128, 32), (5, 4096, 128), (4, 192, 64),
                                          (3, 77, 0), (2, 20000, 0), (2, 20000, 32), (700, 1001, 0)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_quant(cuda, rows, D, group, residual):
    rng = np.random.default_rng(rows + D + group)
    x, w = rnd(rng, rows, D), rnd(rng, D)
    if rows > 2:
        x[1] = 0.0  # scales stay at their least
    r = rnd(rng, rows, D) if residual else None
    if residual and rows > 2:
        r[1] = 0.0
    q, sc, *rest = ops.rms_norm_quant(dev(x, cuda), dev(w, cuda), residual=dev(r, cuda), eps=1e-6, group=group)
    assert len(rest) == int(residual)
    y, _ = ref.rms_norm(x, w, r, 1e-6)
    g = group or D
    yg = y.reshape(rows, D // g, g)
    want = np.maximum(np.abs(yg).max(axis=2) / 448, 2.0 ** -126)
    tol = norm_tol(D) + 4 * E
    within(sc, want, want * tol, "scales")
    scale = to_host(sc).astype(np.float64)[:, :, None]
    qv = to_host(q.float()).reshape(yg.shape).astype(np.float64)
    v = np.clip(yg / scale, -448, 448)
    levels = ref.e4m3_values()
    i = np.searchsorted(levels, np.abs(v)).clip(1, len(levels) - 1)
    nearest = np.minimum(np.abs(levels[i] - np.abs(v)), np.abs(levels[i - 1] - np.abs(v)))
    # q is a nearest level of the value, or of one the rounding of y moved it to
    assert np.isin(np.abs(qv), levels).all()
    assert (np.abs(qv - v) <= nearest + 2 * np.abs(v) * (tol + 4 * E) + TINY).all()
    if rows > 2:
        assert (qv[1] == 0).all() and (scale[1] == 2.0 ** -126).all()


def test_norm_quant_misaligned_groups_equal_aligned(cuda):
    rng = np.random.default_rng(3)
    x = dev(rnd(rng, 5, 257), cuda)
    w = dev(rnd(rng, 256), cuda)
    a, sa = ops.rms_norm_quant(x[:, 1:], w, group=64)
    b, sb = ops.rms_norm_quant(x[:, 1:].contiguous(), w, group=64)
    # the sums of squares run in another order: scales differ by roundings
    within(sa, to_host(sb).astype(np.float64), to_host(sb) * 2 * (norm_tol(256) + 4 * E))
    assert (to_host(a.float()) != to_host(b.float())).mean() < 1e-2


def test_norm_rows_are_independent_of_bad_rows(cuda):
    rng = np.random.default_rng(4)
    for D in (96, 1001, 20000):
        x = rnd(rng, 5, D)
        clean = to_host(ops.rms_norm_fwd(dev(x, cuda), dev(np.ones(D, np.float32), cuda)))
        x[1, 3], x[3, 7] = np.nan, np.inf
        y = to_host(ops.rms_norm_fwd(dev(x, cuda), dev(np.ones(D, np.float32), cuda)))
        np.testing.assert_array_equal(y[[0, 2, 4]], clean[[0, 2, 4]])
        assert np.isnan(y[1]).all() and np.isnan(y[3, 7])
        q, s = ops.rms_norm_quant(dev(x, cuda), dev(np.ones(D, np.float32), cuda))
        s = to_host(s)
        assert np.isnan(s[[1, 3]]).all() and np.isfinite(s[[0, 2, 4]]).all()


def test_norm_empty(cuda):
    import torch

    z = torch.zeros((0, 8), device=cuda)
    w = torch.ones(8, device=cuda)
    assert ops.rms_norm_fwd(z, w).shape == (0, 8)
    dx, dw = ops.rms_norm_bwd(z, w, z)
    assert dx.shape == (0, 8) and to_host(dw).tolist() == [0.0] * 8
    with pytest.raises(RemoraShapeError):
        ops.rms_norm_fwd(torch.zeros((4, 0), device=cuda), torch.zeros(0, device=cuda))


# ------------------------------------------------------------------- conv
def conv_tol(x, w, b, state, lengths, silu):
    """Bound on |y| errors: the sum's, then silu's."""
    a = lambda v: None if v is None else np.abs(v)  # noqa: E731
    W = w.shape[1]
    p, _ = ref.causal_conv(x, w, b, state, lengths, False)
    mag, _ = ref.causal_conv(a(x), a(w), a(b), a(state), lengths, False)
    tol = mag * (W + 3) * E * 1.1
    if silu:
        tol = tol + np.abs(p * ref.sigmoid(p)) * (4 + 1.2 * np.abs(p)) * 2 * E + np.abs(p) * 2.0 ** -120
    return tol


CONVS = [(1, 1, 1, 2), (2, 1, 4, 4), (3, 2, 8, 4), (2, 7, 5, 3), (1, 300, 128, 4), (2, 777, 33, 2), (1, 65, 132, 8),
         (2, 513, 4, 5), (3, 40, 256, 6), (1, 9, 3, 7)]


@pytest.mark.parametrize("B,T,D,W", CONVS)
@pytest.mark.parametrize("silu,full", [(False, False), (True, False), (True, True)])
def test_conv_forward_backward(cuda, B, T, D, W, silu, full):
    rng = np.random.default_rng(B * 1000 + T + D + W)
    x, w, dy = rnd(rng, B, T, D), rnd(rng, D, W), rnd(rng, B, T, D)
    b = rnd(rng, D) if full else None
    state = rnd(rng, B, W - 1, D) if full else None
    dlast = rnd(rng, B, W - 1, D) if full else None
    lengths = rng.integers(0, T + 1, B).astype(np.int32) if full else None
    if full:
        lengths[0] = T
        if B > 1:
            lengths[1] = 0
        for i in range(B):  # what is behind an end is not read
            x[i, lengths[i]:] = np.nan
            dy[i, lengths[i]:] = np.nan
    d = lambda v: dev(v, cuda)  # noqa: E731
    y, last = ops.causal_conv_fwd(d(x), d(w), d(b), state=d(state), lengths=d(lengths), silu=silu, return_state=True)
    x0, dy0 = np.nan_to_num(x), np.nan_to_num(dy)
    ry, rlast = ref.causal_conv(x0, w, b, state, lengths, silu)
    within(y, ry, conv_tol(x0, w, b, state, lengths, silu), "y")
    np.testing.assert_array_equal(to_host(last), rlast.astype(np.float32))
    got = ops.causal_conv_bwd(d(x), d(w), d(dy), d(b), state=d(state), lengths=d(lengths), silu=silu,
                              dstate_out=d(dlast))
    want = ref.causal_conv_bwd(x0, w, b, state, lengths, silu, dy0, dlast)
    a = np.abs
    an = lambda v: None if v is None else a(v)  # noqa: E731
    mag = ref.causal_conv_bwd(a(x0), a(w), None, an(state), lengths, False, a(dy0), an(dlast))
    # silu' is at most 1.1 in size and its error that of the sigmoid and of p
    # (slope at most 0.5): p up to some 10, so 30 units
    pmax = float(ref.causal_conv(a(x0), a(w), an(b), an(state), lengths, False)[0].max())
    k = (W + 4) * E * 1.1 + (((8 + 2.4 * pmax) * 2 * E + pmax * (W + 3) * E) if silu else 0)
    n = B * T
    for name, g, r, m, extra in zip(("dx", "dw", "dbias", "dstate"), got, want, mag, (0, n, n, 0)):
        if g is not None:
            within(g, r, m * (k * 1.2 + extra * E * 1.1), name)
    assert (got[2] is None) == (b is None) and (got[3] is None) == (state is None)


def test_conv_rows_behind_the_end_stay_as_they_were(cuda):
    import torch

    rng = np.random.default_rng(7)
    x, w = dev(rnd(rng, 2, 50, 12), cuda), dev(rnd(rng, 12, 4), cuda)
    lengths = torch.tensor([50, 13], dtype=torch.int32, device=cuda)
    for out in (torch.full((2, 50, 12), 7.0, device=cuda), torch.full((2, 50, 13), 7.0, device=cuda)[:, :, 1:]):
        ops.causal_conv_fwd(x, w, lengths=lengths, out=out)
        assert (to_host(out)[1, 13:] == 7).all() and (to_host(out)[1, :13] != 7).all()
        ops.causal_conv_bwd(x, w, x, lengths=lengths, out=out.fill_(7.0))
        assert (to_host(out)[1, 13:] == 7).all() and (to_host(out)[1, :13] != 7).all()
    wild = torch.tensor([99, -5], dtype=torch.int32, device=cuda)  # as 50 and 0
    full = to_host(ops.causal_conv_fwd(x, w))
    got = to_host(ops.causal_conv_fwd(x, w, lengths=wild))
    np.testing.assert_array_equal(got[0], full[0])
    assert (got[1] == 0).all()


def test_conv_strided_views_equal_contiguous(cuda):
    import torch

    rng = np.random.default_rng(8)
    for D in (8, 13):
        wide = dev(rnd(rng, 2, 90, 2 * D), cuda)
        x, z = wide[:, :, :D], wide[:, :, D:]
        w = dev(rnd(rng, 4, D), cuda).t()
        want = ops.causal_conv_fwd(x.contiguous(), w.contiguous(), silu=True)
        ops.causal_conv_fwd(x, w, silu=True, out=z)  # the other columns of the same buffer
        np.testing.assert_array_equal(to_host(z), to_host(want))
        tm = x.contiguous().transpose(1, 2).contiguous().transpose(1, 2)  # time fastest
        assert tm.stride(1) == 1
        np.testing.assert_array_equal(to_host(ops.causal_conv_fwd(tm, w, silu=True)), to_host(want))
        flip = torch.empty_like(tm)
        dx, dw, _, _ = ops.causal_conv_bwd(tm, w, z, silu=True, out=flip)
        dx2, dw2, _, _ = ops.causal_conv_bwd(x.contiguous(), w.contiguous(), z.contiguous(), silu=True)
        np.testing.assert_array_equal(to_host(dx), to_host(dx2))
        shared = dev(rnd(rng, 1, 1, D), cuda).expand(2, 90, D)  # a broadcast input: strides 0
        np.testing.assert_array_equal(to_host(ops.causal_conv_fwd(shared, w)),
                                      to_host(ops.causal_conv_fwd(shared.contiguous(), w)))


@pytest.mark.parametrize("D,W", [(4, 4), (5, 2), (300, 3), (1024, 8)])
def test_conv_steps_continue_a_prompt(cuda, D, W):
    rng = np.random.default_rng(D + W)
    B, T = 3, 12
    x, w, b = rnd(rng, B, T, D), rnd(rng, D, W), rnd(rng, D)
    full, last = ref.causal_conv(x, w, b, None, None, True)
    tol = conv_tol(x, w, b, None, None, True)
    xd, wd, bd = dev(x, cuda), dev(w, cuda), dev(b, cuda)
    y, state = ops.causal_conv_fwd(xd[:, :5], wd, bd, silu=True, return_state=True)
    within(y, full[:, :5], tol[:, :5])
    y, out = ops.causal_conv_fwd(xd[:, 5:7], wd, bd, silu=True, state=state, state_out=state)  # in place, short
    assert out is state
    within(y, full[:, 5:7], tol[:, 5:7])
    for t in range(7, T):
        y = ops.causal_conv_step(xd[:, t], state, wd, bd, silu=True)
        within(y, full[:, t], tol[:, t], f"step {t}")
    np.testing.assert_array_equal(to_host(state), last.astype(np.float32))


@pytest.mark.parametrize("D", [8, 9])
def test_step_slots(cuda, D):
    """Rows of a pool by index; padding, repeated and out-of-range indices."""
    import torch

    rng = np.random.default_rng(D)
    W, N, S, B = 4, 5, 7, 6
    slots = torch.tensor([3, -1, 6, 3, 7, 0], dtype=torch.int32, device=cuda)
    used, rows = [3, 6, 0], [0, 2, 5]
    x, w, pool = dev(rnd(rng, B, D), cuda), dev(rnd(rng, D, W), cuda), dev(rnd(rng, S, W - 1, D), cuda)
    before = to_host(pool)
    alone = pool[used].clone()
    want = ops.causal_conv_step(x[rows], alone, w, silu=True)
    y = ops.causal_conv_step(x, pool, w, silu=True, slots=slots, out=torch.full((B, D), 7.0, device=cuda))
    y, after = to_host(y), to_host(pool)
    np.testing.assert_array_equal(y[rows], to_host(want))
    assert (y[[1, 3, 4]] == 7).all()
    np.testing.assert_array_equal(after[used], to_host(alone))
    keep = [i for i in range(S) if i not in used]
    np.testing.assert_array_equal(after[keep], before[keep])
    h = dev(rnd(rng, S, D, N), cuda)
    before = to_host(h)
    u, dl, z = (dev(rnd(rng, B, D), cuda) for _ in range(3))
    A, Bm, C = dev(-np.abs(rnd(rng, D, N)), cuda), dev(rnd(rng, B, N), cuda), dev(rnd(rng, B, N), cuda)
    alone = h[used].clone()
    want = ops.selective_scan_step(alone, u[rows], dl[rows], A, Bm[rows], C[rows], z=z[rows], softplus=True)
    other = torch.zeros_like(h)
    y2 = ops.selective_scan_step(h, u, dl, A, Bm, C, z=z, softplus=True, slots=slots, state_out=other)
    np.testing.assert_array_equal(to_host(y2)[rows], to_host(want))
    assert (to_host(y2)[[1, 3, 4]] == 0).all() and (to_host(other)[keep] == 0).all()
    np.testing.assert_array_equal(to_host(other)[used], to_host(alone))
    np.testing.assert_array_equal(to_host(h), before)


# ------------------------------------------------------------------- scan
def scan_inputs(rng, B, T, D, N, G, full):
    v = dict(u=rnd(rng, B, T, D), delta=rnd(rng, B, T, D, scale=0.5),
             A=-np.exp(rnd(rng, D, N, scale=0.3) + np.log(np.arange(1, N + 1))).astype(np.float32),
             B=rnd(rng, B, T, G, N), C=rnd(rng, B, T, G, N), D=None, z=None, bias=None, h0=None)
    if full:
        v.update(D=rnd(rng, D), z=rnd(rng, B, T, D), bias=rnd(rng, D) - 3, h0=rnd(rng, B, D, N))
    return v


def scan_own(v, cuda):
    d = {k: dev(a, cuda) for k, a in v.items()}
    return (d["u"], d["delta"], d["A"], d["B"], d["C"]), d["D"], dict(z=d["z"], delta_bias=d["bias"], h0=d["h0"])


NAMES = ("du", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dh0")
SCANS = [(1, 1, 1, 1, 1), (2, 3, 5, 4, 1), (1, 17, 40, 16, 1), (2, 70, 34, 16, 2), (1, 200, 8, 16, 1),
         (2, 33, 12, 13, 3), (1, 37, 6, 64, 1), (1, 50, 9, 33, 1), (2, 40, 64, 2, 1), (1, 45, 130, 8, 1), (1, 300, 3, 7, 1)]


@pytest.mark.parametrize("B,T,D,N,G", SCANS)
@pytest.mark.parametrize("full", [False, True])
def test_scan_forward_backward(cuda, B, T, D, N, G, full):
    rng = np.random.default_rng(B + T * 7 + D * 3 + N)
    v = scan_inputs(rng, B, T, D, N, G, full)
    softplus = full
    if not softplus:
        v["delta"] = np.abs(v["delta"]) * np.float32(0.2)
    lengths = None
    dy = rnd(rng, B, T, D)
    dlast = rnd(rng, B, D, N) if full else None
    if full and B > 1:
        lengths = rng.integers(1, T + 1, B).astype(np.int32)
        lengths[1] = 0
    clean = {k: None if a is None else a.copy() for k, a in v.items()}
    dyc = dy.copy()
    if lengths is not None:
        for i in range(B):
            for k in ("u", "delta", "B", "C", "z"):
                v[k][i, lengths[i]:] = np.nan
            dy[i, lengths[i]:] = np.nan
    pos, Dv, kw = scan_own(v, cuda)
    ln = dev(lengths, cuda)
    y, last, saved = ops.selective_scan_fwd(*pos, Dv, softplus=softplus, lengths=ln, return_state=True, save=True, **kw)
    args = (*(clean[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), softplus, clean["h0"], lengths)
    ry, rlast = ref.selective_scan(*args)
    my, mlast = ref.selective_scan(*args, absolute=True)
    tol = (6 * T + 64) * E
    within(y, ry, my * tol, "y")
    within(last, rlast, mlast * tol, "h_last")
    got = ops.selective_scan_bwd(*pos, dev(dy, cuda), saved, Dv, softplus=softplus, lengths=ln,
                                 dh_last=dev(dlast, cuda), **kw)
    want = ref.selective_scan_bwd(*args, dyc, dlast)
    mag = ref.selective_scan_bwd(*args, dyc, dlast, absolute=True)
    for name, g in zip(NAMES, got):
        if g is None:
            continue
        extra = {"dA": B * T, "dD": B * T, "ddelta_bias": B * T, "dB": D, "dC": D}.get(name, 0)
        within(g, want[name], mag[name] * (2 * tol + extra * E), name)
    assert [g is None for g in got] == [False] * 5 + [not full] * 4


@pytest.mark.parametrize("T", [1, 31, 32, 33, 640, 1000])
@pytest.mark.parametrize("N", [16, 5])
def test_scan_cut_in_time(cuda, T, N):
    """Few channels and many positions: pieces of the time axis joined; a
    prompt in two calls gives the same."""
    rng = np.random.default_rng(T + N)
    v = scan_inputs(rng, 2, T, 3, N, 1, True)
    lengths = np.array([T, max(0, T - 37)], np.int32)
    pos, Dv, kw = scan_own(v, cuda)
    y, last, saved = ops.selective_scan_fwd(*pos, Dv, softplus=True, lengths=dev(lengths, cuda), return_state=True,
                                            save=True, **kw)
    args = (*(v[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True, v["h0"], lengths)
    ry, rlast = ref.selective_scan(*args)
    my, mlast = ref.selective_scan(*args, absolute=True)
    tol = (6 * T + 64) * E
    within(y, ry, my * tol, "y")
    within(last, rlast, mlast * tol, "h_last")
    dy, dlast = rnd(rng, 2, T, 3), rnd(rng, 2, 3, N)
    got = ops.selective_scan_bwd(*pos, dev(dy, cuda), saved, Dv, softplus=True, lengths=dev(lengths, cuda),
                                 dh_last=dev(dlast, cuda), **kw)
    want = ref.selective_scan_bwd(*args, dy, dlast)
    mag = ref.selective_scan_bwd(*args, dy, dlast, absolute=True)
    for name, g in zip(NAMES, got):
        within(g, want[name], mag[name] * (2 * tol + (2 * T + 8) * E), name)
    if T >= 33:
        cut = T // 2
        first = {k: (a[:, :cut] if k in ("u", "delta", "B", "C", "z") else a) for k, a in v.items()}
        rest = {k: (a[:, cut:] if k in ("u", "delta", "B", "C", "z") else a) for k, a in v.items()}
        pos, Dv, kw = scan_own(first, cuda)
        y1, state = ops.selective_scan_fwd(*pos, Dv, softplus=True, return_state=True, **kw)
        pos, Dv, kw = scan_own(rest, cuda)
        kw["h0"] = state
        y2, out = ops.selective_scan_fwd(*pos, Dv, softplus=True, h_last=state, **kw)  # in place
        assert out is state
        within(np.concatenate([to_host(y1), to_host(y2)], axis=1)[0], ry[0], my[0] * tol, "two calls")
        within(to_host(state)[0], rlast[0], mlast[0] * tol, "two calls' state")


@pytest.mark.parametrize("N", [1, 4, 8, 7, 32, 24, 64, 50])
def test_scan_cut_in_time_of_other_state_counts(cuda, N):
    test_scan_cut_in_time(cuda, 203, N)


@pytest.mark.parametrize("D,N,G", [(6, 16, 1), (10, 13, 2), (64, 4, 1), (33, 64, 3), (3, 1, 1)])
def test_scan_steps_continue_a_prompt(cuda, D, N, G):
    rng = np.random.default_rng(D + N)
    B, T = 3, 9
    v = scan_inputs(rng, B, T, D, N, G, True)
    args = (*(v[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True, v["h0"], None)
    ry, rlast = ref.selective_scan(*args)
    my, mlast = ref.selective_scan(*args, absolute=True)
    tol = (6 * T + 64) * E
    head = {k: (a[:, :4] if k in ("u", "delta", "B", "C", "z") else a) for k, a in v.items()}
    pos, Dv, kw = scan_own(head, cuda)
    y, state = ops.selective_scan_fwd(*pos, Dv, softplus=True, return_state=True, **kw)
    within(y, ry[:, :4], my[:, :4] * tol)
    d = {k: dev(a, cuda) for k, a in v.items()}
    for t in range(4, T):
        y = ops.selective_scan_step(state, d["u"][:, t], d["delta"][:, t], d["A"], d["B"][:, t], d["C"][:, t], d["D"],
                                    z=d["z"][:, t], delta_bias=d["bias"], softplus=True)
        within(y, ry[:, t], my[:, t] * tol, f"step {t}")
    within(state, rlast, mlast * tol, "state")


@pytest.mark.parametrize("N,G", [(16, 1), (16, 3), (13, 1), (12, 2), (8, 1), (7, 1), (24, 1), (64, 2), (33, 1), (4, 1)])
@pytest.mark.parametrize("pool", [False, True])
def test_scan_step_of_many_rows(cuda, N, G, pool):
    """Several rows per thread, the last group of them not full; in a pool some
    rows are left out: padding, out of range, named before in the same group of
    rows and in an earlier one."""
    rng = np.random.default_rng(N * 10 + G)
    B, D = 251, 300
    S = B + 30 if pool else B
    v = {k: None if a is None else a[:, 0] if k in ("u", "delta", "B", "C", "z") else a
         for k, a in scan_inputs(rng, B, 1, D, N, G, True).items()}
    h = rnd(rng, S, D, N)
    slots = np.arange(B, dtype=np.int32)
    out = np.zeros(B, bool)
    if pool:
        slots = rng.permutation(S)[:B].astype(np.int32)
        slots[[0, 101, 102]], slots[9], slots[10], slots[250] = -1, slots[8], S, slots[3]
        out[[0, 9, 10, 101, 102, 250]] = True
    args = (*(v[k][:, None] if k in ("u", "delta", "B", "C", "z") else v[k]
              for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True, h[np.where(out, 0, slots)], 1 - out)
    ry, rlast = ref.selective_scan(*args)
    my, mlast = ref.selective_scan(*args, absolute=True)
    tol = (6 + 64) * E
    d = {k: dev(a, cuda) for k, a in v.items()}
    state = dev(h, cuda)
    y = ops.selective_scan_step(state, d["u"], d["delta"], d["A"], d["B"], d["C"], d["D"], z=d["z"],
                                delta_bias=d["bias"], softplus=True, slots=dev(slots, cuda) if pool else None)
    within(y, ry[:, 0], my[:, 0] * tol, "y")
    after = to_host(state)
    within(after[slots[~out]], rlast[~out], mlast[~out] * tol, "state")
    rest = np.setdiff1d(np.arange(S), slots[~out])
    np.testing.assert_array_equal(after[rest], h[rest])


def test_scan_without_channels(cuda):
    """No channels: the gradients of b and c are sums of nothing."""
    import torch

    z = lambda *s: torch.zeros(s, device=cuda)
    bc = torch.ones(2, 5, 3, device=cuda)
    y, h, saved = ops.selective_scan_fwd(z(2, 5, 0), z(2, 5, 0), z(0, 3), bc, bc, return_state=True, save=True)
    assert y.shape == (2, 5, 0) and h.shape == (2, 0, 3)
    got = ops.selective_scan_bwd(z(2, 5, 0), z(2, 5, 0), z(0, 3), bc, bc, z(2, 5, 0), saved)
    assert (got[3] == 0).all() and (got[4] == 0).all() and got[3].shape == bc.shape


def test_scan_strided_views_equal_contiguous(cuda):
    import torch

    rng = np.random.default_rng(11)
    B, T, D, N = 2, 40, 24, 16
    wide = dev(rnd(rng, B, T, 2 * D + 2 * N + 1), cuda)
    u, delta, Bm, C = wide[:, :, 1:D + 1], wide[:, :, D + 1:2 * D + 1], wide[:, :, 2 * D + 1:2 * D + N + 1], wide[:, :, 2 * D + N + 1:]
    A = dev(-np.abs(rnd(rng, N, D)), cuda).t()
    z = dev(rnd(rng, B, D, T), cuda).transpose(1, 2)
    one = [t.contiguous() for t in (u, delta, A, Bm, C)]
    y1, s1 = ops.selective_scan_fwd(*one, z=z.contiguous(), softplus=True, save=True)
    y2, s2 = ops.selective_scan_fwd(u, delta, A, Bm, C, z=z, softplus=True, save=True)
    np.testing.assert_array_equal(to_host(y2), to_host(y1))
    dy = dev(rnd(rng, D, T, B), cuda).permute(2, 1, 0)
    g1 = ops.selective_scan_bwd(*one, dy.contiguous(), s1, z=z.contiguous(), softplus=True)
    g2 = ops.selective_scan_bwd(u, delta, A, Bm, C, dy, s2, z=z, softplus=True)
    for a, b in zip(g1, g2):
        if a is not None:
            np.testing.assert_array_equal(to_host(a), to_host(b))
    # one step size for all channels, one b and c for all positions: stride 0
    few = dev(np.abs(rnd(rng, B, T, 1)), cuda).expand(B, T, D)
    bc = dev(rnd(rng, 1, 1, N), cuda).expand(B, T, N)
    y3 = ops.selective_scan_fwd(u, few, A, bc, bc)
    y4 = ops.selective_scan_fwd(u.contiguous(), few.contiguous(), A, bc.contiguous(), bc.contiguous())
    np.testing.assert_array_equal(to_host(y3), to_host(y4))
    out = torch.full((B, T, D), 7.0, device=cuda)
    ops.selective_scan_fwd(*one, lengths=torch.tensor([T, 5], dtype=torch.int32, device=cuda), out=out)
    assert (to_host(out)[1, 5:] == 7).all()


@pytest.mark.parametrize("N", [16, 13])
def test_scan_bad_values_stay_in_their_channel(cuda, N):
    rng = np.random.default_rng(12)
    v = scan_inputs(rng, 1, 40, 40, N, 1, True)
    pos, Dv, kw = scan_own(v, cuda)
    clean = to_host(ops.selective_scan_fwd(*pos, Dv, softplus=True, **kw))
    v["u"][0, 10, 3], v["delta"][0, 11, 7] = np.nan, np.inf
    pos, Dv, kw = scan_own(v, cuda)
    y = to_host(ops.selective_scan_fwd(*pos, Dv, softplus=True, **kw))
    others = [d for d in range(40) if d not in (3, 7)]
    np.testing.assert_array_equal(y[:, :, others], clean[:, :, others])
    np.testing.assert_array_equal(y[:, :10], clean[:, :10])
    assert np.isnan(y[0, 10:, 3]).all()
    # a decay of minus infinity forgets the state at once
    v = scan_inputs(rng, 1, 6, 4, N, 1, False)
    v["A"][:] = -np.inf
    v["delta"] = np.abs(v["delta"]) + np.float32(0.1)
    pos, Dv, kw = scan_own(v, cuda)
    y = to_host(ops.selective_scan_fwd(*pos))
    want = v["delta"] * v["u"] * (v["B"][:, :, 0] * v["C"][:, :, 0]).sum(axis=-1, keepdims=True)
    np.testing.assert_allclose(y, want, rtol=1e-4, atol=1e-5)


def test_offsets_past_32_bits(cuda):
    """Rows whose addresses lie more than 2^32 bytes apart, and axes of one
    element with strides that mean nothing."""
    import torch

    rng = np.random.default_rng(13)
    far = 1 << 30  # elements: 4 GiB
    buf = torch.empty(2 * far + (1 << 20), dtype=torch.float32, device=cuda)
    D, N, T = 20, 16, 9
    wide = buf.as_strided((3, T, D), (far, 4 * D, 1))
    x = dev(rnd(rng, 3, T, D), cuda)
    wide.copy_(x)
    w = dev(rnd(rng, D), cuda)
    np.testing.assert_array_equal(to_host(ops.rms_norm_fwd(wide, w)), to_host(ops.rms_norm_fwd(x, w)))
    cw, cb = dev(rnd(rng, D, 4), cuda), dev(rnd(rng, D), cuda)
    np.testing.assert_array_equal(to_host(ops.causal_conv_fwd(wide, cw, cb)), to_host(ops.causal_conv_fwd(x, cw, cb)))
    A, b, c = dev(-np.abs(rnd(rng, D, N)), cuda), dev(rnd(rng, 3, T, N), cuda), dev(rnd(rng, 3, T, N), cuda)
    want = ops.selective_scan_fwd(x, x, A, b, c, softplus=True, z=x, save=True, return_state=True)
    out = buf.as_strided((3, T, D), (far, 4 * D, 1), D)  # beside the input
    got = ops.selective_scan_fwd(wide, wide, A, b, c, softplus=True, z=wide, save=True, return_state=True, out=out)
    for g, r in zip(got, want):
        np.testing.assert_array_equal(to_host(g), to_host(r))
    for g, r in zip(ops.selective_scan_bwd(wide, wide, A, b, c, wide, got[2], z=wide, softplus=True),
                    ops.selective_scan_bwd(x, x, A, b, c, x, want[2], z=x, softplus=True)):
        if g is not None:
            np.testing.assert_array_equal(to_host(g), to_host(r))
    state = buf.as_strided((3, D, N), (far, N, 1), 1 << 12)
    state.copy_(want[1])
    y = ops.selective_scan_step(state, x[:, 0], x[:, 1], A, b[:, 0], c[:, 0], softplus=True)
    plain = want[1].clone()
    np.testing.assert_array_equal(to_host(y), to_host(ops.selective_scan_step(plain, x[:, 0], x[:, 1], A, b[:, 0],
                                                                             c[:, 0], softplus=True)))
    np.testing.assert_array_equal(to_host(state), to_host(plain))
    one = x[:1, :1].as_strided((1, 1, D), (1 << 40, 1 << 40, 1))
    y = ops.selective_scan_fwd(one, one, A, b[:1, :1], c[:1, :1], softplus=True)
    np.testing.assert_array_equal(to_host(y)[0, 0], to_host(ops.selective_scan_fwd(x, x, A, b, c, softplus=True))[0, 0])
    del buf


def test_negative_strides_through_the_c_abi(cuda):
    """Descriptors may run backwards (torch views cannot): time and channels
    reversed give the reversed arrays' results."""
    import ctypes

    import torch

    from remora_b200 import _lib as L
    from remora_b200.abi import make_memref_descriptor, tensor_descriptor
    from remora_b200.runtime import context

    rng = np.random.default_rng(14)
    B, T, D, N = 2, 21, 70, 16
    u, delta = dev(rnd(rng, B, T, D), cuda), dev(rnd(rng, B, T, D), cuda)
    A, b, c = dev(-np.abs(rnd(rng, D, N)), cuda), dev(rnd(rng, B, T, 1, N), cuda), dev(rnd(rng, B, T, 1, N), cuda)
    back = make_memref_descriptor(u.data_ptr(), (B, T, D), (T * D, -D, -1), offset=(T - 1) * D + D - 1)
    y, out = torch.zeros_like(u), torch.zeros_like(u)
    rev = make_memref_descriptor(out.data_ptr(), (B, T, D), (T * D, -D, -1), offset=(T - 1) * D + D - 1)
    want = ops.selective_scan_fwd(u.flip(1, 2).contiguous(), delta, A, b, c, softplus=True)
    descs = [tensor_descriptor(t) for t in (delta, A, b, c)]
    spec = L.RemoraSelectiveScanSpec(1, 0)
    stream = ctypes.c_void_p(torch.cuda.current_stream(cuda).cuda_stream)
    for to, result in ((tensor_descriptor(y), lambda: y), (rev, lambda: out.flip(1, 2))):
        args = L.RemoraSelectiveScanIn(ctypes.addressof(back), *(ctypes.addressof(x) for x in descs))
        n = ctypes.c_size_t()
        lib, ctx = L.lib(), context(0).ptr
        L.check(lib.remora_b200_selective_scan_fwd_scratch(ctx, B, T, D, N, 1, ctypes.byref(n)))
        scratch = torch.empty(n.value + 16, dtype=torch.uint8, device=cuda)
        L.check(lib.remora_b200_selective_scan_fwd(ctx, ctypes.addressof(spec), ctypes.addressof(args),
                                                   ctypes.addressof(to), None, None, 0, scratch.data_ptr(), n.value,
                                                   stream))
        np.testing.assert_array_equal(to_host(result()), to_host(want))
    cw = dev(rnd(rng, D, 3), cuda)
    conv = L.RemoraCausalConvSpec(0, 0)
    wd, to = tensor_descriptor(cw), tensor_descriptor(y)
    L.check(lib.remora_b200_causal_conv_fwd(ctx, ctypes.addressof(conv), ctypes.addressof(back), ctypes.addressof(wd),
                                            None, None, None, ctypes.addressof(to), None, stream))
    np.testing.assert_array_equal(to_host(y), to_host(ops.causal_conv_fwd(u.flip(1, 2).contiguous(), cw)))


def test_rows_of_no_sequence(cuda):
    """Zero in results made by the call, as they were in a caller's."""
    import torch

    rng = np.random.default_rng(15)
    B, T = 3, 90
    lengths = torch.tensor([90, 0, 41], dtype=torch.int32, device=cuda)
    for D, N, G in ((10, 16, 1), (200, 5, 2)):
        v = scan_inputs(rng, B, T, D, N, G, True)
        pos, Dv, kw = scan_own(v, cuda)
        y, saved = ops.selective_scan_fwd(*pos, Dv, softplus=True, lengths=lengths, save=True, **kw)
        grads = ops.selective_scan_bwd(*pos, pos[0], saved, Dv, softplus=True, lengths=lengths, **kw)
        for t in (y, grads[0], grads[1], grads[3], grads[4], grads[6]):
            t = to_host(t)
            assert (t[1] == 0).all() and (t[2, 41:] == 0).all() and (t[2, :41] != 0).any()
        kept = torch.full((B, T, D), 7.0, device=cuda)
        ops.selective_scan_fwd(*pos, Dv, softplus=True, lengths=lengths, out=kept, **kw)
        kept = to_host(kept)
        assert (kept[1] == 7).all() and (kept[2, 41:] == 7).all()
        np.testing.assert_array_equal(kept[2, :41], to_host(y)[2, :41])


def test_norm_of_four_axes(cuda):
    rng = np.random.default_rng(16)
    x = dev(rnd(rng, 3, 2, 5, 4, 12), cuda)[:, 1].permute(1, 0, 2, 3)  # axes that do not collapse
    w = dev(rnd(rng, 12), cuda)
    y = ops.rms_norm_fwd(x, w)
    np.testing.assert_array_equal(to_host(y), to_host(ops.rms_norm_fwd(x.contiguous(), w)))
    q, sc = ops.rms_norm_quant(x, w)
    q2, sc2 = ops.rms_norm_quant(x.contiguous(), w)
    np.testing.assert_array_equal(to_host(q.float()), to_host(q2.float()))
    np.testing.assert_array_equal(to_host(sc), to_host(sc2))
    assert sc.shape == (5, 3, 4, 1)


# ------------------------------------------- together, streams and graphs
def block(ops_in, p, state=None):
    """One residual block: norm, in-projection, conv, scan, out-projection."""
    x, res = ops_in
    y, s = ops.rms_norm_fwd(x, p["w"], residual=res)
    B, T, M = y.shape
    xz = ops.gemm(y.reshape(B * T, M), p["win"], precision="3xtf32").view(B, T, -1)
    D, N = p["A"].shape
    u, z = xz[..., :D], xz[..., D:2 * D]
    delta, Bm, C = xz[..., 2 * D:3 * D], xz[..., 3 * D:3 * D + N], xz[..., 3 * D + N:]
    cs, h = state if state is not None else (None, None)
    c, cs = ops.causal_conv_fwd(u, p["cw"], p["cb"], state=cs, silu=True, return_state=True)
    v, h = ops.selective_scan_fwd(c, delta, p["A"], Bm, C, p["D"], z=z, delta_bias=p["dtb"], softplus=True, h0=h,
                                  return_state=True)
    out = ops.gemm(v.reshape(B * T, D), p["wout"], precision="3xtf32").view(B, T, M)
    return out, s, (cs, h)


def block_step(x, res, p, state):
    y, s = ops.rms_norm_fwd(x, p["w"], residual=res)
    xz = ops.gemm(y, p["win"], precision="3xtf32")
    D, N = p["A"].shape
    c = ops.causal_conv_step(xz[:, :D], state[0], p["cw"], p["cb"], silu=True)
    v = ops.selective_scan_step(state[1], c, xz[:, 2 * D:3 * D], p["A"], xz[:, 3 * D:3 * D + N], xz[:, 3 * D + N:],
                                p["D"], z=xz[:, D:2 * D], delta_bias=p["dtb"], softplus=True)
    return ops.gemm(v, p["wout"], precision="3xtf32"), s


def block_params(rng, cuda, M=32, D=64, N=16):
    return {k: dev(a, cuda) for k, a in dict(
        w=rnd(rng, M) + 1, win=rnd(rng, M, 3 * D + 2 * N, scale=M ** -0.5), cw=rnd(rng, D, 4, scale=0.5), cb=rnd(rng, D),
        A=-np.exp(rnd(rng, D, N, scale=0.3)).astype(np.float32), D=rnd(rng, D), dtb=rnd(rng, D) - 2,
        wout=rnd(rng, D, M, scale=D ** -0.5)).items()}


def block_reference(x, res, p):
    p = {k: to_host(v).astype(np.float64) for k, v in p.items()}
    y, s = ref.rms_norm(x, p["w"], res, 1e-6)
    D, N = p["A"].shape
    xz = y @ p["win"]
    c, _ = ref.causal_conv(xz[..., :D], p["cw"], p["cb"], None, None, True)
    v, _ = ref.selective_scan(c, xz[..., 2 * D:3 * D], p["A"], xz[..., None, 3 * D:3 * D + N], xz[..., None, 3 * D + N:],
                              p["D"], xz[..., D:2 * D], p["dtb"], True, None, None)
    return v @ p["wout"], s


def test_block_prompt_then_tokens(cuda):
    """A prompt through the block, then its continuation token by token, gives
    what the whole sequence gives; both against the 64-bit block.  The GEMMs
    bound the tolerance: 3xTF32 products are within 1e-4 of the largest value."""
    rng = np.random.default_rng(21)
    p = block_params(rng, cuda)
    B, T, cut = 3, 24, 15
    x, res = rnd(rng, B, T, 32), rnd(rng, B, T, 32)
    want, s = block_reference(x, res, p)
    top = np.abs(want).max()
    xd, rd = dev(x, cuda), dev(res, cuda)
    out, total, _ = block((xd, rd), p)
    np.testing.assert_allclose(to_host(out), want, rtol=0, atol=5e-4 * top)
    np.testing.assert_array_equal(to_host(total), x + res)
    out, _, state = block((xd[:, :cut], rd[:, :cut]), p)
    np.testing.assert_allclose(to_host(out), want[:, :cut], rtol=0, atol=5e-4 * top)
    for t in range(cut, T):
        out, _ = block_step(xd[:, t], rd[:, t], p, state)
        np.testing.assert_allclose(to_host(out), want[:, t], rtol=0, atol=5e-4 * top)


def test_block_gradient_against_differences(cuda):
    """The block's loss gradient, assembled from the operators' gradients and
    GEMMs, against central differences of the 64-bit block: the operators'
    own error (1e-4 of the largest, the GEMMs') bounds the tolerance."""
    rng = np.random.default_rng(22)
    M, D, N = 8, 16, 4
    p = block_params(rng, cuda, M, D, N)
    B, T = 2, 20
    x, res, dout = rnd(rng, B, T, M), rnd(rng, B, T, M), rnd(rng, B, T, M)
    xd, rd, g = dev(x, cuda), dev(res, cuda), dev(dout, cuda)
    y, s = ops.rms_norm_fwd(xd, p["w"], residual=rd)
    xz = ops.gemm(y.reshape(-1, M), p["win"]).view(B, T, -1)
    u, z, delta = xz[..., :D], xz[..., D:2 * D], xz[..., 2 * D:3 * D]
    Bm, C = xz[..., 3 * D:3 * D + N], xz[..., 3 * D + N:]
    c = ops.causal_conv_fwd(u, p["cw"], p["cb"], silu=True)
    kw = dict(z=z, delta_bias=p["dtb"], softplus=True)
    v, saved = ops.selective_scan_fwd(c, delta, p["A"], Bm, C, p["D"], save=True, **kw)
    dv = ops.gemm(g.reshape(-1, M), p["wout"].t()).view(B, T, D)
    dc, ddelta, dA, dB, dC, dD, dz, dtb, _ = ops.selective_scan_bwd(c, delta, p["A"], Bm, C, dv, saved, p["D"], **kw)
    du, dcw, dcb, _ = ops.causal_conv_bwd(u, p["cw"], dc, p["cb"], silu=True)
    import torch

    dxz = torch.cat([du, dz, ddelta, dB, dC], dim=2)
    dyv = ops.gemm(dxz.reshape(B * T, -1), p["win"].t()).view(B, T, M)
    dx, dw = ops.rms_norm_bwd(s, p["w"], dyv)
    host = {k: to_host(a).astype(np.float64) for k, a in p.items()}

    def loss(xx, pp):
        yv, _ = ref.rms_norm(xx, pp["w"], res.astype(np.float64), 1e-6)
        q = yv @ pp["win"]
        cc, _ = ref.causal_conv(q[..., :D], pp["cw"], pp["cb"], None, None, True)
        vv, _ = ref.selective_scan(cc, q[..., 2 * D:3 * D], pp["A"], q[..., None, 3 * D:3 * D + N],
                                   q[..., None, 3 * D + N:], pp["D"], q[..., D:2 * D], pp["dtb"], True, None, None)
        return ((vv @ pp["wout"]) * dout).sum()

    x6 = x.astype(np.float64)
    for name, got, arr in (("x", dx, x6), ("w", dw, host["w"]), ("cw", dcw, host["cw"]), ("cb", dcb, host["cb"]),
                           ("A", dA, host["A"]), ("D", dD, host["D"]), ("dtb", dtb, host["dtb"])):
        got = to_host(got).astype(np.float64)
        top = np.abs(got).max()
        idx = [np.unravel_index(int(i), arr.shape) for i in rng.integers(0, arr.size, 6)]
        for i in idx:
            keep = arr[i]
            arr[i] = keep + 1e-5
            hi = loss(x6, host)
            arr[i] = keep - 1e-5
            lo = loss(x6, host)
            arr[i] = keep
            assert abs((hi - lo) / 2e-5 - got[i]) <= 1e-3 * top, (name, i)


def test_calls_on_another_stream_and_in_graphs(cuda):
    """The same bits eagerly, on a side stream, and from two captured graphs
    replayed at once with other inputs in their buffers."""
    import torch

    rng = np.random.default_rng(31)
    p = block_params(rng, cuda)
    xs = [dev(rnd(rng, 2, 200, 32), cuda) for _ in range(2)]
    rs = [dev(rnd(rng, 2, 200, 32), cuda) for _ in range(2)]

    def train(x, r):
        y, s = ops.rms_norm_fwd(x, p["w"], residual=r)
        wide = torch.cat([y, y], dim=2)  # 64 channels
        c = ops.causal_conv_fwd(wide, p["cw"], p["cb"], silu=True)
        bc = wide[..., :16]
        v, last, saved = ops.selective_scan_fwd(c, wide, p["A"], bc, bc, p["D"], softplus=True, return_state=True, save=True)
        grads = ops.selective_scan_bwd(c, wide, p["A"], bc, bc, v, saved, p["D"], softplus=True, dh_last=last)
        du, dw, db, _ = ops.causal_conv_bwd(wide, p["cw"], grads[0], p["cb"], silu=True)
        dx, dnw = ops.rms_norm_bwd(s, p["w"], du[..., :32].contiguous(), dsum=y)
        q, sc, _ = ops.rms_norm_quant(x, p["w"], residual=r, group=32)
        return [v, last, *(t for t in grads if t is not None), du, dw, db, dx, dnw, q.float(), sc]

    want = [[to_host(t) for t in train(x, r)] for x, r in zip(xs, rs)]
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        got = train(xs[0], rs[0])
    side.synchronize()
    for a, b in zip(got, want[0]):
        np.testing.assert_array_equal(to_host(a), b)
    bufs = [(torch.zeros_like(x), torch.zeros_like(r)) for x, r in zip(xs, rs)]
    graphs, outs = [], []
    for b in bufs:
        with torch.cuda.stream(side):
            train(*b)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(train(*b))
        graphs.append(g)
    for order in ((0, 1), (1, 0)):
        for k in (0, 1):
            bufs[k][0].copy_(xs[order[k]])
            bufs[k][1].copy_(rs[order[k]])
        torch.cuda.synchronize(cuda)
        streams = [torch.cuda.Stream(cuda) for _ in graphs]
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize(cuda)
        for k in (0, 1):
            for a, b in zip(outs[k], want[order[k]]):
                np.testing.assert_array_equal(to_host(a), b)
    del graphs


def test_python_refusals(cuda):
    import torch

    x, w = torch.zeros((2, 4), device=cuda), torch.ones(4, device=cuda)
    with pytest.raises(RemoraUnsupportedError):
        ops.rms_norm_fwd(x.half(), w)
    with pytest.raises(RemoraUnsupportedError):
        ops.rms_norm_quant(x, w, out=torch.zeros((2, 4), device=cuda, dtype=torch.uint8))
    with pytest.raises(RemoraUnsupportedError):
        ops.causal_conv_fwd(torch.zeros((1, 3, 4), device=cuda), torch.zeros((4, 3), device=cuda),
                            lengths=torch.tensor([3], device=cuda))  # int64
    with pytest.raises(RemoraB200Error):
        ops.rms_norm_fwd(x, torch.ones(4))
    with pytest.raises(RemoraShapeError):
        ops.rms_norm_fwd(x, w, residual=torch.zeros((3, 4), device=cuda))
    with pytest.raises(RemoraB200Error):
        ops.rms_norm_fwd(x, w, sum_out=x)
    y = torch.zeros((1, 3, 4), device=cuda)
    with pytest.raises(RemoraShapeError):
        ops.causal_conv_fwd(y[0], torch.zeros((4, 3), device=cuda))
    with pytest.raises(RemoraShapeError):
        ops.selective_scan_fwd(y, y, torch.zeros((4, 5), device=cuda), torch.zeros((1, 3, 5), device=cuda),
                               torch.zeros((1, 3, 1, 5), device=cuda))
    with pytest.raises(RemoraB200Error):
        ops.causal_conv_fwd(y, torch.zeros((4, 3), device=cuda), out=y)
    with pytest.raises(RemoraUnsupportedError):
        ops.selective_scan_fwd(y, y, torch.zeros((4, 65), device=cuda), torch.zeros((1, 3, 65), device=cuda),
                               torch.zeros((1, 3, 65), device=cuda))


def test_no_memory_for_a_result(cuda):
    """What torch raises, before any launch."""
    import torch

    row = torch.ones(1, 1 << 20, device=cuda)
    with pytest.raises(torch.OutOfMemoryError):
        ops.rms_norm_fwd(row.expand(1 << 22, -1), row[0])  # 16 TiB
    np.testing.assert_array_equal(to_host(ops.rms_norm_fwd(row, row[0], eps=0.0)), to_host(row))


def test_calls_from_two_threads(cuda):
    """Each on a stream of its own: the results of one thread alone, bit for bit."""
    import threading

    import torch

    rng = np.random.default_rng(77)
    v = [scan_inputs(rng, 2, 150, 70, 16, 1, True) for _ in range(2)]
    given = [scan_own(x, cuda) for x in v]

    def train(i):
        pos, Dv, kw = given[i]
        y, saved = ops.selective_scan_fwd(*pos, Dv, softplus=True, save=True, **kw)
        grads = ops.selective_scan_bwd(*pos, y, saved, Dv, softplus=True, **kw)
        n, q = ops.rms_norm_fwd(y, Dv), ops.causal_conv_fwd(y, pos[2][:, :4], Dv, silu=True)
        return [y, n, q, *grads]

    alone = [train(i) for i in range(2)]
    torch.cuda.synchronize()
    seen, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    seen[i].append(train(i))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for want, runs in zip(alone, seen):
        for got in runs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("N,T", [(64, 140), (16, 40), (8, 140)])
def test_scan_captured_and_replayed(cuda, N, T):
    """With new inputs in the captured call's tensors."""
    import torch

    rng = np.random.default_rng(N + T)
    v = scan_inputs(rng, 2, T, 40, N, 1, True)
    pos, Dv, kw = scan_own(v, cuda)

    def train():
        y, saved = ops.selective_scan_fwd(*pos, Dv, softplus=True, save=True, **kw)
        return [y, *ops.selective_scan_bwd(*pos, y, saved, Dv, softplus=True, **kw)]

    train()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = train()
    for _ in range(2):
        pos[0].copy_(dev(rnd(rng, 2, T, 40), cuda))
        pos[3].copy_(dev(rnd(rng, 2, T, 1, N), cuda))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, train()))
