"""Sequence operators on the GPU at the edges of what their calls allow: values
next to a rounding's border, the ends of the f32 range, layouts and sizes that
other kernels take, against 64-bit definitions (tests/seq_reference.py)."""

from __future__ import annotations

import numpy as np
import pytest

import seq_reference as ref
import test_gpu_seq as base
from conftest import to_host
from remora_b200 import ops
from test_gpu_seq import E, dev, norm_tol, rnd, within

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- norm
@pytest.mark.parametrize("rows,D,group", [(8192, 4096, 128), (4096, 4096, 0), (4000, 1001, 0), (60, 20000, 32),
                                          (60, 20000, 0)])
def test_quant_is_the_quotient_rounded(cuda, rows, D, group):
    """q is the f32 quotient of rms_norm_fwd's y and the scale, rounded to e4m3,
    in every element: the same rows give the same y, and numpy's division is
    IEEE's."""
    import torch

    rng = np.random.default_rng(rows + D + group)
    x, w = dev(rnd(rng, rows, D), cuda), dev(rnd(rng, D), cuda)
    y = to_host(ops.rms_norm_fwd(x, w)).reshape(rows, -1, group or D)
    q, scales = ops.rms_norm_quant(x, w, group=group)
    scales = to_host(scales).reshape(rows, -1, 1)
    np.testing.assert_array_equal(scales, np.maximum(np.abs(y).max(axis=2, keepdims=True) / np.float32(448),
                                                     np.float32(2.0 ** -126)))
    want = torch.from_numpy(y / scales).to(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(to_host(q.float()).reshape(want.shape), want)


@pytest.mark.parametrize("rows,D", [(5, 77), (700, 32), (700, 300), (700, 1001), (3, 8191), (700, 8191), (1, 1)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_of_operands_aligned_differently(cuda, rows, D, residual):
    """Rows whose starts lie differently on 16-byte boundaries are read by single
    elements, one to eight (backward sixteen) per thread."""
    rng = np.random.default_rng(rows + D)
    x, w, dy = rnd(rng, rows, D), rnd(rng, D), rnd(rng, rows, D)
    r = rnd(rng, rows, D) if residual else None
    beside = lambda a: dev(np.concatenate([a[:, :1], a], axis=1), cuda)[:, 1:]  # noqa: E731  (rows D + 1 apart)
    xd, wd, rd = beside(x), dev(w, cuda), dev(r, cuda)
    y, s = ref.rms_norm(x, w, r, 1e-5)
    tol = np.abs(y) * (norm_tol(D) + E) + np.abs(w) * np.abs(y / np.where(w == 0, 1, w)) * E
    got = ops.rms_norm_fwd(xd, wd, residual=rd, eps=1e-5)
    if residual:
        got, total = got
        np.testing.assert_array_equal(to_host(total), x + r)
    within(got, y, tol, "y")
    q, scales, *_ = ops.rms_norm_quant(xd, wd, residual=rd, eps=1e-5)
    want = np.maximum(np.abs(y).max(axis=1, keepdims=True) / 448, 2.0 ** -126)
    within(scales, want, want * (norm_tol(D) + 4 * E), "scales")
    # to a level off by half its distance: 2^-4 of the value, or 2^-10 of the scale below 2^-6
    within(to_host(q.float()) * to_host(scales).astype(np.float64), y, np.abs(y) * 2.0 ** -4 * (1 + 1e-5) + want * 2.0 ** -10)
    s32 = x if r is None else x + r
    rx, rw = ref.rms_norm_bwd(s32, w, dy, dy, 1e-5)
    s6 = s32.astype(np.float64)
    rstd = 1 / np.sqrt((s6 * s6).mean(axis=1, keepdims=True) + 1e-5)
    mean = np.abs(s6 * rstd * w * dy).mean(axis=1, keepdims=True)
    mag = rstd * (np.abs(w * dy) + np.abs(s6 * rstd) * mean) + np.abs(dy)
    wmag = np.abs(dy * s6 * rstd).sum(axis=0) * (norm_tol(D) + rows * E + 8 * E)
    sd, gd = beside(s32), dev(dy, cuda)
    for out in (None, sd):
        dx, dw = ops.rms_norm_bwd(sd, wd, gd, dsum=gd, eps=1e-5, out=out)
        within(dx, rx, mag * 4 * norm_tol(D), "dx")
        within(dw, rw, wmag, "dw")
    assert dx is sd


@pytest.mark.parametrize("rows,D", [(700, 256), (700, 4096), (3, 4096)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("residual", [False, True])
def test_groups_over_several_vectors_of_a_thread(cuda, rows, D, group, residual):
    base.test_norm_quant(cuda, rows, D, group, residual)


# ------------------------------------------------------------------- silu
def test_silu_far_from_zero(cuda):
    """v / (1 + exp(-v)) within 6 + |v| units (E) of the sigmoid, where exp(-v)
    counts beside 1, and one of each product.  Below -87 the sigmoid is less than
    the least normal number, and may be 0.  silu' = s (1 + v (1 - s)) carries the
    sigmoid's error |v| times."""
    v = np.concatenate([np.linspace(-87, 88, 3000), [-1e30, -200, -120, -100, -90, -88, 120, 1e30]]).astype(np.float32)
    want = v.astype(np.float64) * ref.sigmoid(v.astype(np.float64))
    units = (10 + np.minimum(np.abs(v.astype(np.float64)), 88) * (v < 17)) * E  # exp(-17) is below E
    bound = np.abs(want) * units + np.where(v < -87, np.minimum(np.abs(want), np.abs(v.astype(np.float64)) * 2.0 ** -126), 0)
    n = len(v)
    x, w = dev(v.reshape(1, 1, n), cuda), dev(np.tile(np.float32([0, 1]), (n, 1)), cuda)
    one = dev(np.ones((1, 1, n), np.float32), cuda)
    within(ops.causal_conv_fwd(x, w, silu=True)[0, 0], want, bound, "conv")
    state = dev(np.zeros((1, 1, n), np.float32), cuda)
    within(ops.causal_conv_step(x[0], state, w, silu=True)[0], want, bound, "conv step")
    s = ref.sigmoid(v.astype(np.float64))
    slope = s * (1 + v * (1 - s))
    tiny = np.where(v < -87, np.abs(slope), 0)
    steep = np.minimum(np.abs(v.astype(np.float64)), 200)  # behind it s is 0 or 1
    within(ops.causal_conv_bwd(x, w, one, silu=True)[0][0, 0], slope, s * (1 + steep) * units + tiny, "conv gradient")
    zero = dev(np.zeros((1, 1, 4), np.float32), cuda)
    A, D = dev(-np.ones((n, 4), np.float32), cuda), dev(np.ones(n, np.float32), cuda)
    within(ops.selective_scan_fwd(one, one, A, zero, zero, D, z=x)[0, 0], want, bound, "scan")
    h = dev(np.zeros((1, n, 4), np.float32), cuda)
    within(ops.selective_scan_step(h, one[0], one[0], A, zero[0], zero[0], D, z=x[0])[0], want, bound, "scan step")


# ------------------------------------------------------------------- scan
BIG = [2.3e38, 2.5e38, 3.2e38, 3.4e38]


@pytest.mark.parametrize("length", [1, 5, 200])
def test_softplus_of_the_largest_steps(cuda, length):
    """softplus(v) is v, and its slope 1, at the top of the f32 range; both are 0
    at the bottom.  In the long axis, which is cut, such steps stand apart."""
    D, N = len(BIG), 4
    delta = np.full((2, length, D), -4.0, np.float32)
    delta[0, -1], delta[1, -1] = BIG, [-v for v in BIG]
    u = np.full(delta.shape, 1e-30, np.float32)
    A, B, C = -np.ones((D, N), np.float32), np.ones((2, length, N), np.float32), np.full((2, length, N), 0.125, np.float32)
    h0, dy = np.ones((2, D, N), np.float32), np.zeros_like(delta)
    dy[:, -1] = 1
    d = lambda v: dev(v, cuda)  # noqa: E731
    args = d(u), d(delta), d(A), d(B), d(C)
    y, last, saved = ops.selective_scan_fwd(*args, softplus=True, h0=d(h0), return_state=True, save=True)
    du, ddelta, dA, *_ = ops.selective_scan_bwd(*args, d(dy), saved, softplus=True, h0=d(h0))
    s, few = np.array(BIG, np.float32), 16 * 2.0 ** -24
    # nothing is left of the state ahead of the first row's last step, all of it in the other
    np.testing.assert_allclose(to_host(last)[0, :, 0], s * u[0, 0, 0], rtol=few)
    np.testing.assert_allclose(to_host(y)[0, -1], s * u[0, 0, 0] / 2, rtol=few)
    np.testing.assert_allclose(to_host(du)[0, -1], s / 2, rtol=few)
    np.testing.assert_allclose(to_host(ddelta)[0, -1], u[0, 0] / 2, rtol=few)
    decay = np.exp(-np.logaddexp(-4.0, 0) * (length - 1))
    np.testing.assert_allclose(to_host(y)[1, -1], decay / 2, rtol=6 * length * 2.0 ** -24 + few)
    assert (to_host(du)[1, -1] == 0).all() and (to_host(ddelta)[1, -1] == 0).all()
    assert np.isfinite(to_host(dA)).all()
    y = ops.selective_scan_step(d(h0), d(u[:, -1]), d(delta[:, -1]), d(A), d(B[:, -1]), d(C[:, -1]), softplus=True)
    np.testing.assert_allclose(to_host(y)[0], s * u[0, 0, 0] / 2, rtol=few)
    np.testing.assert_allclose(to_host(y)[1], 0.5, rtol=few)


@pytest.mark.parametrize("N", [1, 4, 5, 13, 16, 33, 64])
@pytest.mark.parametrize("length,at", [(9, 6), (300, 170)])
def test_an_infinite_step_leaves_what_is_ahead_of_it(cuda, N, length, at):
    """A step that is inf forgets the state, whatever the number of states: ahead of
    it everything is as in the sequence cut there, in both directions, and from it
    on the states of positive inputs are +inf."""
    rng = np.random.default_rng(N + length)
    D = 6
    pos = lambda *shape: rng.uniform(0.5, 1.5, shape).astype(np.float32)  # noqa: E731
    u, delta, B, C = pos(1, length, D), rnd(rng, 1, length, D) - 3, pos(1, length, N), pos(1, length, N)
    A, h0, dy = -pos(D, N), pos(1, D, N), rnd(rng, 1, length, D)
    delta[:, at], dy[:, at:] = np.inf, 0
    d = lambda v: dev(v, cuda)  # noqa: E731
    args = [d(v) for v in (u, delta, A, B, C)]
    cut = d(np.array([at], np.int32))
    outs, grads = [], []
    for lengths in (None, cut):
        y, saved = ops.selective_scan_fwd(*args, softplus=True, h0=d(h0), lengths=lengths, save=True)
        g = ops.selective_scan_bwd(*args, d(dy), saved, softplus=True, h0=d(h0), lengths=lengths)
        outs.append(to_host(y))
        grads.append([to_host(g[k])[:, :at] if k < 8 else to_host(g[k]) for k in (0, 1, 3, 4, 8)])
    np.testing.assert_array_equal(outs[0][:, :at], outs[1][:, :at])
    assert np.isfinite(outs[1]).all() and (outs[0][:, at:] == np.inf).all()
    for a, b in zip(*grads):
        assert np.isfinite(b).all()
        np.testing.assert_array_equal(a, b)
    y = ops.selective_scan_step(d(h0), *(d(v[:, at]) for v in (u, delta)), d(A), d(B[:, at]), d(C[:, at]), softplus=True)
    assert (to_host(y) == np.inf).all()


@pytest.mark.parametrize("N", [1, 4, 5, 13, 16, 33])
@pytest.mark.parametrize("T", [7, 300])
def test_large_steps_of_either_sign(cuda, N, T):
    """Without softplus a step may be negative and large, where the rates are small:
    the decay is e^2 at most here."""
    rng = np.random.default_rng(N + T)
    D, tol = 6, (6 * T + 64) * E
    delta = (rnd(rng, 2, T, D) * np.float32(0.01)).astype(np.float32)
    delta[0, T // 2], delta[1, T // 3] = -200, 200
    v = dict(u=rnd(rng, 2, T, D), delta=delta, A=-rng.uniform(0.001, 0.01, (D, N)).astype(np.float32), B=rnd(rng, 2, T, 1, N),
             C=rnd(rng, 2, T, 1, N), D=None, z=None, bias=None, h0=rnd(rng, 2, D, N))
    dy = rnd(rng, 2, T, D)
    pos, Dv, kw = base.scan_own(v, cuda)
    y, last, saved = ops.selective_scan_fwd(*pos, Dv, return_state=True, save=True, **kw)
    args = (*(v[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), False, v["h0"], None)
    for got, want, mag in zip((y, last), ref.selective_scan(*args), ref.selective_scan(*args, absolute=True)):
        within(got, want, mag * tol)
    got = ops.selective_scan_bwd(*pos, dev(dy, cuda), saved, Dv, **kw)
    want, mag = (ref.selective_scan_bwd(*args, dy, None, absolute=a) for a in (False, True))
    for name, g in zip(base.NAMES, got):
        if g is not None:
            extra = {"dA": 2 * T, "dB": D, "dC": D}.get(name, 0)
            within(g, want[name], mag[name] * (2 * tol + extra * E), name)
    for row, t in ((0, T // 2), (1, T // 3)):
        one = [dev(v[k][row:row + 1, t], cuda) for k in ("u", "delta", "B", "C")]
        y = ops.selective_scan_step(dev(v["h0"][row:row + 1], cuda), *one[:2], pos[2], *one[2:])
        cut = tuple(a if k in (2, 5, 6, 7, 8, 9, 10) else a[:, t:t + 1] for k, a in enumerate(args))
        within(y[0], ref.selective_scan(*cut)[0][row, 0], ref.selective_scan(*cut, absolute=True)[0][row, 0] * 70 * E)


@pytest.mark.parametrize("N", [3, 8, 13, 16, 33, 64])
@pytest.mark.parametrize("full", [False, True])
def test_long_axes_that_are_not_cut(cuda, N, full):
    """444 blocks of channels (here: groups) and more leave the time axis whole in
    both directions, however long it is."""
    base.test_scan_forward_backward(cuda, 3, 400, 148, N, 148, full)


@pytest.mark.parametrize("B,T,D,N", [(300, 5, 3, 13), (260, 3, 10, 64), (30, 300, 3, 4), (30, 300, 40, 33)])
def test_sums_over_many_pieces(cuda, B, T, D, N):
    """More than 256 rows of partial sums of da, dd and ddelta_bias: a batch of more
    sequences than that, or nine pieces of each of 30; one channel block or two."""
    base.test_scan_forward_backward(cuda, B, T, D, N, 1, True)


# ------------------------------------------------------------------ results
def test_in_place_results_leave_a_lazy_clone_alone(cuda):
    import torch

    rng = np.random.default_rng(0)
    x, w, state = dev(rnd(rng, 3, 8), cuda), dev(rnd(rng, 8, 4), cuda), dev(rnd(rng, 3, 3, 8), cuda)
    before, mine = to_host(state), torch._lazy_clone(state)
    ops.causal_conv_step(x, mine, w)
    np.testing.assert_array_equal(to_host(mine)[:, -1], to_host(x))
    np.testing.assert_array_equal(to_host(state), before)
    y, copy = torch._lazy_clone(x), to_host(x)
    ops.rms_norm_fwd(y, dev(np.ones(8, np.float32), cuda), out=y)
    np.testing.assert_array_equal(to_host(x), copy)
    assert (to_host(y) != copy).any()


def test_given_results_count_as_modified(cuda):
    """A value that autograd keeps is not replaced unnoticed."""
    import torch

    rng = np.random.default_rng(1)
    t = lambda *shape: dev(rnd(rng, *shape), cuda)  # noqa: E731
    x, w, state, pool = t(3, 8), t(8, 4), t(3, 3, 8), t(3, 8, 4)
    seq, ones, total = t(3, 5, 8), torch.ones(8, device=cuda), t(3, 8)
    calls = [(lambda o: ops.rms_norm_fwd(x, ones, out=o), x),
             (lambda o: ops.rms_norm_fwd(x, ones, residual=total, sum_out=o), total),
             (lambda o: ops.rms_norm_bwd(x, ones, total, out=o), total),
             (lambda o: ops.causal_conv_fwd(seq, w, state=o, state_out=o), state),
             (lambda o: ops.causal_conv_bwd(seq, w, seq, out=o), t(3, 5, 8)),
             (lambda o: ops.causal_conv_step(x, o, w), state),
             (lambda o: ops.selective_scan_step(o, x, x, -pool[0].abs(), pool[:, 0], pool[:, 1]), pool.clone())]
    for call, out in calls:
        leaf = torch.ones_like(out, requires_grad=True)
        kept = leaf * out  # keeps `out` for its gradient
        call(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.sum().backward()
    with torch.inference_mode():
        ops.causal_conv_step(x.clone(), state.clone(), w)


# ------------------------------------------------------------------ strides
@pytest.mark.parametrize("N", [4, 16])
def test_few_channels_far_apart(cuda, N):
    """Three channels 2^28 elements from one another, upwards and (by descriptors
    alone) downwards, time likewise."""
    import ctypes

    import torch

    from remora_b200 import _lib as L
    from remora_b200.abi import make_memref_descriptor, tensor_descriptor
    from remora_b200.runtime import context

    rng = np.random.default_rng(N)
    T, D, far = 21, 3, 1 << 28
    buf = torch.empty((D - 1) * far + 2 * T, dtype=torch.float32, device=cuda)
    wide, out = (buf.as_strided((1, T, D), (0, 1, far), at) for at in (0, T))
    u, dy = dev(rnd(rng, 1, T, D), cuda), dev(rnd(rng, 1, T, D), cuda)
    A, b, c = dev(-np.abs(rnd(rng, D, N)), cuda), dev(rnd(rng, 1, T, N), cuda), dev(rnd(rng, 1, T, N), cuda)
    wide.copy_(u)
    want, saved = ops.selective_scan_fwd(u, u, A, b, c, z=u, softplus=True, save=True)
    got, kept = ops.selective_scan_fwd(wide, wide, A, b, c, z=wide, softplus=True, save=True, out=out)
    np.testing.assert_array_equal(to_host(got), to_host(want))
    for g, r in zip(ops.selective_scan_bwd(wide, wide, A, b, c, dy, kept, z=wide, softplus=True),
                    ops.selective_scan_bwd(u, u, A, b, c, dy, saved, z=u, softplus=True)):
        if g is not None:
            np.testing.assert_array_equal(to_host(g), to_host(r))
    turned = u.flip(1, 2).contiguous()
    want = ops.selective_scan_fwd(turned, turned, A, b, c, softplus=True)
    back = make_memref_descriptor(buf.data_ptr(), (1, T, D), (0, -1, -far), offset=T - 1 + (D - 1) * far)
    y = torch.empty_like(u)
    descs = [tensor_descriptor(t) for t in (A, b.unsqueeze(2), c.unsqueeze(2))]
    args = L.RemoraSelectiveScanIn(ctypes.addressof(back), ctypes.addressof(back), *(ctypes.addressof(x) for x in descs))
    spec, to = L.RemoraSelectiveScanSpec(1, 0), tensor_descriptor(y)
    stream = ctypes.c_void_p(torch.cuda.current_stream(cuda).cuda_stream)
    L.check(L.lib().remora_b200_selective_scan_fwd(context(0).ptr, ctypes.addressof(spec), ctypes.addressof(args),
                                                   ctypes.addressof(to), None, None, 0, None, 0, stream))
    np.testing.assert_array_equal(to_host(y), to_host(want))
    del buf


# ----------------------------------------------------------------- refusals
def test_operands_that_are_missing_or_no_tensors_are_refused(cuda):
    """Every operand that a call needs, left out or of another type, and weights
    without taps: the framework's own errors, before anything is launched."""
    import torch

    from remora_b200 import _lib as L
    from remora_b200.errors import RemoraB200Error

    t = lambda *shape: torch.zeros(shape, device=cuda)  # noqa: E731
    y, saved = ops.selective_scan_fwd(t(2, 5, 8), t(2, 5, 8), t(8, 4), t(2, 5, 4), t(2, 5, 4), save=True)
    scan = dict(u=t(2, 5, 8), delta=t(2, 5, 8), A=t(8, 4), B=t(2, 5, 4), C=t(2, 5, 4))
    step = dict(state=t(2, 8, 4), u=t(2, 8), delta=t(2, 8), A=t(8, 4), B=t(2, 4), C=t(2, 4))
    calls = [(ops.rms_norm_fwd, dict(x=t(2, 8), w=t(8))), (ops.rms_norm_quant, dict(x=t(2, 8), w=t(8))),
             (ops.rms_norm_bwd, dict(s=t(2, 8), w=t(8), dy=t(2, 8))),
             (ops.causal_conv_fwd, dict(x=t(2, 5, 8), w=t(8, 3))),
             (lambda **k: ops.causal_conv_fwd(**k, return_state=True), dict(x=t(2, 5, 8), w=t(8, 3))),
             (ops.causal_conv_bwd, dict(x=t(2, 5, 8), w=t(8, 3), dy=t(2, 5, 8))),
             (ops.causal_conv_step, dict(x=t(2, 8), state=t(2, 2, 8), w=t(8, 3))),
             (ops.selective_scan_fwd, scan), (lambda **k: ops.selective_scan_fwd(**k, return_state=True), scan),
             (ops.selective_scan_bwd, dict(scan, dy=t(2, 5, 8), saved=saved)), (ops.selective_scan_step, step)]
    before = L.launch_count()
    for call, good in calls:
        for name in good:
            for bad in (None, 3.0, [1.0], t(), t(3).cpu()):
                with pytest.raises(RemoraB200Error):
                    call(**{**good, name: bad})
        if "w" in good and good["w"].dim() == 2:
            with pytest.raises(RemoraB200Error):
                call(**{**good, "w": t(8, 0)})
    assert L.launch_count() == before
