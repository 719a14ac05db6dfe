"""Sequence operators without a GPU: calls that the entry points have to refuse, or
to take, and the host's side of a call.  The C entry points check every argument
before any CUDA call."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from remora_b200 import _lib as L
from test_seq_host import BASE, FAKE, desc

FAR = [BASE + (k << 24) for k in range(32)]
KEPT: list = []


def ad(d):
    """A descriptor's address; the descriptor lives as long as the tests."""
    KEPT.append(d)
    return ctypes.addressof(d) if d is not None else None


# what a call that is refused for want of memory answers: every other check is behind it
LAST = L.ERR_LIMIT


def device_present() -> bool:
    import torch

    return torch.cuda.is_available()


def scan_fwd(y, h_last=None, saved=(BASE, 8), scratch=(None, 0), **members):
    """A call whose last refusal is that of its eight bytes of saved states."""
    m = {**dict.fromkeys(("u", "delta", "a", "b", "c", "d", "z", "delta_bias", "h0", "lengths")), **members}
    args, spec = L.RemoraSelectiveScanIn(*(ad(v) for v in m.values())), L.RemoraSelectiveScanSpec(1, 0)
    return L.lib().remora_b200_selective_scan_fwd(FAKE, ctypes.addressof(spec), ctypes.addressof(args), ad(y),
                                                  ad(h_last), *saved, *scratch, None)


def scan_operands(B, T, D, N):
    return dict(u=desc(B, T, D, at=FAR[0]), delta=desc(B, T, D, at=FAR[1]), a=desc(D, N, at=FAR[2]),
                b=desc(B, T, 1, N, at=FAR[3]), c=desc(B, T, 1, N, at=FAR[4]))


# ------------------------------------------------------------------ overlap
def test_each_output_may_lie_over_its_own_inputs_only():
    """The state behind the sequences may replace the one ahead of them; y may
    not, not even where the two have the same shape.  The gradient of a single
    row's weights is no gradient in place of its input."""
    n = 16
    m, h0 = scan_operands(2, n, n, n), desc(2, n, n, at=FAR[5])
    y, other = desc(2, n, n, at=FAR[6]), desc(2, n, n, at=FAR[7])
    assert scan_fwd(y, h0, h0=h0, **m) == LAST
    assert scan_fwd(y, other, h0=h0, **m) == LAST
    assert scan_fwd(h0, other, h0=h0, **m) == L.ERR_ARG
    assert scan_fwd(h0, None, h0=h0, **m) == L.ERR_ARG
    spec = L.RemoraNormSpec(1e-6, 0)
    s, w, dy, dx, dw = (desc(8, at=FAR[k]) for k in range(5))
    bwd = lambda dx, dw: L.lib().remora_b200_rms_norm_bwd(  # noqa: E731
        FAKE, ctypes.addressof(spec), ad(s), ad(w), ad(dy), None, ad(dx), ad(dw), 1, None, 0, None)
    assert bwd(dx, dw) == LAST and bwd(s, dw) == LAST and bwd(dy, dw) == LAST
    assert bwd(dx, s) == L.ERR_ARG and bwd(dx, dy) == L.ERR_ARG
    x, q, scales, r = desc(4, 1, at=FAR[0]), desc(4, 1, at=FAR[1]), desc(4, 1, at=FAR[2]), desc(4, 1, at=FAR[3])
    quant = lambda scales, s: L.lib().remora_b200_rms_norm_quant(  # noqa: E731
        FAKE, ctypes.addressof(spec), ad(x), ad(r), ad(desc(1, at=FAR[4])), ad(q), ad(scales), ad(s), 2, None)
    assert quant(x, None) == L.ERR_ARG and quant(r, None) == L.ERR_ARG and quant(scales, scales) == L.ERR_ARG


def conv_bwd(shape, dx):
    """A backward of the convolution without scratch, which is refused last."""
    B, T, D = shape
    x, w, dy = desc(B, T, D, at=1 << 48), desc(D, 3, at=FAR[1]), desc(B, T, D, at=1 << 49)
    spec, dw = L.RemoraCausalConvSpec(1, 0), desc(D, 3, at=FAR[3])
    return L.lib().remora_b200_causal_conv_bwd(FAKE, ctypes.addressof(spec), ad(x), ad(w), None, None, None, ad(dy), None,
                                               ad(dx), ad(dw), None, None, None, 0, None)


def test_outputs_whose_elements_share_addresses_are_refused():
    """Against enumeration: random small views as dx of a convolution's backward."""
    rng = np.random.default_rng(1)
    seen = {False: 0, True: 0}
    for _ in range(600):
        shape = [int(rng.integers(1, 5)) for _ in range(3)]
        strides = [int(rng.choice([-1, 1])) * int(rng.integers(0, 25)) for _ in range(3)]
        cells = sum(strides[k] * np.arange(shape[k]).reshape([-1 if j == k else 1 for j in range(3)]) for k in range(3))
        shared = len(np.unique(cells)) < cells.size
        st = conv_bwd(shape, desc(*shape, at=FAR[5], strides=strides))
        assert st == (L.ERR_ARG if shared else LAST), (shape, strides, L.last_error())
        seen[shared] += 1
    assert min(seen.values()) > 100
    # large views are decided without trying their elements
    n = 1 << 10
    for strides, shared in (((n * n, n, 1), False), ((1, n, n * n), False), ((n * n - 1, n, 1), True),
                            ((n * n, n - 1, 1), True), ((2 * n * n, 2 * n, 2), False)):
        assert conv_bwd((n, n, n), desc(n, n, n, at=1 << 44, strides=list(strides))) == (L.ERR_ARG if shared else LAST)


def test_every_entry_point_refuses_such_outputs():
    """Strides 1 and 1 over the last two axes, one output at a time."""
    def own(*shape):
        return desc(*shape, at=FAR[20], strides=[*([1000] * (len(shape) - 2)), 1, 1])

    m = scan_operands(2, 5, 4, 3)
    assert scan_fwd(own(2, 5, 4), **m) == L.ERR_ARG
    assert scan_fwd(desc(2, 5, 4, at=FAR[6]), own(2, 4, 3), **m) == L.ERR_ARG
    shapes = [(2, 5, 4), (2, 5, 4), (4, 3), (2, 5, 1, 3), (2, 5, 1, 3), (4,), (2, 5, 4), (4,), (2, 4, 3)]
    args = L.RemoraSelectiveScanIn(*(ad(m.get(k)) for k, _ in L.RemoraSelectiveScanIn._fields_))
    args.z = ad(desc(2, 5, 4, at=FAR[7]))
    spec = L.RemoraSelectiveScanSpec(1, 0)
    for bad in (None, 0, 1, 2, 6, 8):
        outs = [own(*s) if k == bad else desc(*s, at=FAR[10 + k]) for k, s in enumerate(shapes)]
        grads = L.RemoraSelectiveScanGrads(*(ad(v) for v in outs))
        st = L.lib().remora_b200_selective_scan_bwd(FAKE, ctypes.addressof(spec), ctypes.addressof(args),
                                                    ad(desc(2, 5, 4, at=FAR[8])), None, None, 0, ctypes.addressof(grads),
                                                    None, 0, None)
        assert st == (LAST if bad is None else L.ERR_ARG), L.last_error()
    # the calls below have no later refusal: without these they would be launched
    if device_present():
        return
    x, w, y = desc(4, 8, at=FAR[0]), desc(8, at=FAR[1]), desc(4, 8, at=FAR[2])
    norm = L.RemoraNormSpec(1e-6, 0)
    lib, at = L.lib(), ctypes.addressof
    r, other = desc(4, 8, at=FAR[3]), desc(4, 8, at=FAR[4])
    for out, s in ((own(4, 8), other), (y, own(4, 8))):
        assert lib.remora_b200_rms_norm_fwd(FAKE, at(norm), ad(x), ad(r), ad(w), ad(out), ad(s), 2, None) == L.ERR_ARG
        q = lib.remora_b200_rms_norm_quant(FAKE, at(norm), ad(x), ad(r), ad(w), ad(out), ad(desc(4, 1, at=FAR[6])), ad(s), 2, None)
        assert q == L.ERR_ARG
    assert lib.remora_b200_rms_norm_bwd(FAKE, at(norm), ad(x), ad(w), ad(y), None, ad(own(4, 8)), ad(desc(8, at=FAR[5])),
                                        2, FAR[9], 1 << 20, None) == L.ERR_ARG
    conv, taps, state = L.RemoraCausalConvSpec(1, 0), desc(8, 3, at=FAR[7]), desc(4, 2, 8, at=FAR[8])
    for out, s in ((own(4, 8), state), (y, own(4, 2, 8))):
        st = lib.remora_b200_causal_conv_step(FAKE, at(conv), ad(x), ad(state), ad(taps), None, None, ad(out), ad(s), None)
        assert st == L.ERR_ARG
        three = [desc(4, 1, 8, at=v.aligned, strides=[v.stride0, 8, v.stride1]) for v in (x, out)]
        if s is not state:
            st = lib.remora_b200_causal_conv_fwd(FAKE, at(conv), ad(three[0]), ad(taps), None, ad(state), None,
                                                 ad(three[1]), ad(s), None)
            assert st == L.ERR_ARG
    h, a, b = desc(4, 8, 3, at=FAR[8]), desc(8, 3, at=FAR[7]), desc(4, 1, 3, at=FAR[9])
    step = L.RemoraSelectiveStepIn(ad(h), ad(x), ad(r), ad(a), ad(b), ad(b))
    for out, s in ((own(4, 8), h), (y, own(4, 8, 3))):
        assert lib.remora_b200_selective_scan_step(FAKE, at(spec), at(step), ad(out), ad(s), None) == L.ERR_ARG


# ------------------------------------------------------------------ binding
def test_a_result_does_not_share_memory_with_a_lazy_clone():
    """Storage that a lazy clone shares is made a result's own before its address is
    taken, in whatever order the operands come; an operand that is only read
    stays shared."""
    import torch

    from remora_b200 import _binding

    def aligned(address):
        return ctypes.cast(address, ctypes.POINTER(ctypes.c_uint64))[1]

    source = torch.arange(6.0)
    at_first = source.data_ptr()  # asking a clone's source for it would make that one's own, too
    clone = torch._lazy_clone(source)
    f32 = torch.float32
    _, (out,), read, written = _binding.describe(-1, (("state", clone[2:], 1), ("state_out", clone[2:], 1, f32, None)), 0)
    assert aligned(read) == aligned(written) != at_first
    shared = torch._lazy_clone(source)
    keep, _, at = _binding.describe(-1, (("x", shared, 1),), 0)
    assert aligned(at) == at_first
    assert source.tolist() == shared.tolist() == list(range(6))


def test_written_raises_versions():
    import torch

    from remora_b200 import _binding

    a, b = torch.zeros(3), torch.zeros(4)
    _binding.written(a, None, b[1:])
    assert (a._version, b._version) == (1, 1)
    with torch.inference_mode():
        _binding.written(torch.zeros(2))
    with pytest.raises(TypeError):
        _binding.written(3.0)


# ------------------------------------------------------------------ strides
def test_reach_counts_the_channels_and_steps_that_there_are():
    """A scan's operands may be as far apart as 2^30 elements within a block: of its
    channels and steps, those that the operand has."""
    far = 1 << 44

    def call(B, T, D, N, strides, offset=0):
        m = scan_operands(B, T, D, N)
        m["u"] = desc(B, T, D, at=far, strides=strides, offset=offset)
        st = scan_fwd(desc(B, T, D, at=1 << 50), **m)
        assert st == LAST
        return "spread" in L.last_error()

    assert not call(1, 5, 2, 4, [0, 1, 1 << 25])
    assert not call(1, 5, 2, 4, [0, 1, (1 << 30) - 1])
    assert not call(1, 5, 2, 4, [0, -1, -(1 << 30) + 1], offset=1 << 40)
    assert not call(1, 2, 2, 64, [0, 1 << 28, 1])
    assert not call(1, 5, 2, 4, [0, 1 << 40, 1])  # one lane per channel: no two steps share a base
    assert not call(2, 5, 300, 4, [1 << 40, 1 << 22, 1 << 22])
    assert call(1, 5, 2, 4, [0, 1, 1 << 30])
    assert call(1, 5, 3, 4, [0, 1, 1 << 29])
    assert call(1, 2, 2, 64, [0, (1 << 30) - 1, 1])
    assert call(1, 5, 300, 4, [0, 1, 1 << 23])  # 256 channels of a block
