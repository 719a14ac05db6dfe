"""Sequence operators without a GPU: calls that the entry points have to refuse, or
to take, and the host's side of a call.  The C entry points check every argument
before any CUDA call."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from remora_b200 import _lib as L
from test_seq_host import BASE, FAKE, ad, desc

FAR = [BASE + (k << 24) for k in range(32)]
# what a call that is refused for want of memory answers: every other check is behind it
LAST = L.ERR_LIMIT


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
