"""Sequence operators on the GPU at the edges of what their calls allow: values
next to a rounding's border, the ends of the f32 range, layouts and sizes that
other kernels take, against 64-bit definitions (tests/seq_reference.py)."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import to_host
from remora_b200 import ops
from test_gpu_seq import dev, rnd

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
