"""Sequence operators without a GPU: the struct layouts, the refusals of the
C entry points (which check every argument before any CUDA call), and the
64-bit references' gradients against central differences."""

from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest

import seq_reference as ref
from conftest import ROOT
from remora_b200 import _lib as L
from remora_b200.abi import make_memref_descriptor

# a context that is never used: every call below is refused before that
FAKE = ctypes.create_string_buffer(4096)
BASE = 1 << 20  # addresses that nothing reads


def desc(*shape, at=BASE, strides=None, offset=0):
    if strides is None:
        strides = np.cumprod([1, *reversed(shape[1:])])[::-1].tolist() if shape else []
    return make_memref_descriptor(at, shape, strides, offset=offset)


def ad(d):
    return ctypes.addressof(d) if d is not None else None


def test_struct_layouts_match_a_c_compiler(tmp_path):
    structs = [L.RemoraNormSpec, L.RemoraCausalConvSpec, L.RemoraSelectiveScanSpec, L.RemoraSelectiveScanIn,
               L.RemoraSelectiveScanGrads, L.RemoraSelectiveStepIn]
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "remora_b200_seq.h"', "int main(void) {"]
    for s in structs:
        lines.append(f'printf("{s.__name__} %zu\\n", sizeof({s.__name__}));')
        lines += [f'printf("{s.__name__}.{f} %zu\\n", offsetof({s.__name__}, {f}));' for f, _ in s._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join([*lines, "return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for s in structs:
        assert int(got[s.__name__]) == ctypes.sizeof(s)
        for f, _ in s._fields_:
            assert int(got[f"{s.__name__}.{f}"]) == getattr(s, f).offset


# --------------------------------------------------------------- refusals
def norm_fwd(x, w, y, r=None, s=None, rank=2, eps=1e-6):
    spec = L.RemoraNormSpec(eps, 0)
    return L.lib().remora_b200_rms_norm_fwd(FAKE, ctypes.addressof(spec), ad(x), ad(r), ad(w), ad(y), ad(s), rank, None)


def test_norm_refusals():
    far = [BASE + (k << 16) for k in range(8)]
    x, w, y = desc(4, 8, at=far[0]), desc(8, at=far[1]), desc(4, 8, at=far[2])
    n0 = L.launch_count()
    assert L.lib().remora_b200_rms_norm_fwd(None, None, None, None, None, None, None, 2, None) == L.ERR_ARG
    assert norm_fwd(x, w, desc(4, 9, at=far[2])) == L.ERR_SHAPE
    assert norm_fwd(x, desc(7, at=far[1]), y) == L.ERR_SHAPE
    assert norm_fwd(x, w, y, r=desc(3, 8, at=far[3])) == L.ERR_SHAPE
    assert norm_fwd(x, w, y, s=desc(4, 8, at=far[3])) == L.ERR_ARG  # sum without a residual
    assert norm_fwd(x, w, y, eps=-1.0) == L.ERR_ARG
    assert norm_fwd(x, w, y, eps=float("nan")) == L.ERR_ARG
    assert norm_fwd(x, w, y, rank=5) == L.ERR_RANK
    assert norm_fwd(desc(4, 0), desc(0), desc(4, 0)) == L.ERR_SHAPE
    assert norm_fwd(desc(4, 8, at=far[0] + 2), w, y) == L.ERR_ARG  # not aligned to its elements
    assert norm_fwd(x, w, desc(4, 8, at=far[0] + 16)) == L.ERR_ARG  # overlaps x, not in place
    assert norm_fwd(x, w, desc(4, 8, at=far[0], strides=[16, 1])) == L.ERR_ARG  # same start, other strides
    assert norm_fwd(x, w, desc(4, 8, at=far[2], strides=[0, 1])) == L.ERR_ARG
    both = desc(4, 8, at=far[3])
    assert norm_fwd(x, w, both, r=desc(4, 8, at=far[4]), s=both) == L.ERR_ARG
    spec = L.RemoraNormSpec(1e-6, 48)
    q, sc = desc(4, 96, at=far[2]), desc(4, 2, at=far[3])
    args = lambda sp, sc: (FAKE, ctypes.addressof(sp), ad(desc96), None, ad(w96), ad(q), ad(sc), None, 2, None)  # noqa: E731
    desc96, w96 = desc(4, 96, at=far[0]), desc(96, at=far[1])
    assert L.lib().remora_b200_rms_norm_quant(*args(spec, sc)) == L.ERR_UNSUPPORTED
    assert L.lib().remora_b200_rms_norm_quant(*args(L.RemoraNormSpec(1e-6, 64), sc)) == L.ERR_SHAPE
    assert L.lib().remora_b200_rms_norm_quant(*args(L.RemoraNormSpec(1e-6, 32), sc)) == L.ERR_SHAPE  # 3 scales
    n = ctypes.c_size_t()
    assert L.lib().remora_b200_rms_norm_bwd_scratch(FAKE, 100, 8, ctypes.byref(n)) == 0 and n.value > 0
    spec = L.RemoraNormSpec(1e-6, 0)
    bwd = lambda scratch, have: L.lib().remora_b200_rms_norm_bwd(  # noqa: E731
        FAKE, ctypes.addressof(spec), ad(x), ad(w), ad(y), None, ad(both), ad(dw), 2, scratch, have, None)
    dw = desc(8, at=far[5])
    assert bwd(None, 0) == L.ERR_LIMIT and bwd(BASE, 16) == L.ERR_LIMIT and bwd(BASE + 4, 1 << 20) == L.ERR_ARG
    assert L.launch_count() == n0


def test_conv_refusals():
    far = [BASE + (k << 16) for k in range(10)]
    spec = L.RemoraCausalConvSpec(1, 0)
    x, w, y = desc(2, 9, 8, at=far[0]), desc(8, 4, at=far[1]), desc(2, 9, 8, at=far[2])
    state = desc(2, 3, 8, at=far[3])

    def fwd(x=x, w=w, bias=None, state=None, lengths=None, y=y, out=None):
        return L.lib().remora_b200_causal_conv_fwd(FAKE, ctypes.addressof(spec), ad(x), ad(w), ad(bias), ad(state),
                                                   ad(lengths), ad(y), ad(out), None)

    assert fwd(w=desc(8, 9, at=far[1])) == L.ERR_UNSUPPORTED
    assert fwd(w=desc(8, 1, at=far[1])) == L.ERR_UNSUPPORTED
    assert fwd(w=desc(7, 4, at=far[1])) == L.ERR_SHAPE
    assert fwd(bias=desc(7, at=far[4])) == L.ERR_SHAPE
    assert fwd(state=desc(2, 4, 8, at=far[3])) == L.ERR_SHAPE
    assert fwd(lengths=desc(3, at=far[4])) == L.ERR_SHAPE
    assert fwd(y=desc(2, 9, 8, at=far[0])) == L.ERR_ARG  # in place: other threads still read x
    assert fwd(state=state, out=desc(2, 3, 8, at=far[3] + 4)) == L.ERR_ARG
    assert fwd(out=desc(2, 3, 8, at=far[2])) == L.ERR_ARG  # state_out over y
    assert fwd(x=None) == L.ERR_ARG
    # columns of one wider array do not overlap: this is refused for its shape only
    wide = [desc(2, 9, 8, at=far[0], strides=[9 * 16, 16, 1], offset=o) for o in (0, 8)]
    assert fwd(x=wide[0], y=wide[1], bias=desc(7, at=far[4])) == L.ERR_SHAPE
    assert fwd(x=wide[0], y=desc(2, 9, 8, at=far[0], strides=[9 * 16, 16, 1], offset=7)) == L.ERR_ARG

    def step(x, state, y, out, slots=None):
        return L.lib().remora_b200_causal_conv_step(FAKE, ctypes.addressof(spec), ad(x), ad(state), ad(w), None,
                                                    ad(slots), ad(y), ad(out), None)

    x1, y1 = desc(3, 8, at=far[5]), desc(3, 8, at=far[6])
    assert step(x1, state, y1, state) == L.ERR_SHAPE  # three rows, two states
    assert step(x1, state, y1, state, slots=desc(2, at=far[4])) == L.ERR_SHAPE
    big, bigs = desc(70000, 8, at=far[5]), desc(70000, at=far[9])
    assert step(big, state, desc(70000, 8, at=far[9] + (1 << 24)), state, slots=bigs) == L.ERR_LIMIT
    n = ctypes.c_size_t()
    assert L.lib().remora_b200_causal_conv_bwd_scratch(FAKE, 2, 9, 8, 9, ctypes.byref(n)) == L.ERR_UNSUPPORTED
    assert L.lib().remora_b200_causal_conv_bwd_scratch(FAKE, -1, 9, 8, 4, ctypes.byref(n)) == L.ERR_ARG


def test_scan_refusals():
    far = [BASE + (k << 16) for k in range(16)]
    spec = L.RemoraSelectiveScanSpec(1, 0)
    good = dict(u=desc(2, 9, 6, at=far[0]), delta=desc(2, 9, 6, at=far[1]), a=desc(6, 5, at=far[2]),
                b=desc(2, 9, 2, 5, at=far[3]), c=desc(2, 9, 2, 5, at=far[4]), d=None, z=None, delta_bias=None, h0=None,
                lengths=None)

    def fwd(y=desc(2, 9, 6, at=far[5]), h=None, saved=(None, 0), **kw):
        m = {**good, **kw}
        args = L.RemoraSelectiveScanIn(*(ad(v) for v in m.values()))
        return L.lib().remora_b200_selective_scan_fwd(FAKE, ctypes.addressof(spec), ctypes.addressof(args), ad(y), ad(h),
                                                      *saved, None, 0, None)

    assert fwd(u=None) == L.ERR_ARG
    assert fwd(delta=desc(2, 8, 6, at=far[1])) == L.ERR_SHAPE
    assert fwd(a=desc(6, 65, at=far[2])) == L.ERR_UNSUPPORTED
    assert fwd(b=desc(2, 9, 4, 5, at=far[3])) == L.ERR_SHAPE  # six channels in four groups
    assert fwd(c=desc(2, 9, 1, 5, at=far[4])) == L.ERR_SHAPE
    assert fwd(z=desc(2, 9, 5, at=far[6])) == L.ERR_SHAPE
    assert fwd(h0=desc(2, 6, 4, at=far[6])) == L.ERR_SHAPE
    assert fwd(lengths=desc(1, at=far[6])) == L.ERR_SHAPE
    assert fwd(y=desc(2, 9, 6, at=far[0])) == L.ERR_ARG
    assert fwd(h0=desc(2, 6, 5, at=far[6]), h=desc(2, 6, 5, at=far[6] + 8)) == L.ERR_ARG
    assert fwd(saved=(BASE, 8)) == L.ERR_LIMIT
    assert fwd(saved=(BASE + 4, 1 << 20)) == L.ERR_ARG
    n = ctypes.c_size_t()
    lib = L.lib()
    assert lib.remora_b200_selective_scan_fwd_scratch(FAKE, 1, 4096, 64, 16, 1, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.remora_b200_selective_scan_bwd_scratch(FAKE, 1, 10, 64, 0, 1, ctypes.byref(n)) == L.ERR_UNSUPPORTED
    assert lib.remora_b200_selective_scan_bwd_scratch(FAKE, 1, 10, 64, 16, 0, ctypes.byref(n)) == L.ERR_SHAPE
    assert lib.remora_b200_selective_scan_bwd_scratch(None, 1, 10, 64, 16, 1, ctypes.byref(n)) == L.ERR_ARG
    args = L.RemoraSelectiveScanIn(*(ad(v) for v in good.values()))
    outs = [desc(2, 9, 6, at=far[8]), desc(2, 9, 6, at=far[9]), desc(6, 5, at=far[10]), desc(2, 9, 2, 5, at=far[11]),
            desc(2, 9, 2, 5, at=far[12]), None, None, None, None]

    def bwd(outs):
        g = L.RemoraSelectiveScanGrads(*(ad(v) for v in outs))
        dy = desc(2, 9, 6, at=far[7])
        return lib.remora_b200_selective_scan_bwd(FAKE, ctypes.addressof(spec), ctypes.addressof(args), ad(dy), None,
                                                  None, 0, ctypes.addressof(g), None, 0, None)

    assert bwd(outs) == L.ERR_LIMIT  # no saved states
    assert bwd([None, *outs[1:]]) == L.ERR_ARG
    assert bwd([*outs[:6], desc(2, 9, 6, at=far[13]), None, None]) == L.ERR_ARG  # dz without z
    assert bwd([outs[0], outs[0], *outs[2:]]) == L.ERR_ARG  # one array for two gradients


def test_scan_step_refusals():
    far = [BASE + (k << 40) for k in range(12)]
    spec = L.RemoraSelectiveScanSpec(1, 0)
    good = dict(state=desc(4, 6, 5, at=far[0]), u=desc(2, 6, at=far[1]), delta=desc(2, 6, at=far[2]),
                a=desc(6, 5, at=far[3]), b=desc(2, 2, 5, at=far[4]), c=desc(2, 2, 5, at=far[5]), d=None, z=None,
                delta_bias=None, slots=None)

    def step(y=desc(2, 6, at=far[6]), out=None, **kw):
        m = {**good, **kw}
        args = L.RemoraSelectiveStepIn(*(ad(v) for v in m.values()))
        return L.lib().remora_b200_selective_scan_step(FAKE, ctypes.addressof(spec), ctypes.addressof(args), ad(y),
                                                       ad(out or m["state"]), None)

    assert step(u=None) == L.ERR_ARG
    assert step(state=desc(1, 6, 5, at=far[0])) == L.ERR_SHAPE  # two rows, one state
    assert step(state=desc(4, 6, 4, at=far[0])) == L.ERR_SHAPE
    assert step(b=desc(2, 4, 5, at=far[4])) == L.ERR_SHAPE  # six channels in four groups
    assert step(slots=desc(3, at=far[7])) == L.ERR_SHAPE
    assert step(y=desc(2, 6, at=far[1])) == L.ERR_ARG
    assert step(out=desc(4, 6, 5, at=far[0] + 8)) == L.ERR_ARG  # neither the state nor apart from it
    assert step(state=desc(4, 6, 5, at=far[0], strides=[1 << 31, 5, 1])) == L.ERR_LIMIT
    assert step(state=desc(1 << 29, 6, 5, at=far[0])) == L.ERR_LIMIT
    assert step(u=desc(2, 6, at=far[1], strides=[-(1 << 31), 1], offset=1 << 31)) == L.ERR_LIMIT


def test_overlap_is_decided_by_the_elements():
    """Against enumeration: random small views of one buffer as s and dx of a
    norm's backward, refused as overlapping exactly where they share an element
    and are not the same view; the others are refused for want of scratch."""
    rng = np.random.default_rng(0)
    spec = L.RemoraNormSpec(1e-6, 0)
    seen = set()
    for _ in range(400):
        n, d = int(rng.integers(1, 5)), int(rng.integers(1, 6))
        views, cells = [], []
        for _ in range(2):
            strides = [int(rng.integers(-14, 15)), int(rng.choice([-2, -1, 1, 2, 3]))]
            strides = [x if x or k else 9 for k, x in enumerate(strides)]
            off = int(rng.integers(60, 90))
            views.append(desc(n, d, at=BASE, strides=strides, offset=off))
            cells.append({off + i * strides[0] + j * strides[1] for i in range(n) for j in range(d)})
        r, w = desc(n, d, at=BASE + (1 << 17)), desc(d, at=BASE + (1 << 18), strides=[1])
        st = L.lib().remora_b200_rms_norm_bwd(FAKE, ctypes.addressof(spec), ad(views[1]), ad(w), ad(r), None,
                                              ad(views[0]), ad(desc(d, at=BASE + (1 << 19))), 2, None, 0, None)
        in_place = (views[0].offset == views[1].offset and (n == 1 or views[0].stride0 == views[1].stride0)
                    and (d == 1 or views[0].stride1 == views[1].stride1))
        shared = bool(cells[0] & cells[1]) and not in_place
        assert st == (L.ERR_ARG if shared else L.ERR_LIMIT), L.last_error()
        seen.add((shared, in_place))
    assert {(True, False), (False, False)} <= seen


def test_ops_take_cuda_tensors():
    import torch

    from remora_b200 import ops
    from remora_b200.errors import RemoraB200Error

    t = torch.zeros
    with pytest.raises(RemoraB200Error, match="CUDA"):
        ops.rms_norm_fwd(t(2, 4), t(4))
    with pytest.raises(RemoraB200Error, match="CUDA"):
        ops.causal_conv_fwd(t(2, 3, 4), t(4, 3))
    with pytest.raises(RemoraB200Error, match="CUDA"):
        ops.selective_scan_fwd(t(2, 3, 4), t(2, 3, 4), t(4, 5), t(2, 3, 5), t(2, 3, 5))


def test_binding_lays_out_descriptors():
    """The binding's buffer holds the descriptors that tensor_descriptor makes
    (the view's start in `offset`), and refuses what does not fit."""
    import torch

    from remora_b200 import _binding
    from remora_b200.abi import tensor_descriptor

    base = torch.arange(120.0).reshape(4, 5, 6)
    views = [base, base[1:, ::2, 3:].permute(2, 0, 1), base[0, 0, 0], torch.zeros(0, 3), base[:, :1].expand(4, 5, 6)]
    operands = tuple((f"t{k}", t, t.dim()) for k, t in enumerate(views)) + (
        ("none", None, 2), ("ints", torch.arange(3, dtype=torch.int32), 1, torch.int32))
    for table in (0, 2, len(operands)):
        buf, results, *at = _binding.describe(-1, operands, table)
        assert results == ()
        if table:
            first = ctypes.cast(at[0], ctypes.POINTER(ctypes.c_uint64))
            at = [first[k] or None for k in range(table)] + at[1:]
        assert len(at) == len(operands) and at[5] is None
        for (_, t, *_rest), address in zip(operands, at):
            if t is None:
                continue
            want = tensor_descriptor(t)
            if not t.numel():
                want.allocated = want.aligned = 0
            assert ctypes.string_at(address, ctypes.sizeof(want)) == bytes(want)
    one = torch.zeros(2, 3)
    got = _binding.describe(-1, (("a", None, 2, torch.float32, one.t()), ("b", one, 2, torch.float32, one),
                                 ("c", None, 2, torch.float32, None), ("d", None, 1, torch.int32, (7,))), 0)
    made, given, absent, ints = got[1]
    assert made.shape == (3, 2) and made.is_contiguous() and made.dtype == torch.float32
    assert given is one and absent is None and ints.shape == (7,) and ints.dtype == torch.int32
    assert got[4] is None
    for address, t in zip((got[2], got[3], got[5]), (made, one, ints)):
        want = tensor_descriptor(t)
        assert ctypes.string_at(address, ctypes.sizeof(want)) == bytes(want)
    for bad in (("x", one, 3), ("x", one.double(), 2), ("x", one, 2, torch.int32), ("x", 3.0, 0), ("x", one.to_sparse(), 2)):
        assert _binding.describe(-1, (bad,), 0) is None
    assert _binding.describe(0, (("x", one, 2),), 0) is None  # another device
    room, address = _binding.room(-1, 48)
    assert room.shape == (48,) and room.dtype == torch.uint8 and room.data_ptr() == address
    with pytest.raises(RuntimeError):
        _binding.room(-1, -1)
    negated = torch.zeros(2, 3, dtype=torch.complex64).conj().imag  # its storage holds the negatives
    assert negated.is_neg() and _binding.describe(-1, (("x", negated, 2),), 0) is None
    for wrong in ((-1, [("x", one, 2)], 0), (-1, (("x", one),), 0), (-1, (("x", one, 2, "f32"),), 0), (-1, (("x", one, 2),), 2)):
        with pytest.raises((TypeError, ValueError)):
            _binding.describe(*wrong)


# ------------------------------------------------- the references' gradients
def central(f, x, eps=1e-5):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        v = x[i]
        x[i] = v + eps
        hi = f()
        x[i] = v - eps
        lo = f()
        x[i] = v
        g[i] = (hi - lo) / (2 * eps)
    return g


# A central difference with step h of a smooth function is off by f''' h^2 / 6
# (1e-10 here) and by the rounding of f over h (1e-16 |f| / 1e-5 = 1e-11 |f|).
TOL = dict(rtol=1e-7, atol=1e-8)


def test_reference_norm_gradient():
    rng = np.random.default_rng(0)
    s, w, dy, ds = rng.normal(size=(3, 5)), rng.normal(size=5), rng.normal(size=(3, 5)), rng.normal(size=(3, 5))
    f = lambda: (ref.rms_norm(s, w, None, 1e-3)[0] * dy).sum() + (s * ds).sum()  # noqa: E731
    dx, dw = ref.rms_norm_bwd(s, w, dy, ds, 1e-3)
    np.testing.assert_allclose(dx, central(f, s), **TOL)
    np.testing.assert_allclose(dw, central(f, w), **TOL)


@pytest.mark.parametrize("silu", [False, True])
def test_reference_conv_gradient(silu):
    rng = np.random.default_rng(1)
    x, w, b, s = rng.normal(size=(3, 5, 2)), rng.normal(size=(2, 4)), rng.normal(size=2), rng.normal(size=(3, 3, 2))
    dy, dl, lengths = rng.normal(size=x.shape), rng.normal(size=s.shape), [5, 2, 0]

    def f():
        y, last = ref.causal_conv(x, w, b, s, lengths, silu)
        return (y * dy).sum() + (last * dl).sum()

    for got, at in zip(ref.causal_conv_bwd(x, w, b, s, lengths, silu, dy, dl), (x, w, b, s)):
        np.testing.assert_allclose(got, central(f, at), **TOL)


def test_reference_scan_gradient():
    rng = np.random.default_rng(2)
    nb, Lt, D, N, G = 2, 4, 4, 3, 2
    v = dict(u=rng.normal(size=(nb, Lt, D)), delta=rng.normal(size=(nb, Lt, D)), A=-rng.uniform(0.2, 2, (D, N)),
             B=rng.normal(size=(nb, Lt, G, N)), C=rng.normal(size=(nb, Lt, G, N)), D=rng.normal(size=D),
             z=rng.normal(size=(nb, Lt, D)), bias=rng.normal(size=D), h0=rng.normal(size=(nb, D, N)))
    dy, dl, lengths = rng.normal(size=(nb, Lt, D)), rng.normal(size=(nb, D, N)), [4, 2]
    call = lambda: (v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], True, v["h0"], lengths)  # noqa: E731

    def f():
        y, last = ref.selective_scan(*call())
        return (y * dy).sum() + (last * dl).sum()

    got = ref.selective_scan_bwd(*call(), dy, dl)
    for k, name in (("u", "du"), ("delta", "ddelta"), ("A", "dA"), ("B", "dB"), ("C", "dC"), ("D", "dD"), ("z", "dz"),
                    ("bias", "ddelta_bias"), ("h0", "dh0")):
        np.testing.assert_allclose(got[name], central(f, v[k]), **TOL)
