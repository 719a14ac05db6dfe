"""Device-tensor API over the C ABI.

Each function takes CUDA tensors (torch is only the allocator and stream
provider here), builds Remora descriptors for them — views keep their storage
base in ``aligned`` and their start in ``offset`` — and calls the matching
``remora_b200_*`` entry point on the current torch stream.  Nothing here
computes on the host.
"""

from __future__ import annotations

import ctypes
from typing import Any, Sequence

from remora_b200 import _lib as L
from remora_b200.abi import tensor_descriptor
from remora_b200.codegen import fold_spec, scan_spec
from remora_b200.errors import RemoraB200Error, RemoraShapeError, RemoraUnsupportedError
from remora_b200.program import Expr, compile_program
from remora_b200.runtime import context


def _torch():
    import torch

    return torch


def dtype_of(t) -> int:
    torch = _torch()
    if t.dtype == torch.float32:
        return L.F32
    if t.dtype == torch.int32:
        return L.I32
    if t.dtype in (torch.bool, torch.uint8):
        return L.BOOL
    raise RemoraB200Error(f"unsupported tensor dtype {t.dtype}")


def torch_dtype(code: int):
    torch = _torch()
    return {L.F32: torch.float32, L.I32: torch.int32, L.BOOL: torch.bool}[code]


def _stream(t) -> ctypes.c_void_p:
    torch = _torch()
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _ctx(t):
    return context(t.device.index if t.device.index is not None else 0)


def _check_cuda(*ts) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RemoraB200Error("remora_b200 ops take CUDA tensors (there is no CPU path)")


def _desc_arrays(tensors: Sequence[Any]):
    descs = [tensor_descriptor(t) for t in tensors]
    ptrs = (ctypes.c_void_p * max(1, len(descs)))()
    ranks = (ctypes.c_int32 * max(1, len(descs)))()
    for k, (d, t) in enumerate(zip(descs, tensors)):
        ptrs[k] = ctypes.addressof(d)
        ranks[k] = t.dim()
    return descs, ptrs, ranks


def frame_shape(tensors: Sequence[Any]) -> tuple[int, ...]:
    """Principal frame under prefix agreement: the highest-rank operand's
    shape, every other operand's shape being a prefix of it."""
    best = max(tensors, key=lambda t: t.dim())
    shape = tuple(best.shape)
    for t in tensors:
        if tuple(t.shape) != shape[: t.dim()]:
            raise RemoraShapeError(f"shapes {tuple(t.shape)} and {shape} do not agree on a prefix frame")
    return shape


# ------------------------------------------------------------------- maps
def map(expr_or_program: Expr | L.RemoraMapProgram, *inputs, out=None, out_dtype: object | None = None,
        compute: object | None = None):
    """Lifted map of an expression over the inputs' common prefix frame."""
    torch = _torch()
    _check_cuda(*inputs)
    if isinstance(expr_or_program, L.RemoraMapProgram):
        prog = expr_or_program
    else:
        comp = compute if compute is not None else (dtype_of(inputs[0]) if inputs else L.F32)
        if comp == L.BOOL and out_dtype is None:
            pass
        prog = compile_program(expr_or_program, len(inputs), compute=comp,
                               out=out_dtype, in_dtypes=[dtype_of(t) for t in inputs])
    if out is None:
        shape = frame_shape(inputs) if inputs else ()
        out = torch.empty(shape, dtype=torch_dtype(prog.out_dtype), device=inputs[0].device)
    _check_cuda(out)
    descs, ptrs, ranks = _desc_arrays(inputs)
    od = tensor_descriptor(out)
    L.check(L.lib().remora_b200_map(_ctx(out).ptr, ctypes.byref(prog), ptrs, ranks, len(inputs),
                                    ctypes.addressof(od), out.dim(), _stream(out)), "map")
    return out


# ------------------------------------------------------------------ folds
def fold(*inputs, op: str = "+", init: float | int = 0, mode: str = "cell", cell_rank: int = 1,
         premap: Expr | None = None, epilogue: str | None = None, out=None, dtype: object | None = None):
    """Cell-frame fold (mode='cell': fold the trailing ``cell_rank`` axes of
    every frame cell) or whole-array fold (mode='all'), optionally fused with a
    premap over one or two inputs and a sqrt epilogue."""
    torch = _torch()
    _check_cuda(*inputs)
    dt = dtype if dtype is not None else dtype_of(inputs[0])
    sp = fold_spec(op=op, init=init, mode=mode, cell_rank=cell_rank, dtype=dt, premap=premap,
                   n_inputs=len(inputs), epilogue=epilogue,
                   premap_in_dtypes=[dtype_of(t) for t in inputs] if premap is not None else None)
    if out is None:
        shape = () if mode == "all" else tuple(inputs[0].shape[: inputs[0].dim() - cell_rank])
        out = torch.empty(shape, dtype=torch_dtype(sp.dtype), device=inputs[0].device)
    descs, ptrs, ranks = _desc_arrays(inputs)
    od = tensor_descriptor(out)
    L.check(L.lib().remora_b200_fold(_ctx(out).ptr, ctypes.byref(sp), ptrs, ranks, len(inputs),
                                     ctypes.addressof(od), out.dim(), _stream(out)), "fold")
    return out


def array_fold(x, init, *, op: str = "+", out=None):
    """Leading-axis fold with an array accumulator: init op x[0] op x[1] ..."""
    torch = _torch()
    _check_cuda(x, init)
    sp = fold_spec(op=op, dtype=dtype_of(x))
    if out is None:
        out = torch.empty(tuple(x.shape[1:]), dtype=x.dtype, device=x.device)
    xd, idd, od = tensor_descriptor(x), tensor_descriptor(init), tensor_descriptor(out)
    L.check(L.lib().remora_b200_array_fold(_ctx(out).ptr, ctypes.byref(sp), ctypes.addressof(xd), x.dim(),
                                           ctypes.addressof(idd), ctypes.addressof(od), _stream(out)),
            "array_fold")
    return out


def scan(x, *, op: str = "+", init: float | int = 0, exclusive: bool = False, right: bool = False, out=None):
    torch = _torch()
    _check_cuda(x)
    sp = scan_spec(op=op, init=init, dtype=dtype_of(x), exclusive=exclusive, right=right)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    xd, od = tensor_descriptor(x), tensor_descriptor(out)
    L.check(L.lib().remora_b200_scan(_ctx(out).ptr, ctypes.byref(sp), ctypes.addressof(xd),
                                     ctypes.addressof(od), x.dim(), _stream(out)), "scan")
    return out


# ------------------------------------------------------------- dense core
def gemm(a, b, *, precision: str = "3xtf32", out=None):
    """C = A . B (rank 2, or batched rank 3) on tcgen05 tensor cores."""
    torch = _torch()
    _check_cuda(a, b)
    prec = {"tf32": L.PREC_TF32, "3xtf32": L.PREC_3XTF32}[precision]
    if out is None:
        shape = (*a.shape[:-1], b.shape[-1])
        out = torch.empty(shape, dtype=torch.float32, device=a.device)
    spec = L.RemoraGemmSpec(prec, 0)
    ad, bd, cd = tensor_descriptor(a), tensor_descriptor(b), tensor_descriptor(out)
    L.check(L.lib().remora_b200_gemm(_ctx(out).ptr, ctypes.byref(spec), ctypes.addressof(ad),
                                     ctypes.addressof(bd), ctypes.addressof(cd), out.dim(), _stream(out)), "gemm")
    return out


# ---------------------------------------------------------- convolution
def _conv_spec(stride: int, pad: int, precision: str) -> L.RemoraConvSpec:
    return L.RemoraConvSpec(int(stride), int(pad), {"tf32": L.PREC_TF32, "3xtf32": L.PREC_3XTF32,
                                                    "2xtf32": L.PREC_2XTF32}[precision], 0)


def conv2d_fwd(x, w, bias=None, *, stride: int = 1, pad: int = 1, precision: str = "3xtf32", out=None):
    torch = _torch()
    _check_cuda(x, w, bias)
    N, C, H, W = x.shape
    K, _, R, S = w.shape
    OH, OW = (H + 2 * pad - R) // stride + 1, (W + 2 * pad - S) // stride + 1
    if out is None:
        out = torch.empty((N, K, OH, OW), dtype=torch.float32, device=x.device)
    sp = _conv_spec(stride, pad, precision)
    xd, wd, yd = tensor_descriptor(x), tensor_descriptor(w), tensor_descriptor(out)
    bd = tensor_descriptor(bias) if bias is not None else None
    L.check(L.lib().remora_b200_conv2d_fwd(_ctx(out).ptr, ctypes.byref(sp), ctypes.addressof(xd),
                                           ctypes.addressof(wd), ctypes.addressof(bd) if bd is not None else None,
                                           ctypes.addressof(yd), _stream(out)), "conv2d_fwd")
    return out


def conv2d_dgrad(dy, w, input_shape, *, stride: int = 1, pad: int = 1, precision: str = "3xtf32", out=None):
    torch = _torch()
    _check_cuda(dy, w)
    if out is None:
        out = torch.empty(tuple(input_shape), dtype=torch.float32, device=dy.device)
    sp = _conv_spec(stride, pad, precision)
    dyd, wd, dxd = tensor_descriptor(dy), tensor_descriptor(w), tensor_descriptor(out)
    L.check(L.lib().remora_b200_conv2d_dgrad(_ctx(out).ptr, ctypes.byref(sp), ctypes.addressof(dyd),
                                             ctypes.addressof(wd), ctypes.addressof(dxd), _stream(out)),
            "conv2d_dgrad")
    return out


def conv2d_wgrad(x, dy, weight_shape, *, stride: int = 1, pad: int = 1, precision: str = "3xtf32", out=None):
    torch = _torch()
    _check_cuda(x, dy)
    if out is None:
        out = torch.empty(tuple(weight_shape), dtype=torch.float32, device=x.device)
    sp = _conv_spec(stride, pad, precision)
    xd, dyd, dwd = tensor_descriptor(x), tensor_descriptor(dy), tensor_descriptor(out)
    L.check(L.lib().remora_b200_conv2d_wgrad(_ctx(out).ptr, ctypes.byref(sp), ctypes.addressof(xd),
                                             ctypes.addressof(dyd), ctypes.addressof(dwd), _stream(out)),
            "conv2d_wgrad")
    return out


# ---------------------------------------------------------------- layout
def im2col(image, kh: int, kw: int, stride: int = 1, out=None):
    torch = _torch()
    _check_cuda(image)
    H, W = image.shape
    oh, ow = (H - kh) // stride + 1, (W - kw) // stride + 1
    if out is None:
        out = torch.empty((oh * ow, kh * kw), dtype=torch.float32, device=image.device)
    sp = L.RemoraIm2colSpec(kh, kw, stride, 0)
    idd, cd = tensor_descriptor(image), tensor_descriptor(out)
    L.check(L.lib().remora_b200_im2col(_ctx(out).ptr, ctypes.byref(sp), ctypes.addressof(idd),
                                       ctypes.addressof(cd), _stream(out)), "im2col")
    return out


def col2im(cols, image_shape: tuple[int, int], kh: int, kw: int, stride: int = 1, out=None):
    torch = _torch()
    _check_cuda(cols)
    if out is None:
        out = torch.empty(tuple(image_shape), dtype=torch.float32, device=cols.device)
    sp = L.RemoraIm2colSpec(kh, kw, stride, 0)
    cd, idd = tensor_descriptor(cols), tensor_descriptor(out)
    L.check(L.lib().remora_b200_col2im(_ctx(out).ptr, ctypes.byref(sp), ctypes.addressof(cd),
                                       ctypes.addressof(idd), _stream(out)), "col2im")
    return out


def transpose(x, out=None):
    torch = _torch()
    _check_cuda(x)
    if out is None:
        out = torch.empty((x.shape[1], x.shape[0]), dtype=x.dtype, device=x.device)
    xd, od = tensor_descriptor(x), tensor_descriptor(out)
    L.check(L.lib().remora_b200_transpose(_ctx(out).ptr, dtype_of(x), ctypes.addressof(xd),
                                          ctypes.addressof(od), _stream(out)), "transpose")
    return out


def synchronize(device: int | None = None) -> None:
    """Synchronise the current stream and surface any device-side timeout."""
    torch = _torch()
    dev = torch.cuda.current_device() if device is None else device
    s = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
    L.check(L.lib().remora_b200_synchronize(context(dev).ptr, s), "synchronize")


def wait_check(limit_cycles: int, signal: bool = False, device: int | None = None) -> None:
    """Enqueue the bounded-wait check (remora_b200_wait_check) on the current
    stream: a wait on a barrier that only `signal` completes, given up after
    `limit_cycles`.  The next synchronize() raises RemoraTimeoutError when it
    ran out."""
    torch = _torch()
    dev = torch.cuda.current_device() if device is None else device
    s = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
    L.check(L.lib().remora_b200_wait_check(context(dev).ptr, int(limit_cycles), int(bool(signal)), s), "wait_check")


# ------------------------------------------- the C runtime helpers on GPU
_CMP = {"<": L.OP_LT, "<=": L.OP_LE, ">": L.OP_GT, ">=": L.OP_GE, "==": L.OP_EQ, "!=": L.OP_NE}


def _sort_like(x, out, grade: bool):
    torch = _torch()
    _check_cuda(x)
    if x.dim() not in (1, 2):
        raise RemoraShapeError(f"{'grade' if grade else 'sort'} takes rank 1 or 2, got rank {x.dim()}")
    if out is None:
        out = torch.empty(x.shape, dtype=torch.int32 if grade else x.dtype, device=x.device)
    xd, od = tensor_descriptor(x), tensor_descriptor(out)
    fn = L.lib().remora_b200_grade if grade else L.lib().remora_b200_sort
    L.check(fn(_ctx(out).ptr, dtype_of(x), ctypes.addressof(xd), ctypes.addressof(od), x.dim(), _stream(out)),
            "grade" if grade else "sort")
    return out


def sort(x, out=None):
    """Ascending sort of a rank-1 array, or of every row of a rank-2 array
    (the reference's remora_sort_* runtime helper)."""
    return _sort_like(x, out, grade=False)


def grade(x, out=None):
    """Stable ascending argsort (int32), per row for rank 2 (remora_grade_*)."""
    return _sort_like(x, out, grade=True)


def filter(x, mask=None, *, pred: tuple[str, float | int] | None = None, out=None, count=None, sync: bool = True):
    """Keeps x[i] where mask[i] != 0 (i32 or bool mask) or where `x[i] op lit`
    for pred = (op, lit), in order (remora_filter_*).  With sync, returns the
    kept values (the count is read back to the host); otherwise returns
    (out, count) with count a device int64 scalar."""
    torch = _torch()
    _check_cuda(x)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if count is None:
        count = torch.zeros((), dtype=torch.int64, device=x.device)
    xd, od, cd = tensor_descriptor(x), tensor_descriptor(out), tensor_descriptor(count)
    if (mask is None) == (pred is None):
        raise RemoraB200Error("filter takes exactly one of mask and pred")
    if pred is not None:
        op, lit = pred
        pr = L.RemoraFilterPred(_CMP[op], float(lit), int(lit), 0)
        st = L.lib().remora_b200_filter(_ctx(out).ptr, dtype_of(x), ctypes.addressof(xd), None, 0,
                                        ctypes.byref(pr), ctypes.addressof(od), ctypes.addressof(cd), _stream(out))
    else:
        _check_cuda(mask)
        md = tensor_descriptor(mask)
        st = L.lib().remora_b200_filter(_ctx(out).ptr, dtype_of(x), ctypes.addressof(xd), ctypes.addressof(md),
                                        dtype_of(mask), None, ctypes.addressof(od), ctypes.addressof(cd),
                                        _stream(out))
    L.check(st, "filter")
    if not sync:
        return out, count
    return out[: int(count.item())]


def replicate(x, counts, out=None, *, total=None, sync: bool = True):
    """x[0] repeated counts[0] times, then x[1] counts[1] times, ...
    (remora_replicate_*; a negative count repeats nothing).  Without `out`
    the total is computed first and read back to size the result."""
    torch = _torch()
    _check_cuda(x, counts)
    if total is None:
        total = torch.zeros((), dtype=torch.int64, device=x.device)
    xd, cd, td = tensor_descriptor(x), tensor_descriptor(counts), tensor_descriptor(total)
    lib = L.lib()
    if out is None:
        L.check(lib.remora_b200_replicate(_ctx(x).ptr, dtype_of(x), ctypes.addressof(xd), ctypes.addressof(cd),
                                          None, ctypes.addressof(td), _stream(x)), "replicate")
        out = torch.empty((int(total.item()),), dtype=x.dtype, device=x.device)
    od = tensor_descriptor(out)
    L.check(lib.remora_b200_replicate(_ctx(x).ptr, dtype_of(x), ctypes.addressof(xd), ctypes.addressof(cd),
                                      ctypes.addressof(od), ctypes.addressof(td), _stream(x)), "replicate")
    if not sync:
        return out, total
    return out[: min(int(total.item()), out.shape[0])]


def rotate(x, shift: int, out=None):
    """out[i] = x[(i + shift) mod N] along axis 0 (remora_rotate_*)."""
    torch = _torch()
    _check_cuda(x)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    xd, od = tensor_descriptor(x), tensor_descriptor(out)
    L.check(L.lib().remora_b200_rotate(_ctx(out).ptr, dtype_of(x), int(shift), ctypes.addressof(xd),
                                       ctypes.addressof(od), x.dim(), _stream(out)), "rotate")
    return out


def append(a, b, out=None):
    """a followed by b along axis 0 (remora_append_*)."""
    torch = _torch()
    _check_cuda(a, b)
    if out is None:
        out = torch.empty((a.shape[0] + b.shape[0], *a.shape[1:]), dtype=a.dtype, device=a.device)
    ad, bd, od = tensor_descriptor(a), tensor_descriptor(b), tensor_descriptor(out)
    L.check(L.lib().remora_b200_append(_ctx(out).ptr, dtype_of(a), ctypes.addressof(ad), ctypes.addressof(bd),
                                       ctypes.addressof(od), a.dim(), _stream(out)), "append")
    return out


# ------------------------------------------------------- sequence operators
# Root-mean-square norm, depthwise causal convolution and selective state
# space scan (include/remora_b200_seq.h).  f32 CUDA tensors with any strides;
# nothing synchronises, and scratch comes from torch on the current stream, so
# every call can be captured into a CUDA graph.  With `lengths`, rows behind a
# sequence's end are never read; results made here are zero there, and those
# rows of a given `out` stay as they were.
def _operands(what: str, **named):
    """Checks that the tensors given are f32 (int32: lengths, slots) on one
    CUDA device; returns their descriptors by name (None for None)."""
    torch = _torch()
    device, descs = None, {}
    for name, t in named.items():
        if t is None:
            descs[name] = None
            continue
        if not t.is_cuda:
            raise RemoraB200Error("remora_b200 ops take CUDA tensors (there is no CPU path)")
        want = torch.int32 if name in ("lengths", "slots") else torch.float8_e4m3fn if name == "q" else torch.float32
        if t.dtype != want:
            raise RemoraUnsupportedError(f"{what}: {name} is {t.dtype}, not {want}")
        if device is None:
            device = t.device
        elif t.device != device:
            raise RemoraB200Error(f"{what}: {name} is on {t.device}, the others on {device}")
        descs[name] = tensor_descriptor(t)
    return descs


def _rank(what: str, t, *ranks: int) -> None:
    if t is not None and t.dim() not in ranks:
        raise RemoraShapeError(f"{what} has rank {t.dim()}, not {' or '.join(f'{r}' for r in ranks)}")


def _at(d):
    return ctypes.addressof(d) if d is not None else None


def _scratch(fn, what: str, device, *sizes):
    """A byte tensor of the size that a _scratch entry point asks for."""
    n = ctypes.c_size_t()
    L.check(fn(*sizes, ctypes.byref(n)), what)
    return _torch().empty((n.value,), dtype=_torch().uint8, device=device) if n.value else None


def _ptr(t):
    return (t.data_ptr(), t.numel() * t.element_size()) if t is not None else (None, 0)


def _fresh(lengths):
    """torch.zeros where some rows will not be written, else torch.empty."""
    return _torch().zeros if lengths is not None else _torch().empty


def rms_norm_fwd(x, w, *, residual=None, eps: float = 1e-6, out=None, sum_out=None):
    """s = x + residual; y = s / sqrt(mean(s^2) + eps) * w over the last axis
    (rank 1 to 4).  Returns y, and (y, s) with a residual.  `out` or `sum_out`
    may be x or the residual itself."""
    torch = _torch()
    _rank("rms_norm_fwd: x", x, 1, 2, 3, 4)
    _rank("rms_norm_fwd: w", w, 1)
    y = out if out is not None else torch.empty(x.shape, dtype=torch.float32, device=x.device)
    s = sum_out
    if s is None and residual is not None:
        s = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    for name, t in (("residual", residual), ("out", y), ("sum_out", s)):
        _rank(f"rms_norm_fwd: {name}", t, x.dim())
    d = _operands("rms_norm_fwd", x=x, w=w, residual=residual, out=y, sum_out=s)
    spec = L.RemoraNormSpec(eps, 0)
    L.check(L.lib().remora_b200_rms_norm_fwd(_ctx(x).ptr, ctypes.addressof(spec), _at(d["x"]), _at(d["residual"]),
                                             _at(d["w"]), _at(d["out"]), _at(d["sum_out"]), x.dim(), _stream(x)),
            "rms_norm_fwd")
    return y if residual is None else (y, s)


def rms_norm_quant(x, w, *, residual=None, eps: float = 1e-6, group: int = 0, out=None, scales=None, sum_out=None):
    """rms_norm_fwd's y as e4m3 values with f32 scales, one per row (group 0)
    or per `group` (32, 64 or 128) columns: y ~ q * scale with scale =
    max(max|y| / 448, 2^-126).  Returns (q, scales), and (q, scales, s) with a
    residual."""
    torch = _torch()
    _rank("rms_norm_quant: x", x, 1, 2, 3, 4)
    _rank("rms_norm_quant: w", w, 1)
    q = out if out is not None else torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    if scales is None:
        scales = torch.empty((*x.shape[:-1], x.shape[-1] // group if group > 0 else 1), dtype=torch.float32,
                             device=x.device)
    s = sum_out
    if s is None and residual is not None:
        s = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    for name, t in (("residual", residual), ("out", q), ("scales", scales), ("sum_out", s)):
        _rank(f"rms_norm_quant: {name}", t, x.dim())
    d = _operands("rms_norm_quant", x=x, w=w, residual=residual, q=q, scales=scales, sum_out=s)
    spec = L.RemoraNormSpec(eps, group)
    L.check(L.lib().remora_b200_rms_norm_quant(_ctx(x).ptr, ctypes.addressof(spec), _at(d["x"]), _at(d["residual"]),
                                               _at(d["w"]), _at(d["q"]), _at(d["scales"]), _at(d["sum_out"]), x.dim(),
                                               _stream(x)), "rms_norm_quant")
    return (q, scales) if residual is None else (q, scales, s)


def rms_norm_bwd(s, w, dy, *, dsum=None, eps: float = 1e-6, out=None):
    """Gradients of rms_norm_fwd from its s (x itself without a residual):
    (dx, dw), dx being the gradient of x and of the residual alike; dsum is
    the gradient that reaches s from its other readers.  `out` (dx) may be s,
    dy or dsum itself."""
    torch = _torch()
    _rank("rms_norm_bwd: s", s, 1, 2, 3, 4)
    _rank("rms_norm_bwd: w", w, 1)
    dx = out if out is not None else torch.empty(s.shape, dtype=torch.float32, device=s.device)
    dw = torch.empty(w.shape, dtype=torch.float32, device=s.device)
    for name, t in (("dy", dy), ("dsum", dsum), ("out", dx)):
        _rank(f"rms_norm_bwd: {name}", t, s.dim())
    d = _operands("rms_norm_bwd", s=s, w=w, dy=dy, dsum=dsum, out=dx, dw=dw)
    lib, ctx = L.lib(), _ctx(s).ptr
    dim = s.shape[-1]
    scratch = _scratch(lib.remora_b200_rms_norm_bwd_scratch, "rms_norm_bwd", s.device, ctx,
                       s.numel() // dim if dim else 0, dim)
    spec = L.RemoraNormSpec(eps, 0)
    L.check(lib.remora_b200_rms_norm_bwd(ctx, ctypes.addressof(spec), _at(d["s"]), _at(d["w"]), _at(d["dy"]),
                                         _at(d["dsum"]), _at(d["out"]), _at(d["dw"]), s.dim(), *_ptr(scratch),
                                         _stream(s)), "rms_norm_bwd")
    return dx, dw


def causal_conv_fwd(x, w, bias=None, *, state=None, lengths=None, silu: bool = False, out=None, state_out=None,
                    return_state: bool = False):
    """Depthwise causal convolution of x [B, L, D] with w [D, W] (2 to 8 taps)
    along time, with an optional bias [D] and SiLU.  The W - 1 rows ahead of a
    sequence are `state` [B, W - 1, D] (zeros without one).  With
    return_state (or state_out, which may be `state` itself) returns
    (y, the state that continues the sequence), else y."""
    torch = _torch()
    _rank("causal_conv_fwd: x", x, 3)
    _rank("causal_conv_fwd: w", w, 2)
    if out is None:
        out = _fresh(lengths)(x.shape, dtype=torch.float32, device=x.device)
    if state_out is None and return_state:
        state_out = torch.empty((x.shape[0], max(w.shape[1] - 1, 0), x.shape[2]), dtype=torch.float32, device=x.device)
    for name, t, r in (("bias", bias, 1), ("state", state, 3), ("lengths", lengths, 1), ("out", out, 3),
                       ("state_out", state_out, 3)):
        _rank(f"causal_conv_fwd: {name}", t, r)
    d = _operands("causal_conv_fwd", x=x, w=w, bias=bias, state=state, lengths=lengths, out=out, state_out=state_out)
    spec = L.RemoraCausalConvSpec(int(bool(silu)), 0)
    L.check(L.lib().remora_b200_causal_conv_fwd(_ctx(x).ptr, ctypes.addressof(spec), _at(d["x"]), _at(d["w"]),
                                                _at(d["bias"]), _at(d["state"]), _at(d["lengths"]), _at(d["out"]),
                                                _at(d["state_out"]), _stream(x)), "causal_conv_fwd")
    return out if state_out is None else (out, state_out)


def causal_conv_bwd(x, w, dy, bias=None, *, state=None, lengths=None, silu: bool = False, dstate_out=None, out=None):
    """Gradients of causal_conv_fwd: (dx, dw, dbias, dstate), dbias and dstate
    None where bias or state is.  dstate_out is the gradient that reaches the
    returned state; `out` receives dx."""
    torch = _torch()
    _rank("causal_conv_bwd: x", x, 3)
    _rank("causal_conv_bwd: w", w, 2)
    B, T, D = x.shape
    dx = out if out is not None else _fresh(lengths)(x.shape, dtype=torch.float32, device=x.device)
    dw = torch.empty(w.shape, dtype=torch.float32, device=x.device)
    dbias = torch.empty(bias.shape, dtype=torch.float32, device=x.device) if bias is not None else None
    dstate = torch.empty(state.shape, dtype=torch.float32, device=x.device) if state is not None else None
    for name, t, r in (("bias", bias, 1), ("state", state, 3), ("lengths", lengths, 1), ("dy", dy, 3), ("out", dx, 3),
                       ("dstate_out", dstate_out, 3)):
        _rank(f"causal_conv_bwd: {name}", t, r)
    d = _operands("causal_conv_bwd", x=x, w=w, bias=bias, state=state, lengths=lengths, dy=dy, dstate_out=dstate_out,
                  out=dx, dw=dw, dbias=dbias, dstate=dstate)
    lib, ctx = L.lib(), _ctx(x).ptr
    scratch = _scratch(lib.remora_b200_causal_conv_bwd_scratch, "causal_conv_bwd", x.device, ctx, B, T, D, w.shape[1])
    spec = L.RemoraCausalConvSpec(int(bool(silu)), 0)
    L.check(lib.remora_b200_causal_conv_bwd(ctx, ctypes.addressof(spec), _at(d["x"]), _at(d["w"]), _at(d["bias"]),
                                            _at(d["state"]), _at(d["lengths"]), _at(d["dy"]), _at(d["dstate_out"]),
                                            _at(d["out"]), _at(d["dw"]), _at(d["dbias"]), _at(d["dstate"]),
                                            *_ptr(scratch), _stream(x)), "causal_conv_bwd")
    return dx, dw, dbias, dstate


def causal_conv_step(x, state, w, bias=None, *, silu: bool = False, slots=None, out=None, state_out=None):
    """One token per row of x [B, D]: y, with the window state [S, W - 1, D]
    moved on in place (or into state_out).  Row i uses state row slots[i], or
    row i without slots; a row whose slot is -1 or was named by an earlier row
    is left out (its y is zero, or as it was in a given `out`)."""
    torch = _torch()
    _rank("causal_conv_step: x", x, 2)
    if out is None:
        out = _fresh(slots)(x.shape, dtype=torch.float32, device=x.device)
    if state_out is None:
        state_out = state
    for name, t, r in (("state", state, 3), ("w", w, 2), ("bias", bias, 1), ("slots", slots, 1), ("out", out, 2),
                       ("state_out", state_out, 3)):
        _rank(f"causal_conv_step: {name}", t, r)
    d = _operands("causal_conv_step", x=x, state=state, w=w, bias=bias, slots=slots, out=out, state_out=state_out)
    spec = L.RemoraCausalConvSpec(int(bool(silu)), 0)
    L.check(L.lib().remora_b200_causal_conv_step(_ctx(x).ptr, ctypes.addressof(spec), _at(d["x"]), _at(d["state"]),
                                                 _at(d["w"]), _at(d["bias"]), _at(d["slots"]), _at(d["out"]),
                                                 _at(d["state_out"]), _stream(x)), "causal_conv_step")
    return out


def _scan_inputs(what: str, u, delta, A, B, C, D, z, delta_bias, h0, lengths):
    for name, t, *ranks in (("u", u, 3), ("delta", delta, 3), ("A", A, 2), ("B", B, 3, 4), ("C", C, 3, 4), ("D", D, 1),
                            ("z", z, 3), ("delta_bias", delta_bias, 1), ("h0", h0, 3), ("lengths", lengths, 1)):
        _rank(f"{what}: {name}", t, *ranks)
    if B.dim() != C.dim():
        raise RemoraShapeError(f"{what}: B has rank {B.dim()} and C rank {C.dim()}")
    return (B, C) if B.dim() == 4 else (B.unsqueeze(2), C.unsqueeze(2))


def selective_scan_fwd(u, delta, A, B, C, D=None, *, z=None, delta_bias=None, softplus: bool = False, h0=None,
                       lengths=None, out=None, h_last=None, return_state: bool = False, save: bool = False):
    """Selective state space scan of u [B, L, D] (see
    remora_b200_selective_scan_fwd): with s = softplus(delta + delta_bias),
    h_t = exp(s A) h_{t-1} + s u B_t per channel and state, y = C_t . h_t + D u,
    times silu(z) with a gate z.  A is [D, N] (N up to 64), B and C are
    [B, L, N] or, shared by groups of channels, [B, L, G, N].  Returns y, then
    the state behind each sequence's end with return_state (or h_last, which
    may be h0 itself), then with save what selective_scan_bwd needs."""
    torch = _torch()
    Bg, Cg = _scan_inputs("selective_scan_fwd", u, delta, A, B, C, D, z, delta_bias, h0, lengths)
    if out is None:
        out = _fresh(lengths)(u.shape, dtype=torch.float32, device=u.device)
    batch, length, dim = u.shape
    states = A.shape[1]
    if h_last is None and return_state:
        h_last = torch.empty((batch, dim, states), dtype=torch.float32, device=u.device)
    _rank("selective_scan_fwd: out", out, 3)
    _rank("selective_scan_fwd: h_last", h_last, 3)
    d = _operands("selective_scan_fwd", u=u, delta=delta, A=A, B=Bg, C=Cg, D=D, z=z, delta_bias=delta_bias, h0=h0,
                  lengths=lengths, out=out, h_last=h_last)
    args = L.RemoraSelectiveScanIn(*(_at(d[k]) for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0",
                                                          "lengths")))
    lib, ctx = L.lib(), _ctx(u).ptr
    scratch = _scratch(lib.remora_b200_selective_scan_fwd_scratch, "selective_scan_fwd", u.device, ctx, batch, length,
                       dim, states, Bg.shape[2])
    saved = None
    if save:
        n = ctypes.c_size_t()
        L.check(lib.remora_b200_selective_scan_saved(batch, length, dim, states, ctypes.byref(n)), "selective_scan_fwd")
        saved = torch.empty((n.value // 4,), dtype=torch.float32, device=u.device)
    spec = L.RemoraSelectiveScanSpec(int(bool(softplus)), 0)
    L.check(lib.remora_b200_selective_scan_fwd(ctx, ctypes.addressof(spec), ctypes.addressof(args), _at(d["out"]),
                                               _at(d["h_last"]), *_ptr(saved), *_ptr(scratch), _stream(u)),
            "selective_scan_fwd")
    results = (out,) + ((h_last,) if h_last is not None else ()) + ((saved,) if save else ())
    return results if len(results) > 1 else out


def selective_scan_bwd(u, delta, A, B, C, dy, saved, D=None, *, z=None, delta_bias=None, softplus: bool = False,
                       h0=None, lengths=None, dh_last=None):
    """Gradients of selective_scan_fwd on the same inputs, from dy and what the
    forward returned with save=True: (du, ddelta, dA, dB, dC, dD, dz,
    ddelta_bias, dh0), None where the input is None.  dh_last is the gradient
    that reaches the returned state."""
    torch = _torch()
    Bg, Cg = _scan_inputs("selective_scan_bwd", u, delta, A, B, C, D, z, delta_bias, h0, lengths)
    _rank("selective_scan_bwd: dy", dy, 3)
    _rank("selective_scan_bwd: dh_last", dh_last, 3)
    _rank("selective_scan_bwd: saved", saved, 1)

    def like(t, fresh):
        return fresh(t.shape, dtype=torch.float32, device=u.device) if t is not None else None

    rows = _fresh(lengths)
    grads = dict(du=like(u, rows), ddelta=like(delta, rows), dA=like(A, torch.empty), dB=like(Bg, rows),
                 dC=like(Cg, rows), dD=like(D, torch.empty), dz=like(z, rows), ddelta_bias=like(delta_bias, torch.empty),
                 dh0=like(h0, torch.empty))
    d = _operands("selective_scan_bwd", u=u, delta=delta, A=A, B=Bg, C=Cg, D=D, z=z, delta_bias=delta_bias, h0=h0,
                  lengths=lengths, dy=dy, dh_last=dh_last, saved=saved, **grads)
    args = L.RemoraSelectiveScanIn(*(_at(d[k]) for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0",
                                                          "lengths")))
    outs = L.RemoraSelectiveScanGrads(*(_at(d[k]) for k in grads))
    if not saved.is_contiguous():
        raise RemoraUnsupportedError("selective_scan_bwd: saved is not the forward's contiguous tensor")
    lib, ctx = L.lib(), _ctx(u).ptr
    batch, length, dim = u.shape
    scratch = _scratch(lib.remora_b200_selective_scan_bwd_scratch, "selective_scan_bwd", u.device, ctx, batch, length,
                       dim, A.shape[1], Bg.shape[2])
    spec = L.RemoraSelectiveScanSpec(int(bool(softplus)), 0)
    L.check(lib.remora_b200_selective_scan_bwd(ctx, ctypes.addressof(spec), ctypes.addressof(args), _at(d["dy"]),
                                               _at(d["dh_last"]), *_ptr(saved), ctypes.addressof(outs), *_ptr(scratch),
                                               _stream(u)), "selective_scan_bwd")
    if B.dim() == 3:
        grads["dB"], grads["dC"] = grads["dB"].squeeze(2), grads["dC"].squeeze(2)
    return tuple(grads.values())


def selective_scan_step(state, u, delta, A, B, C, D=None, *, z=None, delta_bias=None, softplus: bool = False,
                        slots=None, out=None, state_out=None):
    """One token per row of u [B, D] (B and C: [B, N] or [B, G, N]): y, with
    the state [S, D, N] moved on in place (or into state_out).  Row i uses
    state row slots[i], or row i without slots; a row whose slot is -1 or was
    named by an earlier row is left out, as in causal_conv_step."""
    torch = _torch()
    for name, t, *ranks in (("state", state, 3), ("u", u, 2), ("delta", delta, 2), ("A", A, 2), ("B", B, 2, 3),
                            ("C", C, 2, 3), ("D", D, 1), ("z", z, 2), ("delta_bias", delta_bias, 1),
                            ("slots", slots, 1)):
        _rank(f"selective_scan_step: {name}", t, *ranks)
    if B.dim() != C.dim():
        raise RemoraShapeError(f"selective_scan_step: B has rank {B.dim()} and C rank {C.dim()}")
    if B.dim() == 2:
        B, C = B.unsqueeze(1), C.unsqueeze(1)
    if out is None:
        out = _fresh(slots)(u.shape, dtype=torch.float32, device=u.device)
    if state_out is None:
        state_out = state
    _rank("selective_scan_step: out", out, 2)
    _rank("selective_scan_step: state_out", state_out, 3)
    d = _operands("selective_scan_step", state=state, u=u, delta=delta, A=A, B=B, C=C, D=D, z=z,
                  delta_bias=delta_bias, slots=slots, out=out, state_out=state_out)
    args = L.RemoraSelectiveStepIn(*(_at(d[k]) for k in ("state", "u", "delta", "A", "B", "C", "D", "z", "delta_bias",
                                                          "slots")))
    spec = L.RemoraSelectiveScanSpec(int(bool(softplus)), 0)
    L.check(L.lib().remora_b200_selective_scan_step(_ctx(u).ptr, ctypes.addressof(spec), ctypes.addressof(args),
                                                    _at(d["out"]), _at(d["state_out"]), _stream(u)),
            "selective_scan_step")
    return out
