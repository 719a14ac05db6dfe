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
#
# Arrays that a caller gives to be written count as modified in place: autograd
# refuses a backward pass that would have needed their old values.
#
# A single-token call costs what the host does, so the operands of a call are
# checked and laid out, and its results made, natively (csrc/binding.cpp).
def _describe(what: str, device: int, operands, table: int = 0):
    """Checks (name, tensor or None, rank[, dtype[, shape]]) operands, f32
    unless a dtype is given, on CUDA device `device`; one with a shape (a
    tensor's, or a tuple) is a result, made where it is None.  Returns the
    buffer that holds their descriptors, to be kept until the call returns,
    the tuple of results, and the address of each operand (None for None).
    With `table`, one address stands for the first `table`: that of a struct
    of their addresses."""
    described = _binding().describe(device, operands, table)
    if described is None:
        _refuse(what, device, operands)
    return described


def _binding():
    global _binding_module
    if _binding_module is None:
        torch = _torch()  # its libraries are the binding's
        build = "run `python -m remora_b200.csrc.build`"
        try:
            from remora_b200 import _binding as module
        except ImportError as e:
            raise RemoraB200Error(f"remora_b200._binding is not built, or not for the installed torch; {build} ({e})")
        if module.torch_release != torch.__version__:
            raise RemoraB200Error(
                f"remora_b200._binding is built for torch {module.torch_release}, not {torch.__version__}; {build}")
        _binding_module = module
    return _binding_module


_binding_module = None


def _refuse(what: str, device: int, operands) -> None:
    """Raises for the first operand that describe() does not take."""
    torch = _torch()
    for name, t, rank, *more in operands:
        want = more[0] if more else torch.float32
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise RemoraB200Error(f"{what}: {name} is a {type(t).__name__}, not a tensor")
        if not t.is_cuda:
            raise RemoraB200Error("remora_b200 ops take CUDA tensors (there is no CPU path)")
        if t.dtype != want:
            raise RemoraUnsupportedError(f"{what}: {name} is {t.dtype}, not {want}")
        if t.get_device() != device:
            raise RemoraB200Error(f"{what}: {name} is on {t.device}, the first operand on cuda:{device}")
        if t.dim() != rank:
            raise RemoraShapeError(f"{what}: {name} has rank {t.dim()}, not {rank}")
    raise RemoraUnsupportedError(
        f"{what}: an operand has no dense storage, is a lazily negated view, or has a rank over {L.MAX_RANK}")


def _want_tensors(what: str, **operands) -> None:
    """Refuses operands that are no tensors, where a shape is needed ahead of
    _describe or a missing operand's after it."""
    for name, t in operands.items():
        if not isinstance(t, _torch().Tensor):
            raise RemoraB200Error(f"{what}: {name} is a {type(t).__name__}, not a tensor")


def _cuda_index(t) -> int:
    if not isinstance(t, _torch().Tensor):
        raise RemoraB200Error(f"the first operand is a {type(t).__name__}, not a tensor")
    index = t.get_device()
    if index < 0:
        raise RemoraB200Error("remora_b200 ops take CUDA tensors (there is no CPU path)")
    return index


def _raw_stream(device: int) -> int:
    """The current stream's handle, without a Stream object where torch can."""
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


def _scratch(fn, what: str, device: int, *sizes):
    """(byte tensor, address, bytes) of the memory that a _scratch or _saved entry point asks for."""
    n = ctypes.c_size_t()
    L.check(fn(*sizes, ctypes.byref(n)), what)
    if not n.value:
        return None, None, 0
    return *_binding().room(device, n.value), n.value


# indexed by the flag and by zero_rest: set for results made here, whose rows
# outside every sequence shall be zero, not for a caller's
_CONV_SPECS = tuple(tuple(L.RemoraCausalConvSpec(k, zero) for zero in (0, 1)) for k in (0, 1))
_SCAN_SPECS = tuple(tuple(L.RemoraSelectiveScanSpec(k, zero) for zero in (0, 1)) for k in (0, 1))


def _spec(specs, flag, made_here: bool) -> int:
    return ctypes.addressof(specs[1 if flag else 0][1 if made_here else 0])


def rms_norm_fwd(x, w, *, residual=None, eps: float = 1e-6, out=None, sum_out=None):
    """s = x + residual; y = s / sqrt(mean(s^2) + eps) * w over the last axis
    (rank 1 to 4).  Returns y, and (y, s) with a residual.  `out` or `sum_out`
    may be x or the residual itself."""
    device, rank, f32 = _cuda_index(x), x.dim(), _torch().float32
    keep, (y, s), xd, rd, wd, yd, sd = _describe("rms_norm_fwd", device, (
        ("x", x, rank), ("residual", residual, rank), ("w", w, 1), ("out", out, rank, f32, x),
        ("sum_out", sum_out, rank, f32, residual)))
    spec = L.RemoraNormSpec(eps, 0)
    L.check(L.lib().remora_b200_rms_norm_fwd(context(device).ptr, ctypes.addressof(spec), xd, rd, wd, yd, sd, rank,
                                             _raw_stream(device)), "rms_norm_fwd")
    _binding().written(y, s)
    return y if residual is None else (y, s)


def rms_norm_quant(x, w, *, residual=None, eps: float = 1e-6, group: int = 0, out=None, scales=None, sum_out=None):
    """rms_norm_fwd's y as e4m3 values with f32 scales, one per row (group 0)
    or per `group` (32, 64 or 128) columns: y ~ q * scale with scale =
    max(max|y| / 448, 2^-126).  Returns (q, scales), and (q, scales, s) with a
    residual."""
    torch = _torch()
    device, rank, f32 = _cuda_index(x), x.dim(), torch.float32
    columns = x.shape[-1] // group if group > 0 and rank else 1
    keep, (scales, s, q), xd, rd, wd, cd, sd, qd = _describe("rms_norm_quant", device, (
        ("x", x, rank), ("residual", residual, rank), ("w", w, 1), ("scales", scales, rank, f32, (*x.shape[:-1], columns)),
        ("sum_out", sum_out, rank, f32, residual), ("out", out, rank, torch.float8_e4m3fn, x)))
    spec = L.RemoraNormSpec(eps, group)
    L.check(L.lib().remora_b200_rms_norm_quant(context(device).ptr, ctypes.addressof(spec), xd, rd, wd, qd, cd, sd,
                                               rank, _raw_stream(device)), "rms_norm_quant")
    _binding().written(q, scales, s)
    return (q, scales) if residual is None else (q, scales, s)


def rms_norm_bwd(s, w, dy, *, dsum=None, eps: float = 1e-6, out=None):
    """Gradients of rms_norm_fwd from its s (x itself without a residual):
    (dx, dw), dx being the gradient of x and of the residual alike; dsum is
    the gradient that reaches s from its other readers.  `out` (dx) may be s,
    dy or dsum itself."""
    device, rank, f32 = _cuda_index(s), s.dim(), _torch().float32
    keep, (dx, dw), sd, wd, gd, ed, xd, dwd = _describe("rms_norm_bwd", device, (
        ("s", s, rank), ("w", w, 1), ("dy", dy, rank), ("dsum", dsum, rank), ("out", out, rank, f32, s),
        ("dw", None, 1, f32, w)))
    lib, ctx = L.lib(), context(device).ptr
    dim = s.shape[-1] if rank else 0
    scratch, at, size = _scratch(lib.remora_b200_rms_norm_bwd_scratch, "rms_norm_bwd", device, ctx,
                                 s.numel() // dim if dim else 0, dim)
    spec = L.RemoraNormSpec(eps, 0)
    L.check(lib.remora_b200_rms_norm_bwd(ctx, ctypes.addressof(spec), sd, wd, gd, ed, xd, dwd, rank, at, size,
                                         _raw_stream(device)), "rms_norm_bwd")
    _binding().written(dx)
    return dx, dw


def causal_conv_fwd(x, w, bias=None, *, state=None, lengths=None, silu: bool = False, out=None, state_out=None,
                    return_state: bool = False):
    """Depthwise causal convolution of x [B, L, D] with w [D, W] (2 to 8 taps)
    along time, with an optional bias [D] and SiLU.  The W - 1 rows ahead of a
    sequence are `state` [B, W - 1, D] (zeros without one).  With
    return_state (or state_out, which may be `state` itself) returns
    (y, the state that continues the sequence), else y."""
    torch = _torch()
    device, f32 = _cuda_index(x), torch.float32
    if return_state:
        _want_tensors("causal_conv_fwd", w=w)
    wanted = (x.shape[0], max(w.shape[1] - 1, 0), x.shape[2]) if return_state and x.dim() == 3 and w.dim() == 2 else None
    keep, (y, state_out), xd, wd, bd, sd, yd, od, ld = _describe("causal_conv_fwd", device, (
        ("x", x, 3), ("w", w, 2), ("bias", bias, 1), ("state", state, 3), ("out", out, 3, f32, x),
        ("state_out", state_out, 3, f32, wanted), ("lengths", lengths, 1, torch.int32)))
    L.check(L.lib().remora_b200_causal_conv_fwd(context(device).ptr, _spec(_CONV_SPECS, silu, out is None), xd, wd, bd,
                                                sd, ld, yd, od, _raw_stream(device)), "causal_conv_fwd")
    _binding().written(y, state_out)
    return y if state_out is None else (y, state_out)


def causal_conv_bwd(x, w, dy, bias=None, *, state=None, lengths=None, silu: bool = False, dstate_out=None, out=None):
    """Gradients of causal_conv_fwd: (dx, dw, dbias, dstate), dbias and dstate
    None where bias or state is.  dstate_out is the gradient that reaches the
    returned state; `out` receives dx."""
    torch = _torch()
    device, f32 = _cuda_index(x), torch.float32
    _want_tensors("causal_conv_bwd", w=w)
    keep, (dx, dw, dbias, dstate), xd, wd, bd, sd, gd, ed, dxd, dwd, dbd, dsd, ld = _describe("causal_conv_bwd", device, (
        ("x", x, 3), ("w", w, 2), ("bias", bias, 1), ("state", state, 3), ("dy", dy, 3), ("dstate_out", dstate_out, 3),
        ("out", out, 3, f32, x), ("dw", None, 2, f32, w), ("dbias", None, 1, f32, bias),
        ("dstate", None, 3, f32, state), ("lengths", lengths, 1, torch.int32)))
    lib, ctx = L.lib(), context(device).ptr
    scratch, at, size = _scratch(lib.remora_b200_causal_conv_bwd_scratch, "causal_conv_bwd", device, ctx, *x.shape,
                                 w.shape[1])
    L.check(lib.remora_b200_causal_conv_bwd(ctx, _spec(_CONV_SPECS, silu, out is None), xd, wd, bd, sd, ld, gd, ed, dxd,
                                            dwd, dbd, dsd, at, size, _raw_stream(device)), "causal_conv_bwd")
    _binding().written(dx)
    return dx, dw, dbias, dstate


def causal_conv_step(x, state, w, bias=None, *, silu: bool = False, slots=None, out=None, state_out=None):
    """One token per row of x [B, D]: y, with the window state [S, W - 1, D]
    moved on in place (or into state_out).  Row i uses state row slots[i], or
    row i without slots; a row whose slot is -1 or was named by an earlier row
    is left out (its y is zero, or as it was in a given `out`).  Finding those
    takes time that grows with the square of the rows."""
    torch = _torch()
    device = _cuda_index(x)
    if state_out is None:
        state_out = state
    keep, (y, _), xd, sd, wd, bd, yd, od, ld = _describe("causal_conv_step", device, (
        ("x", x, 2), ("state", state, 3), ("w", w, 2), ("bias", bias, 1), ("out", out, 2, torch.float32, x),
        ("state_out", state_out, 3, torch.float32, None), ("slots", slots, 1, torch.int32)))
    L.check(L.lib().remora_b200_causal_conv_step(context(device).ptr, _spec(_CONV_SPECS, silu, out is None), xd, sd, wd,
                                                 bd, ld, yd, od, _raw_stream(device)), "causal_conv_step")
    _binding().written(y, state_out)
    return y


def _groups(what: str, B, C, rank: int):
    """B and C with their group axis: rank - 1 means one group."""
    try:
        b, c = B.dim(), C.dim()
    except AttributeError:
        _want_tensors(what, B=B, C=C)
        raise
    if b != c or not rank - 1 <= b <= rank:
        raise RemoraShapeError(f"{what}: B has rank {b} and C rank {c}, not both {rank - 1} or {rank}")
    return (B, C) if b == rank else (B.unsqueeze(-2), C.unsqueeze(-2))


def selective_scan_fwd(u, delta, A, B, C, D=None, *, z=None, delta_bias=None, softplus: bool = False, h0=None,
                       lengths=None, out=None, h_last=None, return_state: bool = False, save: bool = False):
    """Selective state space scan of u [B, L, D] (see
    remora_b200_selective_scan_fwd): with s = softplus(delta + delta_bias),
    h_t = exp(s A) h_{t-1} + s u B_t per channel and state, y = C_t . h_t + D u,
    times silu(z) with a gate z.  A is [D, N] (N up to 64), B and C are
    [B, L, N] or, shared by groups of channels, [B, L, G, N].  Returns y, then
    the state behind each sequence's end with return_state (or h_last, which
    may be h0 itself), then with save what selective_scan_bwd needs: the states
    of every fourth position (every eighth above 16 states, sixteenth above 32),
    with 16 states 16 bytes per element of u, four times u itself."""
    torch = _torch()
    device = _cuda_index(u)
    _want_tensors("selective_scan_fwd", A=A)
    Bg, Cg = _groups("selective_scan_fwd", B, C, 4)
    f32 = torch.float32
    wanted = (u.shape[0], u.shape[2], A.shape[1]) if return_state and u.dim() == 3 and A.dim() == 2 else None
    keep, (y, h_last), args, yd, hd = _describe("selective_scan_fwd", device, (
        ("u", u, 3), ("delta", delta, 3), ("A", A, 2), ("B", Bg, 4), ("C", Cg, 4), ("D", D, 1), ("z", z, 3),
        ("delta_bias", delta_bias, 1), ("h0", h0, 3), ("lengths", lengths, 1, torch.int32), ("out", out, 3, f32, u),
        ("h_last", h_last, 3, f32, wanted)), table=10)
    lib, ctx = L.lib(), context(device).ptr
    sizes = (*u.shape, A.shape[1])
    scratch, at, size = _scratch(lib.remora_b200_selective_scan_fwd_scratch, "selective_scan_fwd", device, ctx, *sizes,
                                 Bg.shape[2])
    saved, kept, kept_size = None, None, 0
    if save:
        saved, kept, kept_size = _scratch(lib.remora_b200_selective_scan_saved, "selective_scan_fwd", device, *sizes)
        saved = torch.empty((0,), dtype=f32, device=u.device) if saved is None else saved.view(f32)
    L.check(lib.remora_b200_selective_scan_fwd(ctx, _spec(_SCAN_SPECS, softplus, out is None), args, yd, hd, kept,
                                               kept_size, at, size, _raw_stream(device)), "selective_scan_fwd")
    _binding().written(y, h_last)
    results = (y,) + ((h_last,) if h_last is not None else ()) + ((saved,) if save else ())
    return results if len(results) > 1 else y


def selective_scan_bwd(u, delta, A, B, C, dy, saved, D=None, *, z=None, delta_bias=None, softplus: bool = False,
                       h0=None, lengths=None, dh_last=None):
    """Gradients of selective_scan_fwd on the same inputs, from dy and what the
    forward returned with save=True: (du, ddelta, dA, dB, dC, dD, dz,
    ddelta_bias, dh0), None where the input is None.  dh_last is the gradient
    that reaches the returned state."""
    device = _cuda_index(u)
    _want_tensors("selective_scan_bwd", A=A, saved=saved)
    Bg, Cg = _groups("selective_scan_bwd", B, C, 4)

    f32 = _torch().float32
    keep, grads, args, gd, hd, sd, *outs = _describe("selective_scan_bwd", device, (
        ("u", u, 3), ("delta", delta, 3), ("A", A, 2), ("B", Bg, 4), ("C", Cg, 4), ("D", D, 1), ("z", z, 3),
        ("delta_bias", delta_bias, 1), ("h0", h0, 3), ("lengths", lengths, 1, _torch().int32), ("dy", dy, 3),
        ("dh_last", dh_last, 3), ("saved", saved, 1), ("du", None, 3, f32, u), ("ddelta", None, 3, f32, delta),
        ("dA", None, 2, f32, A), ("dB", None, 4, f32, Bg), ("dC", None, 4, f32, Cg), ("dD", None, 1, f32, D),
        ("dz", None, 3, f32, z), ("ddelta_bias", None, 1, f32, delta_bias), ("dh0", None, 3, f32, h0)), table=10)
    if not saved.is_contiguous():
        raise RemoraUnsupportedError("selective_scan_bwd: saved is not what selective_scan_fwd returned")
    to = L.RemoraSelectiveScanGrads(*outs)
    lib, ctx = L.lib(), context(device).ptr
    scratch, at, size = _scratch(lib.remora_b200_selective_scan_bwd_scratch, "selective_scan_bwd", device, ctx, *u.shape,
                                 A.shape[1], Bg.shape[2])
    L.check(lib.remora_b200_selective_scan_bwd(ctx, _spec(_SCAN_SPECS, softplus, True), args, gd, hd, saved.data_ptr(),
                                               4 * saved.numel(), ctypes.addressof(to), at, size, _raw_stream(device)),
            "selective_scan_bwd")
    if B.dim() == 3:
        return (*grads[:3], grads[3].squeeze(2), grads[4].squeeze(2), *grads[5:])
    return grads


def selective_scan_step(state, u, delta, A, B, C, D=None, *, z=None, delta_bias=None, softplus: bool = False,
                        slots=None, out=None, state_out=None):
    """One token per row of u [B, D] (B and C: [B, N] or [B, G, N]): y, with
    the state [S, D, N] moved on in place (or into state_out).  Row i uses
    state row slots[i], or row i without slots; a row whose slot is -1 or was
    named by an earlier row is left out, as in causal_conv_step."""
    device = _cuda_index(u)
    Bg, Cg = _groups("selective_scan_step", B, C, 3)
    torch = _torch()
    if state_out is None:
        state_out = state
    keep, (y, _), args, yd, od = _describe("selective_scan_step", device, (
        ("state", state, 3), ("u", u, 2), ("delta", delta, 2), ("A", A, 2), ("B", Bg, 3), ("C", Cg, 3), ("D", D, 1),
        ("z", z, 2), ("delta_bias", delta_bias, 1), ("slots", slots, 1, torch.int32), ("out", out, 2, torch.float32, u),
        ("state_out", state_out, 3, torch.float32, None)), table=10)
    L.check(L.lib().remora_b200_selective_scan_step(context(device).ptr, _spec(_SCAN_SPECS, softplus, out is None), args,
                                                    yd, od, _raw_stream(device)), "selective_scan_step")
    _binding().written(y, state_out)
    return y
