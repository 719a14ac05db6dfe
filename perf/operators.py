"""The sequence-block operators as they are timed: cases, inputs, plain forms.

Three operators, each for training, for prompts and for single tokens:

* ``norm``: root-mean-square norm of a row, with the residual's addition
  before it and an 8-bit output with scales after it, and its gradients;
* ``conv``: depthwise causal convolution of a few taps along time, with its
  gradients and its single-token form;
* ``scan``: selective state space scan (a gated linear recurrence whose decay,
  input and output weights change from position to position), with its
  gradients and its single-token form.

``run`` computes the plain form, in elementary torch operations, or (with
``own`` true) makes the calls a user makes of ``remora_b200.ops``.  ``exact``
gives the same outputs from the definitions in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

F32 = torch.float32
F64 = torch.float64
E4M3_MAX = 448.0


def _device() -> torch.device:
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


# ------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # one decoding step of four sequences: the norm ahead of an 8-bit
        # product, row scales; a call of a few microseconds
        dict(name="norm_token_e4m3", op="norm", form="quant", rows=4, dim=2048, residual=True, group=0),
        # a prompt's norm, quantised to e4m3 with a scale for every 128 columns
        dict(name="norm_prompt_e4m3", op="norm", form="quant", rows=8192, dim=4096, residual=True, group=128),
        # the norm of a training step over 8 sequences of 2048, both
        # directions, with a gradient that arrives through the residual
        dict(name="norm_train", op="norm", form="train", rows=16384, dim=2048, residual=True),
        # 64 sequences of a server's pool, one token each
        dict(name="conv_token_pool", op="conv", form="step", batch=64, dim=4096, width=4, silu=True, bias=True,
             pool=96),
        # one long prompt that continues an earlier one
        dict(name="conv_prompt", op="conv", form="prompt", batch=1, length=8192, dim=4096, width=4, silu=True,
             bias=True, state=True, ragged=False),
        # a padded batch of short prompts, odd in every size
        dict(name="conv_ragged", op="conv", form="prompt", batch=5, length=777, dim=1001, width=3, silu=True,
             bias=False, state=False, ragged=True),
        # the convolution of a training step, both directions
        dict(name="conv_train", op="conv", form="train", batch=8, length=2048, dim=4096, width=4, silu=True,
             bias=True, state=False, ragged=False),
        # one token of one sequence: launch latency
        dict(name="scan_token", op="scan", form="step", batch=1, dim=2048, states=16, groups=1, gate=True, pool=0),
        # one token for each of 128 sequences: the state's bytes
        dict(name="scan_tokens", op="scan", form="step", batch=128, dim=4096, states=16, groups=1, gate=True, pool=0),
        # a long prompt of one sequence, its state kept for the tokens after it
        dict(name="scan_prompt", op="scan", form="prompt", batch=1, length=4096, dim=2048, states=16, groups=1,
             gate=True, state=True, ragged=False),
        # training on a padded batch with odd sizes and shared groups
        dict(name="scan_train_ragged", op="scan", form="train", batch=3, length=509, dim=388, states=13, groups=2,
             gate=True, state=True, ragged=True),
        # the scan of a training step, both directions
        dict(name="scan_train", op="scan", form="train", batch=4, length=2048, dim=2048, states=16, groups=1,
             gate=True, state=False, ragged=False),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["norm", "conv", "scan"])
    flip = lambda: rng.random() < 0.5  # noqa: E731
    if op == "norm":
        form = rng.choice(["fwd", "quant", "train"])
        dim = _log_int(rng, 64, 8192)
        case = dict(op=op, form=form, rows=_log_int(rng, 1, min(16384, (1 << 25) // dim)), dim=dim, residual=flip())
        if form == "quant":
            group = rng.choice([0, 32, 128])
            if group:
                case["dim"] = max(group, dim // group * group)
            case["group"] = group
        return case
    if op == "conv":
        form = rng.choice(["prompt", "train", "step"])
        dim = _log_int(rng, 64, 4096)
        case = dict(op=op, form=form, dim=dim, width=rng.choice([2, 3, 4]), silu=flip(), bias=flip())
        if form == "step":
            batch = _log_int(rng, 1, 256)
            case.update(batch=batch, pool=batch + rng.randrange(1, 32) if flip() else 0)
            return case
        batch = rng.randrange(1, 9)
        case.update(batch=batch, length=_log_int(rng, 1, min(8192, (1 << 25) // (dim * batch))), state=flip(),
                    ragged=flip())
        return case
    form = rng.choice(["prompt", "train", "step"])
    groups = rng.choice([1, 1, 2])
    dim = _log_int(rng, 64, 2048) // groups * groups
    case = dict(op=op, form=form, dim=dim, states=rng.choice([4, 8, 13, 16, 16, 32]), groups=groups, gate=flip())
    if form == "step":
        batch = _log_int(rng, 1, 256)
        case.update(batch=batch, pool=batch + rng.randrange(1, 32) if flip() else 0)
        return case
    batch = rng.randrange(1, 5)
    cap = (1 << 28) // (dim * batch * case["states"])
    case.update(batch=batch, length=_log_int(rng, 1, min(2048 if form == "train" else 4096, cap)), state=flip(),
                ragged=flip())
    return case


# ------------------------------------------------------------------ inputs
def prepare(case: dict, seed: int) -> dict:
    dev = _device()
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device=dev, dtype=F32).mul_(scale)

    def uniform(lo, hi, *shape):
        return torch.rand(shape, generator=gen, device=dev, dtype=F32).mul_(hi - lo).add_(lo)

    def lengths(batch, length):
        out = torch.randint(0, length + 1, (batch,), generator=gen, device=dev, dtype=torch.int32)
        out[0] = length
        return out

    def slots(batch, pool):
        return torch.randperm(pool, generator=gen, device=dev)[:batch].to(torch.int32)

    s: dict = {"case": dict(case)}
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        s["x"] = normal(rows, dim)
        # a residual stream grows with depth: larger than the block's output
        s["residual"] = normal(rows, dim, scale=3.0) if case["residual"] else None
        s["w"] = normal(dim, scale=0.1).add_(1.0)
        s["eps"] = 1e-5
        if case["form"] == "train":
            s["dy"] = normal(rows, dim)
            s["dsum"] = normal(rows, dim) if case["residual"] else None
        return s
    batch, dim = case["batch"], case["dim"]
    if case["op"] == "conv":
        width = case["width"]
        bound = 1.0 / math.sqrt(width)
        s["w"] = uniform(-bound, bound, dim, width)
        s["bias"] = uniform(-bound, bound, dim) if case["bias"] else None
        if case["form"] == "step":
            pool = case["pool"]
            s["x"] = normal(batch, dim)
            s["state"] = normal(pool or batch, width - 1, dim)
            s["state_out"] = torch.zeros_like(s["state"])
            s["slots"] = slots(batch, pool) if pool else None
            return s
        s["x"] = normal(batch, case["length"], dim)
        s["state"] = normal(batch, width - 1, dim) if case["state"] else None
        s["lengths"] = lengths(batch, case["length"]) if case["ragged"] else None
        if case["form"] == "train":
            s["dy"] = normal(batch, case["length"], dim)
        return s
    states, groups = case["states"], case["groups"]
    # decay rates 1 .. states, as the recurrence is initialised, then trained on
    s["A"] = -torch.exp(torch.log(torch.arange(1, states + 1, device=dev, dtype=F32)) + normal(dim, states, scale=0.1))
    s["D"] = normal(dim, scale=0.1).add_(1.0)
    # step sizes from 0.001 to 0.1 on a logarithmic scale; softplus(bias) gives them
    dt = torch.exp(uniform(math.log(1e-3), math.log(1e-1), dim))
    s["delta_bias"] = dt + torch.log(-torch.expm1(-dt))
    lead = (batch,) if case["form"] == "step" else (batch, case["length"])
    s["u"] = normal(*lead, dim)
    s["delta"] = normal(*lead, dim, scale=0.5)
    s["B"] = normal(*lead, groups, states)
    s["C"] = normal(*lead, groups, states)
    s["z"] = normal(*lead, dim) if case["gate"] else None
    if case["form"] == "step":
        pool = case["pool"]
        s["state"] = normal(pool or batch, dim, states)
        s["state_out"] = torch.zeros_like(s["state"])
        s["slots"] = slots(batch, pool) if pool else None
        return s
    s["h0"] = normal(batch, dim, states) if case["state"] else None
    s["lengths"] = lengths(batch, case["length"]) if case["ragged"] else None
    if case["form"] == "train":
        s["dy"] = normal(*lead, dim)
    return s


# ------------------------------------------------- the framework's own calls
def _run_own(s: dict):
    from remora_b200 import ops

    case = s["case"]
    form = case["form"]
    if case["op"] == "norm":
        if form == "quant":
            return list(ops.rms_norm_quant(s["x"], s["w"], residual=s["residual"], eps=s["eps"],
                                           group=case["group"]))
        out = ops.rms_norm_fwd(s["x"], s["w"], residual=s["residual"], eps=s["eps"])
        y, *total = out if s["residual"] is not None else (out,)
        if form == "fwd":
            return [y, *total]
        normed = total[0] if total else s["x"]
        return [y, *total, *ops.rms_norm_bwd(normed, s["w"], s["dy"], dsum=s["dsum"], eps=s["eps"])]
    if case["op"] == "conv":
        if form == "step":
            y = ops.causal_conv_step(s["x"], s["state"], s["w"], s["bias"], silu=case["silu"], slots=s["slots"],
                                     state_out=s["state_out"])
            return [y, s["state_out"]]
        if form == "prompt":
            return list(ops.causal_conv_fwd(s["x"], s["w"], s["bias"], state=s["state"], lengths=s["lengths"],
                                            silu=case["silu"], return_state=True))
        y = ops.causal_conv_fwd(s["x"], s["w"], s["bias"], state=s["state"], lengths=s["lengths"], silu=case["silu"])
        grads = ops.causal_conv_bwd(s["x"], s["w"], s["dy"], s["bias"], state=s["state"], lengths=s["lengths"],
                                    silu=case["silu"])
        return [y, *(g for g in grads if g is not None)]
    if form == "step":
        y = ops.selective_scan_step(s["state"], s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], z=s["z"],
                                    delta_bias=s["delta_bias"], softplus=True, slots=s["slots"],
                                    state_out=s["state_out"])
        return [y, s["state_out"]]
    common = dict(z=s["z"], delta_bias=s["delta_bias"], softplus=True, h0=s["h0"], lengths=s["lengths"])
    if form == "prompt":
        return list(ops.selective_scan_fwd(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], return_state=True,
                                           **common))
    y, saved = ops.selective_scan_fwd(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], save=True, **common)
    grads = ops.selective_scan_bwd(s["u"], s["delta"], s["A"], s["B"], s["C"], s["dy"], saved, s["D"], **common)
    return [y, *(g for g in grads if g is not None)]


# ------------------------------------------------------------- plain forms
def _plain_norm(s: dict):
    case = s["case"]
    x, w, eps = s["x"], s["w"], s["eps"]
    total = x if s["residual"] is None else x + s["residual"]
    dim = x.shape[1]
    if case["form"] == "quant":
        # in 64 bits: the nearest of the 8-bit values depends on the last bits
        t = total.to(F64)
        y = t / torch.sqrt((t * t).mean(dim=1, keepdim=True) + eps) * w.to(F64)
        width = case["group"] or dim
        yg = y.view(-1, dim // width, width)
        scales = (yg.abs().amax(dim=2) / E4M3_MAX).clamp_min(2.0 ** -126).to(F32)
        q = (yg / scales.to(F64).unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX)
        out = [q.to(F32).to(torch.float8_e4m3fn).view(-1, dim), scales]
        return out if s["residual"] is None else [*out, total]
    rstd = torch.rsqrt((total * total).mean(dim=1, keepdim=True) + eps)
    xhat = total * rstd
    y = xhat * w
    out = [y] if s["residual"] is None else [y, total]
    if case["form"] == "fwd":
        return out
    wdy = s["dy"] * w
    dx = rstd * (wdy - xhat * (wdy * xhat).mean(dim=1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"]
    return [*out, dx, (s["dy"] * xhat).sum(dim=0)]


def _valid(lengths, batch: int, length: int, device):
    """[batch, length, 1] truth values: the position is inside its sequence."""
    if lengths is None:
        return torch.ones(batch, length, 1, dtype=torch.bool, device=device)
    return (torch.arange(length, device=device)[None, :] < lengths[:, None].to(torch.int64)).unsqueeze(-1)


def _plain_conv_step(s: dict):
    case = s["case"]
    rows = torch.arange(case["batch"], device=s["x"].device) if s["slots"] is None else s["slots"].to(torch.int64)
    window = torch.cat([s["state"][rows], s["x"][:, None, :]], dim=1)  # [batch, width, dim]
    pre = (window * s["w"].t()).sum(dim=1)
    if s["bias"] is not None:
        pre = pre + s["bias"]
    y = pre * torch.sigmoid(pre) if case["silu"] else pre
    s["state_out"][rows] = window[:, 1:]
    return [y, s["state_out"]]


def _plain_conv(s: dict):
    case = s["case"]
    x, w, width = s["x"], s["w"], case["width"]
    batch, length, dim = x.shape
    valid = _valid(s["lengths"], batch, length, x.device)
    before = s["state"] if s["state"] is not None else x.new_zeros(batch, width - 1, dim)
    xs = torch.cat([before, torch.where(valid, x, 0.0)], dim=1)
    pre = sum(xs[:, k:k + length] * w[:, k] for k in range(width))
    if s["bias"] is not None:
        pre = pre + s["bias"]
    sig = torch.sigmoid(pre)
    y = torch.where(valid, pre * sig if case["silu"] else pre, 0.0)
    if case["form"] == "prompt":
        ends = torch.full((batch,), length, device=x.device) if s["lengths"] is None else s["lengths"].to(torch.int64)
        rows = ends[:, None] + torch.arange(width - 1, device=x.device)
        return [y, xs.gather(1, rows[:, :, None].expand(-1, -1, dim))]
    g = torch.where(valid, s["dy"], 0.0)
    if case["silu"]:
        g = g * (sig * (1.0 + pre * (1.0 - sig)))
    dxs = torch.zeros_like(xs)
    for k in range(width):
        dxs[:, k:k + length] += g * w[:, k]
    dw = torch.stack([(g * xs[:, k:k + length]).sum(dim=(0, 1)) for k in range(width)], dim=1)
    grads = [torch.where(valid, dxs[:, width - 1:], 0.0), dw]
    if s["bias"] is not None:
        grads.append(g.sum(dim=(0, 1)))
    if s["state"] is not None:
        grads.append(dxs[:, :width - 1].contiguous())
    return [y, *grads]


def _softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))


def _per_channel(t: torch.Tensor, dim: int) -> torch.Tensor:
    """Group rows [..., groups, states] as seen by every channel of the group."""
    return t.repeat_interleave(dim // t.shape[-2], dim=-2)


def _plain_scan_step(s: dict):
    case = s["case"]
    dim = case["dim"]
    rows = torch.arange(case["batch"], device=s["u"].device) if s["slots"] is None else s["slots"].to(torch.int64)
    dt = _softplus(s["delta"] + s["delta_bias"])
    h = torch.exp(dt.unsqueeze(-1) * s["A"]) * s["state"][rows]
    h = h + (dt * s["u"]).unsqueeze(-1) * _per_channel(s["B"], dim)
    y = (h * _per_channel(s["C"], dim)).sum(dim=-1) + s["D"] * s["u"]
    if s["z"] is not None:
        y = y * (s["z"] * torch.sigmoid(s["z"]))
    s["state_out"][rows] = h
    return [y, s["state_out"]]


def _recurrence(decay: torch.Tensor, term: torch.Tensor) -> torch.Tensor:
    """h[:, t] = decay[:, t] * h[:, t - 1] + term[:, t], by doubling: after k
    rounds position t holds the recurrence over the 2^k positions ending at it."""
    length, reach = decay.shape[1], 1
    while reach < length:
        term = torch.cat([term[:, :reach], term[:, reach:] + decay[:, reach:] * term[:, :-reach]], dim=1)
        decay = torch.cat([decay[:, :reach], decay[:, reach:] * decay[:, :-reach]], dim=1)
        reach *= 2
    return term


def _plain_scan(s: dict):
    case = s["case"]
    u, A = s["u"], s["A"]
    batch, length, dim = u.shape
    states, groups = case["states"], case["groups"]
    valid = _valid(s["lengths"], batch, length, u.device)
    raw = s["delta"] + s["delta_bias"]
    dt = torch.where(valid, _softplus(raw), 0.0)  # a step of zero keeps the state
    uv = torch.where(valid, u, 0.0)
    Bc = _per_channel(torch.where(valid.unsqueeze(-1), s["B"], 0.0), dim)
    Cc = _per_channel(torch.where(valid.unsqueeze(-1), s["C"], 0.0), dim)
    decay = torch.exp(dt.unsqueeze(-1) * A)
    term = (dt * uv).unsqueeze(-1) * Bc
    first = s["h0"] if s["h0"] is not None else u.new_zeros(batch, dim, states)
    term[:, 0] += decay[:, 0] * first
    h = _recurrence(decay, term)
    ypre = (h * Cc).sum(dim=-1) + s["D"] * uv
    sig = torch.sigmoid(s["z"]) if s["z"] is not None else None
    y = torch.where(valid, ypre if sig is None else ypre * (s["z"] * sig), 0.0)
    if case["form"] == "prompt":
        return [y, h[:, -1].contiguous()]
    dy = torch.where(valid, s["dy"], 0.0)
    dyp = dy if sig is None else dy * (s["z"] * sig)
    dz = None if sig is None else torch.where(valid, dy * ypre * (sig * (1.0 + s["z"] * (1.0 - sig))), 0.0)
    # the adjoint of h runs from the last position to the first
    later = torch.cat([decay[:, 1:], torch.ones_like(decay[:, :1])], dim=1)
    g = _recurrence(later.flip(1), (Cc * dyp.unsqueeze(-1)).flip(1)).flip(1)
    dC = (h * dyp.unsqueeze(-1)).view(batch, length, groups, -1, states).sum(dim=3)
    dB = (g * (dt * uv).unsqueeze(-1)).view(batch, length, groups, -1, states).sum(dim=3)
    gah = g * decay * torch.cat([first.unsqueeze(1), h[:, :-1]], dim=1)
    gB = (g * Bc).sum(dim=-1)
    du = torch.where(valid, dt * gB + s["D"] * dyp, 0.0)
    ddelta = torch.where(valid, ((gah * A).sum(dim=-1) + uv * gB) * torch.sigmoid(raw), 0.0)
    grads = [du, ddelta, (gah * dt.unsqueeze(-1)).sum(dim=(0, 1)), dB, dC, (dyp * uv).sum(dim=(0, 1)), dz,
             ddelta.sum(dim=(0, 1)), decay[:, 0] * g[:, 0] if s["h0"] is not None else None]
    return [y, *(t for t in grads if t is not None)]


def run(state: dict):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "norm":
        return _plain_norm(state)
    if case["op"] == "conv":
        return _plain_conv_step(state) if case["form"] == "step" else _plain_conv(state)
    return _plain_scan_step(state) if case["form"] == "step" else _plain_scan(state)


# --------------------------------------------------------- exact, in 64 bits
def _round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest value with 3 fraction bits and exponents from -6 (ties to even)."""
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -20))).clamp(-6, 8)
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_norm(s: dict):
    case = s["case"]

    def norm(x, residual, w):
        total = x if residual is None else x + residual
        return total * torch.pow(torch.sum(total ** 2, dim=-1, keepdim=True) / total.shape[-1] + s["eps"], -0.5) * w

    x, w = s["x"].to(F64), s["w"].to(F64)
    residual = None if s["residual"] is None else s["residual"].to(F64)
    total = x if residual is None else x + residual
    if case["form"] == "quant":
        y = norm(x, residual, w)
        width = case["group"] or case["dim"]
        groups = y.reshape(y.shape[0], -1, width)
        scales = torch.clamp(groups.abs().max(dim=-1).values / E4M3_MAX, min=2.0 ** -126)
        out = [_round_e4m3(groups / scales[..., None]).reshape(y.shape), scales]
        return out if residual is None else [*out, total]
    if case["form"] == "fwd":
        return [norm(x, residual, w)] if residual is None else [norm(x, residual, w), total]
    # the gradients by differentiating the definition
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = norm(x, residual, w)
    loss = (y * s["dy"].to(F64)).sum()
    if s["dsum"] is not None:
        loss = loss + ((x + residual) * s["dsum"].to(F64)).sum()
    dx, dw = torch.autograd.grad(loss, [x, w])
    return [y.detach(), dx, dw] if residual is None else [y.detach(), total.detach(), dx, dw]


def _exact_silu(v):
    return v / (1.0 + torch.exp(-v))


def _exact_conv_step(s: dict):
    case = s["case"]
    x, state, w = s["x"].to(F64), s["state"].to(F64), s["w"].to(F64)
    index = list(range(case["batch"])) if s["slots"] is None else s["slots"].tolist()
    out = torch.zeros_like(state)
    state = state[index]
    pre = x * w[:, -1]
    for k in range(case["width"] - 1):
        pre = pre + state[:, k] * w[:, k]
    if s["bias"] is not None:
        pre = pre + s["bias"].to(F64)
    if case["width"] > 2:
        out[index, :-1] = state[:, 1:]
    out[index, -1] = x
    return [_exact_silu(pre) if case["silu"] else pre, out]


def _exact_conv(s: dict):
    case = s["case"]
    width, length = case["width"], case["length"]
    train = case["form"] == "train"
    x, w = s["x"].to(F64), s["w"].to(F64)
    bias = None if s["bias"] is None else s["bias"].to(F64)
    state = None if s["state"] is None else s["state"].to(F64)
    ends = [length] * case["batch"] if s["lengths"] is None else s["lengths"].tolist()
    leaves = [t.requires_grad_(train) for t in (x, w, bias, state) if t is not None]
    y = torch.zeros_like(x)
    lasts, loss = [], 0.0
    for b, n in enumerate(ends):
        rows = x[b, :n]
        head = state[b] if state is not None else rows.new_zeros(width - 1, case["dim"])
        ext = torch.cat([head, rows])
        lasts.append(ext[n:].detach())
        if n == 0:
            continue
        # one filter per channel over that channel's row of values
        pre = (ext.unfold(0, width, 1) * w).sum(dim=-1)
        if bias is not None:
            pre = pre + bias
        out = _exact_silu(pre) if case["silu"] else pre
        y[b, :n] = out.detach()
        if train:
            loss = loss + (out * s["dy"][b, :n].to(F64)).sum()
    if not train:
        return [y, torch.stack(lasts)]
    grads = torch.autograd.grad(loss, leaves, allow_unused=True)
    return [y.detach(), *(torch.zeros_like(t) if g is None else g for g, t in zip(grads, leaves))]


def _exact_scan_step(s: dict):
    case = s["case"]
    index = list(range(case["batch"])) if s["slots"] is None else s["slots"].tolist()
    u, z = s["u"].to(F64), s["z"]
    dt = torch.logaddexp(s["delta"].to(F64) + s["delta_bias"].to(F64), torch.zeros((), dtype=F64, device=u.device))
    group = torch.arange(case["dim"], device=u.device) // (case["dim"] // case["groups"])
    Bx, Cx = s["B"].to(F64)[:, group], s["C"].to(F64)[:, group]
    decay = torch.exp(torch.einsum("bd,dn->bdn", dt, s["A"].to(F64)))
    h = torch.einsum("bdn,bdn->bdn", decay, s["state"].to(F64)[index])
    h = h + torch.einsum("bd,bd,bdn->bdn", dt, u, Bx)
    y = torch.einsum("bdn,bdn->bd", h, Cx) + u * s["D"].to(F64)
    if z is not None:
        y = y * _exact_silu(z.to(F64))
    out = torch.zeros_like(s["state"], dtype=F64)
    out[index] = h
    return [y, out]


def _exact_scan(s: dict):
    """Position by position; the gradients by differentiating that."""
    case = s["case"]
    train = case["form"] == "train"
    length, dim, batch = case["length"], case["dim"], case["batch"]
    ends = [length] * batch if s["lengths"] is None else s["lengths"].tolist()
    group = torch.arange(dim, device=s["u"].device) // (dim // case["groups"])
    names = ["u", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0"]
    v = {k: s[k].to(F64).requires_grad_(train) for k in names if s[k] is not None}
    y = torch.zeros_like(s["u"], dtype=F64)
    lasts, grads = [], {k: torch.zeros_like(t) for k, t in v.items()}
    zero = torch.zeros((), dtype=F64, device=y.device)
    for b, n in enumerate(ends):
        h = v["h0"][b] if "h0" in v else torch.zeros(dim, case["states"], dtype=F64, device=y.device)
        rows = []
        for u, delta, Bt, Ct in zip(*(v[k][b, :n].unbind(0) for k in ("u", "delta", "B", "C"))):
            dt = torch.logaddexp(delta + v["delta_bias"], zero)
            h = torch.exp(dt[:, None] * v["A"]) * h + (dt * u)[:, None] * Bt[group]
            rows.append((h * Ct[group]).sum(dim=1) + v["D"] * u)
        lasts.append(h.detach())
        if n == 0:
            continue
        out = torch.stack(rows)
        if "z" in v:
            out = out * _exact_silu(v["z"][b, :n])
        y[b, :n] = out.detach()
        if train:
            loss = (out * s["dy"][b, :n].to(F64)).sum()
            for k, part in zip(v, torch.autograd.grad(loss, list(v.values()), allow_unused=True)):
                if part is not None:  # one position ahead of no state: no decay was used
                    grads[k] += part
    return [y, *grads.values()] if train else [y, torch.stack(lasts)]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "conv":
        return _exact_conv_step(s) if case["form"] == "step" else _exact_conv(s)
    return _exact_scan_step(s) if case["form"] == "step" else _exact_scan(s)


# -------------------------------------------------------------- work, floor
def work(case: dict) -> dict:
    """Bytes: every input once, every output once.  Operations: a product, a
    sum or an exponential counts one."""
    if case["op"] == "norm":
        n, dim = case["rows"] * case["dim"], case["dim"]
        reads, writes = n + dim, n
        if case["residual"]:
            reads, writes = reads + n, writes + n
        flops = 5 * n
        if case["form"] == "quant":
            groups = case["rows"] * (dim // (case["group"] or dim))
            return {"bytes": 4 * reads + 4 * (writes - n) + n + 4 * groups, "flops": 8 * n}
        if case["form"] == "train":
            reads, writes = reads + n * (2 if case["residual"] else 1), writes + n + dim
            flops += 10 * n
        return {"bytes": 4 * (reads + writes), "flops": flops}
    batch, dim = case["batch"], case["dim"]
    if case["op"] == "conv":
        width = case["width"]
        params = dim * width + (dim if case["bias"] else 0)
        state = batch * (width - 1) * dim
        act = 4 if case["silu"] else 0
        if case["form"] == "step":
            return {"bytes": 4 * (2 * batch * dim + params + 2 * state), "flops": batch * dim * (2 * width + act)}
        n = batch * case["length"] * dim
        if case["form"] == "prompt":
            return {"bytes": 4 * (2 * n + params + (2 if case["state"] else 1) * state),
                    "flops": n * (2 * width + act)}
        return {"bytes": 4 * (4 * n + 2 * params + (2 * state if case["state"] else 0)),
                "flops": n * (6 * width + 4 * act)}
    states, groups = case["states"], case["groups"]
    params = dim * (states + 2)
    hidden = batch * dim * states
    gate = 1 if case["gate"] else 0
    if case["form"] == "step":
        return {"bytes": 4 * ((3 + gate) * batch * dim + 2 * batch * groups * states + params + 2 * hidden),
                "flops": 7 * hidden + 10 * batch * dim}
    positions = batch * case["length"]
    n, bc = positions * dim, 2 * positions * groups * states
    if case["form"] == "prompt":
        return {"bytes": 4 * ((3 + gate) * n + bc + params + (2 if case["state"] else 1) * hidden),
                "flops": n * (7 * states + 10)}
    return {"bytes": 4 * ((6 + 2 * gate) * n + 2 * bc + 2 * params + (2 * hidden if case["state"] else 0)),
            "flops": n * (24 * states + 40)}
