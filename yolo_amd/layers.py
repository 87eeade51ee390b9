"""Layers of a residual block on the gfx950 HIP library, beside the convolutions and the batch norm that
yolo_v3 runs: a matrix product with bias, activation and residual in its epilogue, and the norms after and
before a block fused with the block's gate, residual scale and residual add.

    stream, normed = block_norm(x, before_weight=w0)                 # enter the first block
    up = linear(normed, w1, b1, activation="gelu_tanh")
    out = linear(up, w2, b2)
    stream, normed = block_norm(out, stream, after_weight=w3, gate=g, before_weight=w4)    # on to the next

Both are differentiable in every tensor argument (once; a second derivative raises), take inputs on any GPU and
run on torch's current stream of that GPU.  They allocate outputs and scratch with torch's allocator, so they
can be captured into a HIP graph, keep nothing between calls and never synchronise.  (As anywhere in torch, a
backward pass is captured only while no eager graph of the same leaves is alive.)  Forward-mode derivatives and
traces (torch.jit.trace, make_fx) are refused.  Results depend on the inputs alone: every sum has a fixed order.  Row views (``x[:, :k]``) are read in place; other strides are copied.
There is no CPU implementation: tensors on the CPU raise YoloAmdError.

The reference has no counterpart of either.
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib
from ._lib import BlockNormBackwardDesc, BlockNormDesc, LinearBackwardDesc, LinearDesc, YoloAmdError, check, lib

# A call's own work on the host is what bounds it at few rows: descriptors are filled in one constructor call, the
# stream is asked for as a number, nothing is looked up twice.
_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
_F32 = torch.float32
_empty_like = torch.empty_like
_current_device = torch.cuda.current_device


def _raw_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


_is_tracing = torch._C._is_tracing
_dispatch_modes = torch._C._len_torch_dispatch_stack


def _refuse_transforms(what, tensors):
    """The kernels write through pointers, which torch does not see: a tangent would be dropped (a derivative of zero) and
    a trace would hold the outputs' allocation alone, or calls without the checks of what they are given."""
    if _forward_ad._current_level >= 0 and any(
            t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: there is no forward-mode derivative (an argument has a tangent)")
    if _is_tracing() or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise YoloAmdError(f"{what}: cannot be recorded in a trace (torch.jit.trace, make_fx): the kernels are not torch operators")


def _on_gpu(what, **tensors):
    """Every argument is a tensor (or None) on one GPU, the first one's.  Returns its index."""
    index = None
    if _forward_ad._current_level >= 0 or _is_tracing() or _dispatch_modes():
        _refuse_transforms(what, [t for t in tensors.values() if torch.is_tensor(t)])
    for name, t in tensors.items():
        if t is None:
            continue
        if not torch.is_tensor(t):
            raise TypeError(f"{what}: {name} is not a torch tensor but {type(t).__name__}")
        i = t.get_device() if t.is_cuda else -1
        if index is None:
            index = i
            if i < 0:
                raise YoloAmdError(f"{what}: {name} is on the CPU; this path runs on the GPU only")
        elif i != index:
            raise YoloAmdError(f"{what}: {name} is on {t.device}, the first argument on cuda:{index}")
    return index


def _rows(t):
    """(tensor, row stride): ``t`` as rows of its last dimension at one stride, copied where its strides do not
    allow that."""
    shape = t.shape
    if t.is_contiguous():
        return t, shape[-1]
    if shape[-1] == 1 or t.stride(-1) == 1:
        step = rows = 0                              # dimensions of size 1 have no stride to speak of
        for i in range(t.dim() - 2, -1, -1):
            if shape[i] == 1:
                continue
            if rows == 0:
                step = t.stride(i)
                rows = 1
            elif t.stride(i) != step * rows:
                break
            rows *= shape[i]
        else:
            if step >= shape[-1]:
                return t, step
    t = t.contiguous()
    return t, shape[-1]


def _call(index, fn, desc, what):
    """Run ``fn(desc, current stream)`` on GPU ``index``."""
    if index == _current_device():
        rc = fn(desc, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(desc, _raw_stream(index))
    if rc:
        check(rc, what)


def _like(t):
    """An uninitialised contiguous tensor of t's shape and type, on its GPU (in half the time torch.empty takes)."""
    return _empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _scratch(desc, nbytes, like):
    """Scratch of one call.  Taken from torch's allocator each time: calls on different streams, or in different
    captured graphs, never share it."""
    ws = like.new_empty(nbytes, dtype=torch.uint8)
    desc.workspace, desc.workspace_bytes = ws.data_ptr(), nbytes
    return ws


# --------------------------------------------------------------------------
# linear
# --------------------------------------------------------------------------
def _linear_forward(x, weight, bias, residual, act, out_dtype, keep_pre):
    """Returns (y, pre or None)."""
    n, k = weight.shape
    dt = x.dtype
    x, ldx = _rows(x)
    weight, ldw = _rows(weight)
    shape = x.shape[:-1] + (n,)
    m = x.numel() // k if k else shape.numel() // n if n else 0
    y = x.new_empty(shape) if out_dtype is dt else x.new_empty(shape, dtype=out_dtype)
    b = r = p = ldr = 0
    b32 = r32 = False
    pre = None
    if bias is not None:
        bias = bias.contiguous()
        b, b32 = bias.data_ptr(), bias.dtype is _F32
    if residual is not None:
        residual, ldr = _rows(residual)
        r, r32 = residual.data_ptr(), residual.dtype is _F32
    if keep_pre:
        pre = x.new_empty(shape, dtype=_F32)
        p = pre.data_ptr()
    d = LinearDesc(x.data_ptr(), weight.data_ptr(), b, r, y.data_ptr(), p, m, n, k, ldx, ldw, ldr, n, _TYPES[dt], b32, r32,
                   out_dtype is _F32, act, True)
    nbytes = lib.yolo_amd_linear_workspace_bytes(d)
    ws = _scratch(d, nbytes, y) if nbytes else None      # noqa: F841  (alive over the call)
    _call(x.get_device(), lib.yolo_amd_linear_forward, d, "linear")
    return y, pre


def _linear_backward(ctx, dy):
    if _forward_ad._current_level >= 0 or _is_tracing() or _dispatch_modes():
        _refuse_transforms("linear backward", (dy,))
    need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    act, x_shape, w_shape, dt, b_dtype, r_dtype = ctx.conf
    dres = (dy if dy.dtype is r_dtype else dy.to(r_dtype)) if need_r else None
    if not (need_x or need_w or need_b):
        return None, None, None, dres, None, None
    x, weight, pre = ctx.saved_tensors
    n, k = w_shape
    dyr, lddy = _rows(dy)
    m = dy.numel() // n if n else x_shape[:-1].numel()
    xp = wp = dxp = dwp = dbp = ldx = ldw = 0
    dx = dw = db = None
    if need_x:
        weight, ldw = _rows(weight)
        dx = weight.new_empty(x_shape)
        wp, dxp = weight.data_ptr(), dx.data_ptr()
    if need_w:
        x, ldx = _rows(x)
        dw = x.new_empty(w_shape)
        xp, dwp = x.data_ptr(), dw.data_ptr()
    if need_b:
        db = dy.new_empty(n, dtype=b_dtype)
        dbp = db.data_ptr()
    d = LinearBackwardDesc(dyr.data_ptr(), xp, wp, 0 if pre is None else pre.data_ptr(), dxp, dwp, dbp, m, n, k, lddy, ldx,
                           ldw, _TYPES[dt], dy.dtype is _F32, b_dtype is _F32, act, True)
    nbytes = lib.yolo_amd_linear_backward_workspace_bytes(d)
    ws = _scratch(d, nbytes, dy) if nbytes else None      # noqa: F841
    _call(dy.get_device(), lib.yolo_amd_linear_backward, d, "linear backward")
    return dx, dw, db, dres, None, None


_linear_backward_once = torch.autograd.function.once_differentiable(_linear_backward)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_dtype):
        need = ctx.needs_input_grad
        y, pre = _linear_forward(x, weight, bias, residual, act, out_dtype, act != 0 and (need[0] or need[1] or need[2]))
        ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, pre)
        ctx.conf = (act, x.shape, weight.shape, x.dtype, None if bias is None else bias.dtype,
                    None if residual is None else residual.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        # (the wrapper that refuses a second derivative costs as much as a launch: only where one could follow)
        return (_linear_backward_once if torch.is_grad_enabled() else _linear_backward)(ctx, dy)


def linear(x, weight, bias=None, *, activation=None, residual=None, out_dtype=None):
    """``act(x @ weight.T + bias) + residual`` in one launch; a second one where few output tiles
    share a long reduction, and one ahead of it where rows of x or weight do not start on 16-byte boundaries or are
    no whole multiples of 8 values (they are copied).

    x (..., K) and weight (N, K): bf16 or fp16, the same.  bias (N,): that type or fp32.  residual (..., N), the
    shape of the result: that type or fp32.  activation: None, "leaky" (slope 0.1), "relu", "gelu" (erf),
    "gelu_tanh" or "silu".  The result has ``out_dtype`` (x's type by default, or torch.float32).

    Sums are fp32; the result is rounded once, and so is each gradient.  Where a gradient of x, weight or bias will be
    wanted and there is an activation, ``x @ weight.T + bias`` is kept in fp32 for the backward pass; the products of the
    gradients of x and weight take d(loss)/d(pre-activation) in two parts of x's type where one does not hold it."""
    _on_gpu("linear", x=x, weight=weight, bias=bias, residual=residual)
    dt = x.dtype
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise TypeError(f"linear: x must be bfloat16 or float16, got {dt}")
    if weight.dtype != dt:
        raise TypeError(f"linear: weight is {weight.dtype}, x is {dt}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not go together")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.dtype not in (dt, _F32)):
        raise ValueError(f"linear: bias must be ({weight.shape[0]},) of {dt} or float32, got {tuple(bias.shape)} of {bias.dtype}")
    if residual is not None and (residual.shape != x.shape[:-1] + weight.shape[:1] or residual.dtype not in (dt, _F32)):
        raise ValueError(f"linear: residual must be {tuple(x.shape[:-1] + weight.shape[:1])} of {dt} or float32, got "
                         f"{tuple(residual.shape)} of {residual.dtype}")
    if activation not in _lib.ACT_CODES:
        raise ValueError(f"linear: unknown activation {activation!r}")
    if out_dtype is None:
        out_dtype = dt
    elif out_dtype not in (dt, _F32):
        raise TypeError(f"linear: out_dtype must be {dt} or float32, got {out_dtype}")
    act = _lib.ACT_CODES[activation]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act, out_dtype)
    return _linear_forward(x, weight, bias, residual, act, out_dtype, False)[0]


# --------------------------------------------------------------------------
# block_norm
# --------------------------------------------------------------------------
def _norm_desc(x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf, stream, normed):
    """(descriptor, tensors to keep alive over the call)."""
    norm, after, before, scale, eps, rows_per_gate = conf
    dt = x.dtype
    dim = x.shape[-1]
    x, ldx = _rows(x)
    r = g = aw = ab = bw = bb = ldr = 0
    g32 = a32 = b32 = False
    r32 = dt is _F32
    if residual is not None:
        residual, ldr = _rows(residual)
        r, r32 = residual.data_ptr(), residual.dtype is _F32
    if gate is not None:
        gate = gate.contiguous()
        g, g32 = gate.data_ptr(), gate.dtype is _F32
    if after_weight is not None:
        after_weight = after_weight.contiguous()
        aw, a32 = after_weight.data_ptr(), after_weight.dtype is _F32
    if after_bias is not None:
        after_bias = after_bias.contiguous()
        ab, a32 = after_bias.data_ptr(), after_bias.dtype is _F32
    if before_weight is not None:
        before_weight = before_weight.contiguous()
        bw, b32 = before_weight.data_ptr(), before_weight.dtype is _F32
    if before_bias is not None:
        before_bias = before_bias.contiguous()
        bb, b32 = before_bias.data_ptr(), before_bias.dtype is _F32
    d = BlockNormDesc(x.data_ptr(), r, g, aw, ab, bw, bb, stream, normed, x.numel() // dim, dim, ldx, ldr, rows_per_gate,
                      _TYPES[dt], norm, after, before, r32, g32, a32, b32, eps, scale)
    return d, (x, residual, gate, after_weight, after_bias, before_weight, before_bias)


def _norm_forward(x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf, own_stream):
    """(stream or None where it is x itself, normed or None)."""
    stream = normed = None
    s = n = 0
    if own_stream:
        stream = _like(x if residual is None else residual)
        s = stream.data_ptr()
    if conf[2]:
        normed = _like(x)
        n = normed.data_ptr()
    d, keep = _norm_desc(x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf, s, n)
    _call(x.get_device(), lib.yolo_amd_block_norm_forward, d, "block_norm")
    return stream, normed


def _norm_backward(ctx, dstream, dnormed):
    if _forward_ad._current_level >= 0 or _is_tracing() or _dispatch_modes():
        _refuse_transforms("block_norm backward", (dstream, dnormed))
    tensors = ctx.saved_tensors
    d, keep = _norm_desc(*tensors, ctx.conf, 0, 0)
    ds = dn = 0
    if dnormed is not None:
        dnormed = dnormed.contiguous()
        dn = dnormed.data_ptr()
    if dstream is not None:
        dstream = dstream.contiguous()
        ds = dstream.data_ptr()
    grads = [_like(t) if need else None for t, need in zip(tensors, ctx.needs_input_grad)]
    if grads[2] is not None and tensors[0].numel() == 0:         # no row has a share in a gate's row
        grads[2].zero_()
    b = BlockNormBackwardDesc(d, dn, ds, *[0 if g is None else g.data_ptr() for g in grads])
    nbytes = lib.yolo_amd_block_norm_backward_workspace_bytes(b)
    ws = _scratch(b, nbytes, tensors[0]) if nbytes else None     # noqa: F841
    _call(tensors[0].get_device(), lib.yolo_amd_block_norm_backward, b, "block_norm backward")
    return (*grads, None, None)


_norm_backward_once = torch.autograd.function.once_differentiable(_norm_backward)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf, own_stream):
        out = _norm_forward(x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf, own_stream)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, residual, gate, after_weight, after_bias, before_weight, before_bias)
        ctx.conf = conf
        return out

    @staticmethod
    def backward(ctx, dstream, dnormed):
        return (_norm_backward_once if torch.is_grad_enabled() else _norm_backward)(ctx, dstream, dnormed)


def _gate_rows(x, gate):
    """Rows of x that share a row of the gate."""
    dim, lead = x.shape[-1], x.shape[:-1]
    rows = lead.numel()
    if gate.dim() > x.dim() or gate.dim() < 1 or gate.shape[-1] != dim:
        raise ValueError(f"block_norm: gate {tuple(gate.shape)} does not go with x {tuple(x.shape)}")
    g = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape[:-1])
    shared = 1
    i = len(g)
    while i > 0 and g[i - 1] == 1:               # trailing dimensions it does not have: the rows that share it
        shared *= lead[i - 1]
        i -= 1
    if tuple(g[:i]) != tuple(lead[:i]):
        raise ValueError(f"block_norm: gate {tuple(gate.shape)} does not go with x {tuple(x.shape)}: one gate for all "
                         f"rows, for each row, or for each run of rows (a sequence) is taken")
    return max(1, shared if i else rows)


def _check_norm(name, there, w, b, norm, x):
    for kind, t in (("weight", w), ("bias", b)):
        if t is None:
            continue
        if not there:
            raise ValueError(f"block_norm: {name}_{kind} without the norm it belongs to")
        if t.shape != x.shape[-1:] or (t.dtype is not x.dtype and t.dtype is not _F32):
            raise ValueError(f"block_norm: {name}_{kind} must be ({x.shape[-1]},) of {x.dtype} or float32, got "
                             f"{tuple(t.shape)} of {t.dtype}")
    if b is not None:
        if norm == "rms":
            raise ValueError("block_norm: an rms norm has no bias")
        if w is not None and w.dtype is not b.dtype:
            raise ValueError(f"block_norm: {name}_weight is {w.dtype}, {name}_bias is {b.dtype}")


def block_norm(x, residual=None, *, norm="rms", after=None, after_weight=None, after_bias=None, gate=None,
               residual_scale=1.0, before=True, before_weight=None, before_bias=None, eps=1e-6):
    """What lies between two blocks of a residual network, in one launch:

        p      = norm(x) * after_weight + after_bias    (``after``; x itself without it)
        stream = residual + residual_scale * gate * p
        normed = norm(stream) * before_weight + before_bias    (``before``)

    Returns (stream, normed); normed is None without ``before``.

    x (..., D): the block's output, fp32, bf16 or fp16, D up to 16384; normed has its type.  residual: the residual
    stream, x's shape, x's type or fp32; stream has its type.  Without residual it counts as zero, and if there is
    no ``after``, no gate and residual_scale is 1 as well, stream is x itself.  norm: "rms", v / sqrt(mean(v^2) +
    eps), which has no biases, or "layer".  after: True or False; None means: if after_weight or after_bias is given.
    gate: (D,), (B, 1, ..., D) or x's shape -- one for all rows, one for each run of rows, one for each row.
    Weights, biases and gate are of x's type or fp32 (weight and bias of one norm the same).

    Statistics are fp32; normed is taken from the stream before that is rounded.  The backward pass recomputes
    everything from x and residual (neither may be changed in place before it) and no statistics are kept."""
    _on_gpu("block_norm", x=x, residual=residual, gate=gate, after_weight=after_weight, after_bias=after_bias,
            before_weight=before_weight, before_bias=before_bias)
    dt = x.dtype
    if dt not in _TYPES:
        raise TypeError(f"block_norm: x must be float32, bfloat16 or float16, got {dt}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"block_norm: x {tuple(x.shape)} has no rows of values")
    if norm not in _lib.NORM_CODES:
        raise ValueError(f"block_norm: unknown norm {norm!r}")
    if after is None:
        after = after_weight is not None or after_bias is not None
    _check_norm("after", after, after_weight, after_bias, norm, x)
    _check_norm("before", before, before_weight, before_bias, norm, x)
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (dt, _F32)):
        raise ValueError(f"block_norm: residual must be {tuple(x.shape)} of {dt} or float32, got {tuple(residual.shape)} "
                         f"of {residual.dtype}")
    if gate is not None and gate.dtype not in (dt, _F32):
        raise TypeError(f"block_norm: gate must be {dt} or float32, got {gate.dtype}")
    if torch.is_tensor(residual_scale) or torch.is_tensor(eps):
        raise TypeError("block_norm: residual_scale and eps are numbers (reading one from a tensor would wait for the GPU); a "
                        "learned scale goes in as the gate")
    rows_per_gate = _gate_rows(x, gate) if gate is not None else 1
    scale = float(residual_scale)
    conf = (_lib.NORM_CODES[norm], bool(after), bool(before), scale, float(eps), rows_per_gate)
    own_stream = residual is not None or bool(after) or gate is not None or scale != 1.0
    if not own_stream and not before:
        return x, None
    tensors = (x, residual, gate, after_weight, after_bias, before_weight, before_bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        stream, normed = _BlockNorm.apply(*tensors, conf, own_stream)
    else:
        stream, normed = _norm_forward(*tensors, conf, own_stream)
    return (stream if own_stream else x), normed
