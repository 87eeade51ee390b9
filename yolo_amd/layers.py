"""Layers of a residual block on the gfx950 HIP library, beside the convolutions and the batch norm that
yolo_v3 runs: a matrix product with bias, activation and residual in its epilogue, and the norms after and
before a block fused with the block's gate, residual scale and residual add.

    stream, normed = block_norm(x, before_weight=w0)                 # enter the first block
    up = linear(normed, w1, b1, activation="gelu_tanh")
    out = linear(up, w2, b2)
    stream, normed = block_norm(out, stream, after_weight=w3, gate=g, before_weight=w4)    # on to the next

Both are differentiable in every tensor argument (once; a second derivative raises), take inputs on any GPU and
run on torch's current stream of that GPU.  They allocate outputs and scratch with torch's allocator, so they
can be captured into a HIP graph, keep nothing between calls and never synchronise.  Results depend on the
inputs alone: every sum has a fixed order.  Row views (``x[:, :k]``) are read in place; other strides are copied.
There is no CPU implementation: tensors on the CPU raise YoloAmdError.

The reference has no counterpart of either.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import BlockNormBackwardDesc, BlockNormDesc, LinearBackwardDesc, LinearDesc, YoloAmdError, check, lib

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
_F32 = torch.float32
_byref = ctypes.byref


def _on_gpu(what, first, **others):
    """Every tensor is a GPU tensor on the first one's device."""
    if not torch.is_tensor(first):
        raise TypeError(f"{what}: expected a torch tensor, got {type(first).__name__}")
    dev = first.device
    if dev.type != "cuda":
        raise YoloAmdError(f"{what}: the tensors are on the CPU; this path runs on the GPU only")
    for name, t in others.items():
        if t is None:
            continue
        if not torch.is_tensor(t):
            raise TypeError(f"{what}: {name} is not a torch tensor")
        if t.device != dev:
            raise YoloAmdError(f"{what}: {name} is on {t.device}, the first argument on {dev}")
    return dev


def _rows(t):
    """(tensor, row stride): ``t`` as rows of its last dimension at one stride, copied where its strides do not
    allow that."""
    shape = t.shape
    if t.is_contiguous():
        return t, shape[-1]
    if t.dim() >= 2 and t.stride(-1) == 1 and t.stride(-2) >= shape[-1]:
        step = t.stride(-2)
        for i in range(t.dim() - 3, -1, -1):
            if shape[i] != 1 and t.stride(i) != t.stride(i + 1) * shape[i + 1]:
                break
        else:
            return t, step
    t = t.contiguous()
    return t, shape[-1]


def _call(dev, fn, desc, what):
    """Run ``fn(desc, current stream)`` on ``dev``."""
    if dev.index == torch.cuda.current_device():
        check(fn(_byref(desc), torch.cuda.current_stream(dev).cuda_stream), what)
    else:
        with torch.cuda.device(dev):
            check(fn(_byref(desc), torch.cuda.current_stream(dev).cuda_stream), what)


def _scratch(desc, nbytes, dev):
    """Scratch of one call.  Taken from torch's allocator each time: calls on different streams, or in different
    captured graphs, never share it."""
    if nbytes == 0:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    desc.workspace, desc.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _ptr(t):
    return None if t is None else t.data_ptr()


# --------------------------------------------------------------------------
# linear
# --------------------------------------------------------------------------
def _linear_forward(x, weight, bias, residual, act, out_dtype, keep_pre):
    """Returns (y, pre or None)."""
    n, k = weight.shape
    xr, ldx = _rows(x)
    wr, ldw = _rows(weight)
    shape = x.shape[:-1] + (n,)
    m = x.numel() // k if k else shape.numel() // n if n else 0
    y = torch.empty(shape, dtype=out_dtype, device=x.device)
    d = LinearDesc()
    d.x, d.weight, d.y = xr.data_ptr(), wr.data_ptr(), y.data_ptr()
    d.m, d.n, d.k, d.ldx, d.ldw, d.ldy = m, n, k, ldx, ldw, n
    d.type, d.y_f32, d.activation = _TYPES[x.dtype], out_dtype == _F32, act
    if bias is not None:
        bias = bias.contiguous()
        d.bias, d.bias_f32 = bias.data_ptr(), bias.dtype == _F32
    if residual is not None:
        rr, d.ldr = _rows(residual)
        d.residual, d.residual_f32 = rr.data_ptr(), residual.dtype == _F32
    pre = None
    if keep_pre:
        pre = torch.empty(shape, dtype=x.dtype, device=x.device)
        d.pre = pre.data_ptr()
    ws = _scratch(d, lib.yolo_amd_linear_workspace_bytes(_byref(d)), x.device)     # noqa: F841  (alive over the call)
    _call(x.device, lib.yolo_amd_linear_forward, d, "linear")
    return y, pre


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_dtype):
        need_pre = act != 0 and any(ctx.needs_input_grad[:3])
        y, pre = _linear_forward(x, weight, bias, residual, act, out_dtype, need_pre)
        need = ctx.needs_input_grad
        ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, pre)
        ctx.act, ctx.k = act, weight.shape[1]
        ctx.x_shape, ctx.w_shape, ctx.type = x.shape, weight.shape, x.dtype
        ctx.bias_dtype = bias.dtype if bias is not None else None
        ctx.residual_dtype = residual.dtype if residual is not None else None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dres = None
        if need[3]:
            dres = dy if dy.dtype == ctx.residual_dtype else dy.to(ctx.residual_dtype)
        if not any(need[:3]):
            return None, None, None, dres, None, None
        x, weight, pre = ctx.saved_tensors
        n, k = ctx.w_shape
        dev = dy.device
        dyr, lddy = _rows(dy)
        d = LinearBackwardDesc()
        d.dy, d.lddy, d.dy_f32 = dyr.data_ptr(), lddy, dy.dtype == _F32
        d.m, d.n, d.k = (dy.numel() // n if n else ctx.x_shape[:-1].numel()), n, k
        d.type, d.activation = _TYPES[ctx.type], ctx.act
        d.pre = _ptr(pre)
        dx = dw = db = None
        if need[0]:
            wr, d.ldw = _rows(weight)
            dx = torch.empty(ctx.x_shape, dtype=ctx.type, device=dev)
            d.weight, d.dx = wr.data_ptr(), dx.data_ptr()
        if need[1]:
            xr, d.ldx = _rows(x)
            dw = torch.empty(ctx.w_shape, dtype=ctx.type, device=dev)
            d.x, d.dweight = xr.data_ptr(), dw.data_ptr()
        if need[2]:
            db = torch.empty(n, dtype=ctx.bias_dtype, device=dev)
            d.dbias, d.dbias_f32 = db.data_ptr(), ctx.bias_dtype == _F32
        ws = _scratch(d, lib.yolo_amd_linear_backward_workspace_bytes(_byref(d)), dev)     # noqa: F841
        _call(dev, lib.yolo_amd_linear_backward, d, "linear backward")
        return dx, dw, db, dres, None, None


def linear(x, weight, bias=None, *, activation=None, residual=None, out_dtype=None):
    """``act(x @ weight.T + bias) + residual`` in one launch (two where few output tiles share a long reduction).

    x (..., K) and weight (N, K): bf16 or fp16, the same.  bias (N,): that type or fp32.  residual (..., N), the
    shape of the result: that type or fp32.  activation: None, "leaky" (slope 0.1), "relu", "gelu" (erf),
    "gelu_tanh" or "silu".  The result has ``out_dtype`` (x's type by default, or torch.float32).

    Sums are fp32; the result is rounded once.  Where a gradient of x, weight or bias will be wanted and there is
    an activation, ``x @ weight.T + bias`` is kept in x's type for the backward pass; the gradients of x and
    weight round d(loss)/d(pre-activation) to that type once, as the operand of their products."""
    dev = _on_gpu("linear", x, weight=weight, bias=bias, residual=residual)
    dt = x.dtype
    if dt not in (torch.bfloat16, torch.float16):
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
def _norm_desc(x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf):
    """(descriptor without outputs, tensors to keep alive over the call)."""
    norm, after, before, scale, eps, rows_per_gate = conf
    d = BlockNormDesc()
    dim = x.shape[-1]
    xr, d.ldx = _rows(x)
    keep = [xr]
    d.x, d.rows, d.d = xr.data_ptr(), x.numel() // dim, dim
    d.type, d.norm, d.after, d.before, d.eps, d.scale = _TYPES[x.dtype], norm, after, before, eps, scale
    if residual is not None:
        rr, d.ldr = _rows(residual)
        keep.append(rr)
        d.residual, d.stream_f32 = rr.data_ptr(), residual.dtype == _F32
    else:
        d.stream_f32 = x.dtype == _F32
    if gate is not None:
        gate = gate.contiguous()
        keep.append(gate)
        d.gate, d.gate_f32, d.rows_per_gate = gate.data_ptr(), gate.dtype == _F32, rows_per_gate
    for name, t in (("after_weight", after_weight), ("after_bias", after_bias), ("before_weight", before_weight),
                    ("before_bias", before_bias)):
        if t is not None:
            t = t.contiguous()
            keep.append(t)
            setattr(d, name, t.data_ptr())
            if name[0] == "a":
                d.after_f32 = t.dtype == _F32
            else:
                d.before_f32 = t.dtype == _F32
    return d, keep


def _norm_forward(x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf, own_stream):
    """(stream or None where it is x itself, normed or None)."""
    d, keep = _norm_desc(x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf)
    stream = normed = None
    if own_stream:
        stream = torch.empty(x.shape, dtype=x.dtype if residual is None else residual.dtype, device=x.device)
        d.stream = stream.data_ptr()
    if conf[2]:
        normed = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        d.normed = normed.data_ptr()
    _call(x.device, lib.yolo_amd_block_norm_forward, d, "block_norm")
    return stream, normed


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, after_weight, after_bias, before_weight, before_bias, conf, own_stream):
        tensors = (x, residual, gate, after_weight, after_bias, before_weight, before_bias)
        stream, normed = _norm_forward(*tensors, conf, own_stream)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*tensors)
        ctx.conf = conf
        return stream, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dstream, dnormed):
        tensors = ctx.saved_tensors
        x = tensors[0]
        dev = x.device
        need = ctx.needs_input_grad
        b = BlockNormBackwardDesc()
        d, keep = _norm_desc(*tensors, ctx.conf)
        b.forward = d
        if dnormed is not None:
            dnormed = dnormed.contiguous()
            b.dnormed = dnormed.data_ptr()
        if dstream is not None:
            dstream = dstream.contiguous()
            b.dstream = dstream.data_ptr()
        grads = [None] * 7
        for i, name in enumerate(("dx", "dresidual", "dgate", "dafter_weight", "dafter_bias", "dbefore_weight",
                                  "dbefore_bias")):
            if need[i]:
                grads[i] = torch.empty(tensors[i].shape, dtype=tensors[i].dtype, device=dev)
                setattr(b, name, grads[i].data_ptr())
        ws = _scratch(b, lib.yolo_amd_block_norm_backward_workspace_bytes(_byref(b)), dev)     # noqa: F841
        _call(dev, lib.yolo_amd_block_norm_backward, b, "block_norm backward")
        return (*grads, None, None)


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
    dev = _on_gpu("block_norm", x, residual=residual, gate=gate, after_weight=after_weight, after_bias=after_bias,
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
    for name, flag, w, b in (("after", after, after_weight, after_bias), ("before", before, before_weight, before_bias)):
        for kind, t in (("weight", w), ("bias", b)):
            if t is None:
                continue
            if not flag:
                raise ValueError(f"block_norm: {name}_{kind} without the norm it belongs to")
            if t.shape != x.shape[-1:] or t.dtype not in (dt, _F32):
                raise ValueError(f"block_norm: {name}_{kind} must be ({x.shape[-1]},) of {dt} or float32, got "
                                 f"{tuple(t.shape)} of {t.dtype}")
        if b is not None and norm == "rms":
            raise ValueError("block_norm: an rms norm has no bias")
        if w is not None and b is not None and w.dtype != b.dtype:
            raise ValueError(f"block_norm: {name}_weight is {w.dtype}, {name}_bias is {b.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (dt, _F32)):
        raise ValueError(f"block_norm: residual must be {tuple(x.shape)} of {dt} or float32, got {tuple(residual.shape)} "
                         f"of {residual.dtype}")
    if gate is not None and gate.dtype not in (dt, _F32):
        raise TypeError(f"block_norm: gate must be {dt} or float32, got {gate.dtype}")
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
