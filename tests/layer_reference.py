"""Definitions of yolo_amd.layers in 64 bits, with bounds on how far a correct fp32 computation with the documented
roundings may be from them.  Bounds are first order and follow the chain of operations:

 * rounding to a type t is off by at most U[t] = finfo(t).eps / 2 relative (TINY[t] absolute below its normal range);
 * a matrix product over K accumulates K terms in fp32 in some order, each addition off by at most 2^-23 of the sum of
   magnitudes (2^-24 rounded to nearest; the matrix unit may truncate);
 * EPS32 = 1e-5 covers a chain of fp32 operations with a tree sum of depth <= 40 in it ((40 + 20) * 2^-24 = 3.6e-6,
   twice) and the hardware exp2 / rcp / rsq (1 ulp each, arguments scaled by log2(e)), whose error the framework
   states as at most 6e-6 relative.
"""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
EPS32 = 1e-5
C = math.sqrt(2 / math.pi)


def act64(p, kind):
    if kind is None:
        return p
    if kind == "leaky":
        return torch.where(p > 0, p, 0.1 * p)
    if kind == "relu":
        return p.clamp_min(0)
    if kind == "gelu":
        return 0.5 * p * torch.special.erfc(-p * math.sqrt(0.5))
    if kind == "gelu_tanh":
        return p * torch.sigmoid(2 * C * (p + 0.044715 * p ** 3))
    if kind == "silu":
        return p * torch.sigmoid(p)
    raise KeyError(kind)


def slope64(p, kind):
    if kind is None:
        return torch.ones_like(p)
    if kind == "leaky":
        return torch.where(p > 0, 1.0, 0.1).to(p.dtype)
    if kind == "relu":
        return (p > 0).to(p.dtype)
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-p * math.sqrt(0.5)) + p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        z = torch.sigmoid(2 * C * (p + 0.044715 * p ** 3))
        return z + p * z * (1 - z) * 2 * C * (1 + 3 * 0.044715 * p * p)
    if kind == "silu":
        z = torch.sigmoid(p)
        return z * (1 + p * (1 - z))
    raise KeyError(kind)


def d(t):
    return None if t is None else t.detach().double().cpu()


def rounded(value, bound, dtype):
    """bound plus one rounding of a value that is already `bound` off."""
    return bound + U[dtype] * (value.abs() + bound) + TINY[dtype]


def linear_ref(x, w, bias, residual, kind, out_dtype):
    """(y, bound on y, P, bound on the fp32 P)."""
    x, w, b, r = d(x), d(w), d(bias), d(residual)
    k = w.shape[1]
    p = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if b is not None:
        p, mag = p + b, mag + b.abs()
    ep = (k + 4) * 2.0 ** -23 * mag
    a = act64(p, kind)
    # |act'| <= 1.13 for all of them; 1 + erf cancels: |p| 2^-22 absolute
    ey = 1.13 * ep + (EPS32 * a.abs() + 2.0 ** -22 * p.abs() if kind else 0)
    y = a
    if r is not None:
        y = a + r
        ey = ey + 2.0 ** -23 * (a.abs() + r.abs())
    return y, rounded(y, ey, out_dtype), p, ep


def linear_grad_ref(x, w, p, ep, dy, kind, bias_dtype):
    """((dx, bound), (dw, bound), (db, bound)); p, ep from linear_ref."""
    t = x.dtype
    x, w, dy = d(x), d(w), d(dy)
    s = slope64(p, kind)
    if kind is None:
        es = torch.zeros_like(p)
    elif kind in ("leaky", "relu"):
        # only an element whose sign the sum's rounding can change may take the other slope
        es = (p.abs() <= ep + TINY[t]).to(p.dtype)
    else:
        # |act''| <= 0.8 (gelu and its tanh form; silu 0.5); P is kept rounded to the operands' type
        es = 0.8 * (ep + U[t] * (p.abs() + ep)) + EPS32 * (1 + s.abs())
    dp = dy * s
    edp = dy.abs() * es + 2.0 ** -23 * dp.abs()
    db = dp.sum(0)
    # column sums: runs of at most 64 rows per thread here, then at most 2048 runs
    edb = edp.sum(0) + 512 * 2.0 ** -24 * dp.abs().sum(0)
    eop = edp + U[t] * (dp.abs() + edp) + TINY[t]
    m, n = dp.shape
    dx = dp @ w
    edx = eop @ w.abs() + (n + 4) * 2.0 ** -23 * (dp.abs() @ w.abs())
    dw = dp.t() @ x
    edw = eop.t() @ x.abs() + (m + 4) * 2.0 ** -23 * (dp.abs().t() @ x.abs())
    return ((dx, rounded(dx, edx, t)), (dw, rounded(dw, edw, t)),
            (db, rounded(db, edb, bias_dtype) if bias_dtype else edb))


def _unit(v, norm, eps):
    mean = v.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(v[..., :1])
    f = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    return (v - mean) * f, f


def _m(v):
    return v.mean(-1, keepdim=True)


def norm_ref(x, residual, conf, params, grads=None):
    """64-bit outputs, and gradients where grads = (dstream, dnormed) is given, each as (value, bound before the
    output's rounding).  conf: norm, after, before, scale, eps.  params: gate (expanded to rows or None), after_weight,
    after_bias, before_weight, before_bias."""
    norm, after, before, s, eps = conf
    u = d(x)
    r = d(residual) if residual is not None else torch.zeros_like(u)
    one, zero = torch.ones_like(u), torch.zeros_like(u)
    g = d(params.get("gate"))
    g = g.expand_as(u) if g is not None else one
    wa, ba, wb, bb = (d(params.get(n)) for n in ("after_weight", "after_bias", "before_weight", "before_bias"))
    wa, wb = (one if w is None else w.expand_as(u) for w in (wa, wb))
    ba, bb = (zero if b is None else b.expand_as(u) for b in (ba, bb))
    out = {}
    if after:
        uu, fu = _unit(u, norm, eps)
        au = uu.abs() + fu * _m(u.abs())
        p = uu * wa + ba
        ep = EPS32 * (wa.abs() * au + ba.abs())
    else:
        uu, fu, au, p, ep = u, torch.ones_like(u[..., :1]), u.abs(), u, zero
    h = r + s * g * p
    eh = (s * g).abs() * ep + EPS32 * (r.abs() + (s * g * p).abs())
    out["stream"] = (h, eh)
    if before:
        hh, fh = _unit(h, norm, eps)
        rel = fh * torch.sqrt(_m(eh * eh)) + EPS32
        ehh = fh * (eh + _m(eh)) + hh.abs() * rel + EPS32 * (hh.abs() + fh * _m(h.abs()))
        y = hh * wb + bb
        out["normed"] = (y, wb.abs() * ehh + EPS32 * (y.abs() + bb.abs()))
    if grads is None:
        return out
    dh, dy = d(grads[0]), d(grads[1])
    dh = zero if dh is None else dh
    edH = EPS32 * dh.abs()
    dH = dh
    if dy is not None:
        q = dy * wb
        c0 = _m(q) if norm == "layer" else 0 * _m(q)
        c1 = _m(q * hh)
        a0 = _m(q.abs()) if norm == "layer" else 0 * c0
        a1 = _m((q * hh).abs())
        dH = dh + fh * (q - c0 - hh * c1)
        edH = edH + fh * ((EPS32 + rel) * (q.abs() + a0 + hh.abs() * a1) + ehh * a1 + hh.abs() * _m(q.abs() * ehh))
    out["residual"] = (dH, edH)
    sums = 512 * 2.0 ** -24              # rows in one thread and partial sums: chains of at most 512 additions here
    dg = s * p * dH
    out["gate_rows"] = (dg, abs(s) * (edH * p.abs() + dH.abs() * ep) + EPS32 * dg.abs(), sums)
    dp = s * g * dH
    edp = (s * g).abs() * edH + EPS32 * dp.abs()
    if after:
        q = dp * wa
        eq = wa.abs() * edp + EPS32 * q.abs()
        euu = EPS32 * au
        c0 = _m(q) if norm == "layer" else 0 * _m(q)
        du = fu * (q - c0 - uu * _m(q * uu))
        mq, me = (_m(q.abs()), _m(eq)) if norm == "layer" else (0 * c0, 0 * c0)
        a1 = _m((q * uu).abs())
        edu = fu * (eq + me + uu.abs() * _m(eq * uu.abs()) + 2 * EPS32 * (q.abs() + mq + uu.abs() * a1)
                    + euu * a1 + uu.abs() * _m(q.abs() * euu))
        out["x"] = (du, edu)
        flat = tuple(range(u.dim() - 1))
        out["after_weight"] = ((dp * uu).sum(flat), (edp * uu.abs() + dp.abs() * euu + sums * (dp * uu).abs()).sum(flat))
        out["after_bias"] = (dp.sum(flat), (edp + sums * dp.abs()).sum(flat))
    else:
        out["x"] = (dp, edp)
    if dy is not None:
        flat = tuple(range(u.dim() - 1))
        out["before_weight"] = ((dy * hh).sum(flat), (dy.abs() * ehh + sums * (dy * hh).abs()).sum(flat))
        out["before_bias"] = (dy.sum(flat), (sums * dy.abs()).sum(flat))
    return out


def reduce_gate(dg, shape):
    """Sum the per-row gate gradient (value, bound, sums) over the rows that share a gate."""
    v, e, sums = dg
    e = e + sums * v.abs()
    full = (1,) * (v.dim() - len(shape)) + tuple(shape)
    over = tuple(i for i in range(v.dim()) if full[i] == 1 and v.shape[i] != 1)
    if over:
        v, e = v.sum(over, keepdim=True), e.sum(over, keepdim=True)
    return v.reshape(shape), e.reshape(shape)


def assert_within(got, value, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == value.shape, f"{what}: {tuple(got.shape)} instead of {tuple(value.shape)}"
    off = (got - value).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = int(torch.where(bad, off / bound.clamp_min(1e-300), torch.zeros_like(off)).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds, worst at {i}: "
                             f"{got.flatten()[i]} instead of {value.flatten()[i]} +- {bound.flatten()[i]}")
