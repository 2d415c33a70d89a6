"""Rotary positions of queries and keys, with an optional norm of each head in the same pass (csrc/kernels/rotary.hip;
a torch oracle on the CPU).

For one head x of one token, D wide: ``n = x / sqrt(mean(x^2) + eps) * weight`` (only where a weight is given), then the
first ``R = 2 * len(freqs)`` dims of n turn in pairs by ``angle_i = pos * freqs[i]``:

    a' = mscale (a cos - b sin),  b' = mscale (b cos + a sin),  (a, b) = dims (i, i + R/2), interleaved: (2i, 2i + 1)

and the other dims pass through. ``rotary`` is differentiable in q, k and both weights; ``paged.rotary_append`` is the
serving form that writes keys and values into a paged cache.
"""
from __future__ import annotations

import functools
import math
import typing

import torch
from torch.autograd import forward_ad

from . import _lib as L
from . import raw
from .functional import _acc_grad, _done, _param32

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_DIM = 512
MIN_EPS, MAX_EPS = 2.0 ** -126, 2.0 ** 127


def rotary_freqs(rot_dim: int, theta: float = 10000.0, scaling: typing.Optional[dict] = None,
                 device: typing.Union[str, torch.device, None] = None) -> typing.Tuple[torch.Tensor, float]:
    """(frequencies in radians per position, float64 [rot_dim / 2]; the factor ``mscale`` of the turned dims).

    Plain: ``theta ** (-2 i / rot_dim)``, mscale 1. ``scaling`` stretches them for contexts ``factor`` times as long as
    the trained one: ``{"type": ..., "factor": s}`` with

    * ``"linear"``: positions are divided by s;
    * ``"base"`` (the "NTK-aware" base): theta grows by ``s ** (rot_dim / (rot_dim - 2))``: the slowest pair turns s
      times slower, the fastest as before;
    * ``"ramp"`` (YaRN, Peng et al. 2023): pairs that turn more than ``fast`` (32) times over the trained ``length``
      (2048) keep their frequency, those under ``slow`` (1) turns are divided by s, linear in between over the pair's index
      (from the whole pair before the one to the whole pair after the other, pairs past the last one counted up to
      ``rot_dim - 1``); mscale is ``0.1 ln s + 1``, sharpening the scores that the longer context flattens."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rotary needs an even number of dims, got {rot_dim}")
    if not theta > 0:
        raise ValueError(f"rotary base must be positive, got {theta}")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    mscale = 1.0
    kind, s = None, 1.0
    if scaling:
        unknown = set(scaling) - {"type", "factor", "length", "fast", "slow"}
        if unknown:
            raise ValueError(f"unknown rotary scaling keys {sorted(unknown)}")
        kind, s = scaling["type"], float(scaling["factor"])
        if not s >= 1:
            raise ValueError(f"rotary scaling factor must be at least 1, got {s}")
    if kind == "base":
        if rot_dim < 4:
            raise ValueError("rotary scaling 'base' needs at least 4 dims")
        theta = theta * s ** (rot_dim / (rot_dim - 2))
    freqs = theta ** (-2.0 * i / rot_dim)
    if kind == "linear":
        freqs = freqs / s
    elif kind == "ramp":
        length, fast, slow = (float(scaling.get(k, v)) for k, v in (("length", 2048), ("fast", 32), ("slow", 1)))
        if not (length > 0 and fast > slow > 0 and theta > 1):
            raise ValueError("rotary scaling 'ramp' needs length > 0, fast > slow > 0 and a base above 1")

        def pair_of(turns):     # the (fractional) pair that makes `turns` turns over the trained length
            return rot_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rot_dim - 1)
        far = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        if pair_of(slow) < 0:                                   # also the fastest pair is under `slow` turns
            far = torch.ones_like(i)
        freqs = freqs * (1 - far) + freqs / s * far
        mscale = 0.1 * math.log(s) + 1.0
    elif kind not in (None, "base"):
        raise ValueError(f"unknown rotary scaling type {kind!r} (linear, base, ramp)")
    return freqs.to(device) if device is not None else freqs, mscale


# ----------------------------------------------------------------------------------------------------------------
# argument checks and layouts shared with the serving form. A decode step calls these once per layer and waits for them:
# they touch each tensor attribute once
def tokens_view(t: torch.Tensor) -> typing.Tuple[torch.Tensor, int, int]:
    """[..., H, D] -> (the tensor, token stride, head stride); a copy only where the leading dims are no single stride
    or the last one is not dense"""
    shape = t.shape
    if t.is_contiguous():
        return t, shape[-1] * shape[-2], shape[-1]
    st, n = t.stride(), len(shape)
    # the leading dims that are wider than 1 must follow from one another
    lead = [i for i in range(n - 2) if shape[i] != 1]
    if (st[-1] != 1 and shape[-1] != 1) or any(st[i] != st[j] * shape[j] for i, j in zip(lead, lead[1:])):
        return t.contiguous(), shape[-1] * shape[-2], shape[-1]
    return t, st[lead[-1]] if lead else 0, st[-2]


def check_args(what: str, q, k, pos, freqs, wq, wk, eps: float):
    """(positions over the tokens, frequencies, both contiguous; rotated dims; tokens)"""
    qs, ks, dev = q.shape, k.shape, q.get_device()
    n, D = len(qs), qs[-1] if len(qs) else 0
    if n < 3 or len(ks) != n or ks[-1] != D or qs[:-2] != ks[:-2]:
        raise L.KernelError(f"{what}: q {list(qs)} and k {list(ks)} must be [..., heads, dim] over the same tokens")
    if qs[-2] < 1 or ks[-2] < 1 or not 1 <= D <= MAX_DIM:
        raise L.KernelError(f"{what}: at least one head of 1 to {MAX_DIM} dims, got {list(qs)}, {list(ks)}")
    if k.dtype != q.dtype or k.get_device() != dev:
        raise L.KernelError(f"{what}: q and k must share type and device")
    if dev >= 0 and q.dtype not in DTYPES:
        raise L.KernelError(f"{what}: bf16, fp16 or fp32 on the GPU, got {q.dtype}")
    if pos.dtype != torch.int64 or pos.get_device() != dev:
        raise L.KernelError(f"{what}: positions must be int64 on the device of q")
    lead = qs[:-2]
    if pos.shape != lead:
        try:
            pos = pos.expand(lead)
        except RuntimeError:
            raise L.KernelError(f"{what}: positions {list(pos.shape)} for tokens {list(lead)}") from None
    if not pos.is_contiguous():
        pos = pos.contiguous()
    rot = 0
    if freqs is not None:
        rot = 2 * freqs.numel()
        if freqs.dtype != torch.float64 or freqs.dim() != 1 or freqs.get_device() != dev or rot > D:
            raise L.KernelError(f"{what}: freqs must be float64 [pairs] on the device of q with 2 * pairs <= {D}, got "
                                f"{freqs.dtype} {list(freqs.shape)} on {freqs.device}")
        if not freqs.is_contiguous():
            freqs = freqs.contiguous()
    for w in (wq, wk):
        if w is not None and (w.numel() != D or w.get_device() != dev or not w.dtype.is_floating_point):
            raise L.KernelError(f"{what}: norm weights must be [{D}] on the device of q")
    if not MIN_EPS <= eps < MAX_EPS and not (q.dtype == torch.float64 and eps > 0):
        raise L.KernelError(f"{what}: eps must be positive and a normal number of 32 bits, got {eps}")
    return pos, freqs, rot, math.prod(lead)


def refuse_tangents(what: str, *tensors):
    """the kernels carry no forward-mode derivative: a dual tensor is refused rather than its tangent dropped"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise L.KernelError(f"{what} has no forward-mode derivative")


def kernel_weights(wq, wk):
    """(wq, wk, type code) as the kernels read them: the fp32 master copy of a model parameter, else the tensor itself;
    of two types, both in fp32"""
    w = wk if wq is None else wq
    if w is None:
        return None, None, 0
    if hasattr(wq, "master") or hasattr(wk, "master"):
        wq, wk = _param32(wq), _param32(wk)
        w = wk if wq is None else wq
    if w.dtype not in DTYPES or (wk is not None and wk.dtype != w.dtype):
        wq, wk = (None if x is None else x.float() for x in (wq, wk))
        w = wk if wq is None else wq
    if wq is not None and not wq.is_contiguous():
        wq = wq.contiguous()
    if wk is not None and not wk.is_contiguous():
        wk = wk.contiguous()
    return wq, wk, DTYPES[w.dtype]


# ----------------------------------------------------------------------------------------------------------------
# torch oracle
def turn_t(x, pos, freqs, inter: bool, mscale: float, sign: float = 1.0):
    """[T, H, D] in 32 or 64 bits: the pairs turned by sign * angle, scaled"""
    if freqs is None or freqs.numel() == 0:
        return x
    R = 2 * freqs.numel()
    ang = pos.reshape(-1, 1).to(torch.float64) * freqs
    c, s = ((f(ang) * mscale).to(x.dtype).unsqueeze(1) for f in (torch.cos, torch.sin))
    s = s * sign
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if inter else (x[..., :R // 2], x[..., R // 2:R])
    u, v = a * c - b * s, b * c + a * s
    y = torch.stack((u, v), -1).flatten(-2) if inter else torch.cat((u, v), -1)
    return torch.cat((y, x[..., R:]), -1)


def rotary_t(x, w, pos, freqs, inter: bool, mscale: float, eps: float):
    x2 = raw._f(x).reshape(-1, *x.shape[-2:])
    if w is not None:
        x2 = x2 * torch.rsqrt((x2 * x2).mean(-1, keepdim=True) + eps) * w.to(x2.dtype).reshape(-1)
    return turn_t(x2, pos, freqs, inter, mscale).reshape(x.shape).to(x.dtype)


def rotary_bwd_t(x, w, g, pos, freqs, inter: bool, mscale: float, eps: float):
    g2 = turn_t(raw._f(g).reshape(-1, *g.shape[-2:]), pos, freqs, inter, mscale, -1.0)
    if w is None:
        return g2.reshape(g.shape).to(g.dtype), None
    x2 = raw._f(x).reshape(-1, *x.shape[-2:])
    r = torch.rsqrt((x2 * x2).mean(-1, keepdim=True) + eps)
    u = x2 * r
    dw = (g2 * u).sum((0, 1))
    h = g2 * w.to(g2.dtype).reshape(-1)
    return (r * (h - u * (h * u).mean(-1, keepdim=True))).reshape(g.shape).to(g.dtype), dw


# ----------------------------------------------------------------------------------------------------------------
def _forward(q, k, pos, freqs, wq, wk, rot, T, inter, mscale, eps):
    qs, ks = q.shape, k.shape
    qo, ko = q.new_empty(qs), k.new_empty(ks)
    if T == 0 or q.is_meta:
        return qo, ko
    if q.get_device() < 0:
        w = [None if x is None else _param32(x).detach() for x in (wq, wk)]
        qo.copy_(rotary_t(q, w[0], pos, freqs, inter, mscale, eps))
        ko.copy_(rotary_t(k, w[1], pos, freqs, inter, mscale, eps))
        return qo, ko
    q, q_ts, q_hs = tokens_view(q)
    k, k_ts, k_hs = tokens_view(k)
    wq, wk, wt = kernel_weights(wq, wk)
    L.launch(L.lib().obst_rotary_fwd, q, "rotary", L.ROT_DESC.pack(
        q.data_ptr(), k.data_ptr(), 0, 0, 0, qo.data_ptr(), ko.data_ptr(), 0, L.ptr(wq), L.ptr(wk), L.ptr(freqs),
        pos.data_ptr(), 0, 0, 0, 0, q_ts, q_hs, k_ts, k_hs, 0, 0, 0, 0, 0, 0, T, 0, qs[-2], ks[-2], qs[-1], rot, inter,
        DTYPES[q.dtype], wt, 0, 0, 0, mscale, eps))
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, pos, freqs, cfg):
        ctx.cfg = cfg
        if wq is None and wk is None:
            ctx.save_for_backward(pos, freqs)
        else:
            ctx.save_for_backward(pos, freqs, q, k, wq, wk)
        return _forward(q, k, pos, freqs, wq, wk, *cfg)

    @staticmethod
    def backward(ctx, gq, gk):
        if torch.is_grad_enabled():
            raise L.KernelError("rotary has no second derivative (create_graph)")
        pos, freqs, *normed = ctx.saved_tensors
        dq, dk = gq.new_empty(gq.shape), gk.new_empty(gk.shape)
        if not normed:
            _backward(None, None, gq, gk, dq, dk, None, None, None, None, False, pos, freqs, *ctx.cfg)
            return dq, dk, None, None, None, None, None
        q, k, wq, wk = normed
        # model parameters accumulate into their fp32 main gradient; other weights get theirs back, in their own type where
        # the kernel writes it, else from fp32 (on the CPU fp64 for fp64)
        main = getattr(wq, "main_grad", None) is not None or getattr(wk, "main_grad", None) is not None
        one = wq is None or wk is None or wq.dtype == wk.dtype
        gpu = gq.get_device() >= 0

        def buffer(w):
            if w is None:
                return None, True
            if main:
                return _acc_grad(w)
            if gpu and one and w.dtype in DTYPES:
                return w.new_empty(w.shape), False
            return w.new_zeros(w.shape, dtype=w.dtype if w.dtype == torch.float64 and not gpu else torch.float32), False
        dwq, main_q = buffer(wq)
        dwk, main_k = buffer(wk)
        into = dwk
        if main and dwq is not None and dwk is not None and dwq.data_ptr() == dwk.data_ptr():
            into = torch.zeros_like(dwk)                                   # one parameter for both
        _backward(q, k, gq, gk, dq, dk, wq, wk, dwq, into, main, pos, freqs, *ctx.cfg)
        if into is not dwk:
            dwk.add_(into)
        for w in (wq, wk):
            if w is not None:
                _done(w)
        if not main_q and dwq.dtype != wq.dtype:
            dwq = dwq.to(wq.dtype)
        if not main_k and dwk.dtype != wk.dtype:
            dwk = dwk.to(wk.dtype)
        return dq, dk, None if main_q else dwq, None if main_k else dwk, None, None, None


@functools.lru_cache(None)
def _part(D: int) -> int:
    """floats of the weight sums' workspace"""
    return L.lib().obst_rotary_part(D)


def _backward(q, k, gq, gk, dq, dk, wq, wk, dwq, dwk, add: bool, pos, freqs, rot, T, inter, mscale, eps):
    """dq, dk and the weights' gradients (into dwq, dwk; added to what they hold in fp32 where ``add``)"""
    if gq.get_device() < 0:
        for x, w, g, o, dw in ((q, wq, gq, dq, dwq), (k, wk, gk, dk, dwk)):
            dx, d = rotary_bwd_t(x, None if w is None else _param32(w).detach(), g, pos, freqs, inter, mscale, eps)
            o.copy_(dx)
            if d is not None:
                dw.add_(d.reshape(dw.shape))
        return
    gs = gq.shape
    gq, gq_ts, gq_hs = tokens_view(gq)
    gk, gk_ts, gk_hs = tokens_view(gk)
    q_ts = q_hs = k_ts = k_hs = wt = dt = 0
    part = None
    if q is not None:
        q, q_ts, q_hs = tokens_view(q)
        k, k_ts, k_hs = tokens_view(k)
        part = gq.new_empty(_part(gs[-1]), dtype=torch.float32)
        wq, wk, wt = kernel_weights(wq, wk)
        dt = DTYPES[(dwk if dwq is None else dwq).dtype]
    L.launch(L.lib().obst_rotary_bwd, gq, "rotary_bwd", L.ROT_DESC.pack(
        L.ptr(q), L.ptr(k), 0, gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), 0, L.ptr(wq), L.ptr(wk),
        L.ptr(freqs), pos.data_ptr(), 0, L.ptr(part), L.ptr(dwq), L.ptr(dwk), q_ts, q_hs, k_ts,
        k_hs, 0, 0, gq_ts, gq_hs, gk_ts, gk_hs, T, 0, gs[-2], gk.shape[-2], gs[-1], rot, inter, DTYPES[gq.dtype], wt, dt,
        add, 0, mscale, eps))


def rotary(q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor, freqs: typing.Optional[torch.Tensor],
           interleaved: bool = False, mscale: float = 1.0, q_weight: typing.Optional[torch.Tensor] = None,
           k_weight: typing.Optional[torch.Tensor] = None, eps: float = 1e-5
           ) -> typing.Tuple[torch.Tensor, torch.Tensor]:
    """Queries [..., Hq, D] and keys [..., Hk, D] of the same tokens, normed (each where its weight [D] is given) and
    turned (module docstring); any token and head strides. ``pos`` int64 over the tokens (or broadcastable to them; angles
    are off by up to 2e-15 radians a turn made: a rounding of 32 bits at position 1.8e8 of a pair of frequency 1),
    ``freqs`` float64 from ``rotary_freqs`` (None: no rotation). Returns new contiguous tensors; differentiable in q, k
    and the weights, sums in fp32, weight gradients in a fixed order (the same bits each run). No forward-mode derivative
    on the GPU."""
    pos, freqs, rot, T = check_args("rotary", q, k, pos, freqs, q_weight, k_weight, eps)
    cfg = (rot, T, bool(interleaved), float(mscale), float(eps))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        return _Rotary.apply(q, k, q_weight, k_weight, pos, freqs, cfg)
    if q.get_device() >= 0:
        refuse_tangents("rotary", q, k, q_weight, k_weight)
    return _forward(q, k, pos, freqs, q_weight, k_weight, *cfg)
