"""A key-value cache in pages, and single-token attention over it (csrc/kernels/paged.hip, rotary.hip; torch oracles on
the CPU).

A pool of ``P`` pages of ``page`` tokens is shared by all requests (one pool per layer, one set of page ids for all
layers). Request b's tokens lie in the pages ``table[b, 0], table[b, 1], ...``; unused ids wait on a stack. One step of
a serving loop, without a read-back to the host:

    plan = page_plan(lens, new, table, stack, height, page, tokens=T)     # pages and slots of the new tokens
    q = rotary_append(q, k, v, k_cache, v_cache, plan.slots, plan.pos, freqs)   # per layer
    o = paged_attn(q, k_cache, v_cache, table, plan.lens, scale)                # per layer, one new token a request

Layouts: keys [P, kv heads, page, D], values [P, kv heads, page / 8, D, 8] (eight tokens of one dim side by side: the
order in which the attention's second product reads them); a token's slot is ``page id * page + offset``.
Ids outside the pool and tokens without a slot are passed over, never followed.
"""
from __future__ import annotations

import typing

import torch

from . import _lib as L
from . import raw
from .rotary import DTYPES, MAX_DIM, check_args, kernel_weights, refuse_tangents, rotary_t, tokens_view

HEAD_DIMS = (32, 64, 96, 128, 256)
PAGES = (16, 32, 64, 128, 256)
_MAX_SLOTS = 2 ** 31 - 1
_MAX_LEN = 2 ** 30


def page_pools(pages: int, page: int, kv_heads: int, dim: int, dtype: torch.dtype,
               device: typing.Union[str, torch.device]) -> typing.Tuple[torch.Tensor, torch.Tensor]:
    """uninitialised (key, value) caches of one layer"""
    if pages < 1 or kv_heads < 1 or dim < 1 or page not in PAGES or pages * page > _MAX_SLOTS:
        raise L.KernelError(f"page_pools: {pages} pages of {page} tokens x {kv_heads} heads x {dim}: pages hold "
                            f"{PAGES} tokens, a pool up to {_MAX_SLOTS}")
    return (torch.empty(pages, kv_heads, page, dim, dtype=dtype, device=device),
            torch.empty(pages, kv_heads, page // 8, dim, 8, dtype=dtype, device=device))


class PagePlan(typing.NamedTuple):
    slots: torch.Tensor     # int32 [T]: slot of each new token, -1: none (refused, or behind the last token)
    pos: torch.Tensor       # int64 [T]: its position in its request (0 behind the last token)
    start: torch.Tensor     # int32 [B + 1]: first token of each request, then all tokens
    lens: torch.Tensor      # int32 [B]: tokens held after the step (unchanged where refused)
    nfree: torch.Tensor     # int32 [1]: height of the stack after the step


def plan_buffers(requests: int, tokens: int, device: typing.Union[str, torch.device]) -> PagePlan:
    """buffers for ``page_plan(out=...)``, for a program that keeps them (a captured graph)"""
    if requests < 1 or tokens < 0:
        raise L.KernelError(f"plan_buffers: {requests} requests, {tokens} tokens")

    def i32(n):
        return torch.empty(n, dtype=torch.int32, device=device)
    return PagePlan(i32(tokens), torch.empty(tokens, dtype=torch.int64, device=device), i32(requests + 1),
                    i32(requests), i32(1))


def _ints(what: str, dev: int, *named):
    for name, t in named:
        if t.dtype != torch.int32 or t.get_device() != dev or not t.is_contiguous():
            raise L.KernelError(f"{what}: {name} must be contiguous int32 beside the other tensors, got {t.dtype} on "
                                f"{t.device}")


def _table(what: str, table, B: int, dev: int) -> typing.Tuple[int, int]:
    """(pages a row, row stride) of a block table"""
    shape, st = table.shape, table.stride()
    if (table.dtype != torch.int32 or table.get_device() != dev or len(shape) != 2 or shape[0] != B or shape[1] < 1
            or (shape[1] > 1 and st[1] != 1) or (B > 1 and not shape[1] <= st[0] < 2 ** 31)):
        raise L.KernelError(f"{what}: the table must be int32 [{B}, pages] with dense rows beside the other tensors, got "
                            f"{table.dtype} {list(shape)} strides {list(st)} on {table.device}")
    return shape[1], st[0] if B > 1 else shape[1]


def _shared(written, read) -> bool:
    """whether one of the written tensors overlaps another one"""
    spans = [(t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
             if t.numel() else None for t in (*written, *read)]
    return any(a and b and a[0] < b[1] and b[0] < a[1] for i, a in enumerate(spans[:len(written)]) for b in spans[i + 1:])


def page_plan(cached: torch.Tensor, new: torch.Tensor, table: torch.Tensor, stack: torch.Tensor, nfree: torch.Tensor,
              page: int, tokens: typing.Optional[int] = None, out: typing.Optional[PagePlan] = None) -> PagePlan:
    """Pages, slots and positions of a step's new tokens, on the device: request b holds ``cached[b]`` tokens and
    appends ``new[b]`` (int32 [B], negative counts as 0); the step's tokens lie one request after the other in a buffer
    of ``tokens`` places. New pages come off the top of ``stack`` (int32 [P], ``nfree`` int32 [1] ids of unused pages, 0 to
    P - 1) and are entered into ``table`` (int32 [B, W]) in place.

    Requests are served in order. One is refused -- no slots, its length unchanged -- if its pages pass W, its length
    31 bits, its tokens the buffer, or the pages asked for by the requests up to and including it ``nfree`` (a request
    that needs no new page goes on). ``cached`` and ``nfree`` are not written: the plan holds their new values, and
    the same call again gives the same plan. What is written (``out``, ``table``) must not share memory with anything else
    here."""
    dev, B = cached.get_device(), cached.numel()
    _ints("page_plan", dev, ("cached", cached), ("new", new), ("stack", stack), ("nfree", nfree))
    if cached.dim() != 1 or B < 1 or new.shape != cached.shape or nfree.numel() != 1 or stack.dim() != 1:
        raise L.KernelError(f"page_plan: cached {list(cached.shape)}, new {list(new.shape)}, stack "
                            f"{list(stack.shape)}, nfree {list(nfree.shape)}")
    W, ld = _table("page_plan", table, B, dev)
    P = stack.numel()
    if page < 1 or P < 1 or P * page > _MAX_SLOTS:
        raise L.KernelError(f"page_plan: a pool of {P} pages of {page} tokens (at most {_MAX_SLOTS} tokens)")
    if out is None:
        if tokens is None:
            raise L.KernelError("page_plan: tokens or out")
        out = plan_buffers(B, tokens, cached.device)
    else:
        _ints("page_plan", dev, ("slots", out.slots), ("start", out.start), ("lens", out.lens), ("out.nfree", out.nfree))
        if (out.pos.dtype != torch.int64 or out.pos.get_device() != dev or not out.pos.is_contiguous()
                or out.pos.shape != out.slots.shape or out.slots.dim() != 1 or out.start.numel() != B + 1
                or out.lens.numel() != B or out.nfree.numel() != 1
                or (tokens is not None and tokens != out.slots.numel())):
            raise L.KernelError("page_plan: out does not fit (plan_buffers)")
    T = out.slots.numel()
    if T >= 2 ** 31:
        raise L.KernelError(f"page_plan: {T} tokens")
    if dev >= 0:
        L.launch(L.lib().obst_page_plan, cached, "page_plan", L.PLAN_DESC.pack(
            cached.data_ptr(), new.data_ptr(), table.data_ptr(), stack.data_ptr(), nfree.data_ptr(),
            out.slots.data_ptr(), out.pos.data_ptr(), out.start.data_ptr(), out.lens.data_ptr(), out.nfree.data_ptr(),
            B, W, ld, page, T, P))
        return out
    # ---- torch oracle
    if _shared((table, *out), (cached, new, stack, nfree)):
        raise L.KernelError("page_plan: out or the table shares memory with another argument")
    avail = min(max(int(nfree), 0), P)
    out.slots.fill_(-1)
    out.pos.zero_()
    at = asked = taken = 0
    for b, (c, n) in enumerate(zip(cached.clamp(min=0).tolist(), new.clamp(min=0).tolist())):
        out.start[b] = min(at, 2 ** 31 - 1)
        old, want = -(-c // page), -(-(c + n) // page)
        ok = want <= W and c + n < 2 ** 31 and at + n <= T
        if ok:
            asked += want - old
            ok = want == old or asked <= avail
            if ok and want > old:
                taken = asked
                ids = stack[avail - asked:avail - asked + want - old].flip(0)
                table[b, old:want] = ids
        out.lens[b] = c + n if ok else c
        m = min(n, T - at)
        if m > 0:
            p = torch.arange(c, c + m)
            out.pos[at:at + m] = p
            if ok:
                ids = table[b, p // page].long()
                slot = torch.where((ids >= 0) & (ids < P), ids * page + p % page, -1)
                out.slots[at:at + m] = slot.int()
        at += n
    out.start[B] = min(at, 2 ** 31 - 1)
    out.nfree[0] = avail - taken
    return out


def page_release(done: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, stack: torch.Tensor, nfree: torch.Tensor,
                 page: int) -> None:
    """Requests that are ``done`` (bool [B]) give their pages back: pushed onto ``stack`` in request order, ``nfree``
    raised and their ``lens`` zeroed, all in place. Ids outside the pool are left out, and a stack that is full takes no
    more."""
    dev, B = lens.get_device(), lens.numel()
    _ints("page_release", dev, ("lens", lens), ("stack", stack), ("nfree", nfree))
    if lens.dim() != 1 or B < 1 or done.shape != lens.shape or done.dtype != torch.bool or done.get_device() != dev \
            or not done.is_contiguous() or nfree.numel() != 1 or stack.dim() != 1 or stack.numel() < 1 or page < 1:
        raise L.KernelError(f"page_release: done bool {list(done.shape)}, lens {list(lens.shape)}, page {page}")
    W, ld = _table("page_release", table, B, dev)
    P = stack.numel()
    if dev >= 0:
        L.launch(L.lib().obst_page_release, lens, "page_release", done.data_ptr(), lens.data_ptr(), table.data_ptr(),
                 stack.data_ptr(), nfree.data_ptr(), B, W, ld, page, P)
        return
    at = min(max(int(nfree), 0), P)
    for b in done.nonzero().flatten().tolist():
        ids = table[b, :min(-(-max(int(lens[b]), 0) // page), W)]
        ids = ids[(ids >= 0) & (ids < P)][:P - at]
        stack[at:at + ids.numel()] = ids
        at += ids.numel()
        lens[b] = 0
    nfree[0] = at


# ----------------------------------------------------------------------------------------------------------------
def _pools(what: str, k_cache, v_cache, q, dev: int, D: int, heads: typing.Optional[int] = None
           ) -> typing.Tuple[int, int, int]:
    """(pages, kv heads, page) of a layer's caches"""
    ks, vs, dt = k_cache.shape, v_cache.shape, q.dtype
    if len(ks) != 4:
        raise L.KernelError(f"{what}: caches [P, heads, page, D] and [P, heads, page / 8, D, 8] (page_pools), got "
                            f"{list(ks)}, {list(vs)}")
    P, H, page, d = ks
    if (vs != (P, H, page // 8, D, 8) or page not in PAGES or P < 1 or d != D or (heads is not None and H != heads)
            or P * page > _MAX_SLOTS):
        raise L.KernelError(f"{what}: caches {list(ks)}, {list(vs)} for heads {heads} x {D}, pages of {PAGES} tokens")
    if (k_cache.dtype != dt or v_cache.dtype != dt or k_cache.get_device() != dev or v_cache.get_device() != dev
            or not k_cache.is_contiguous() or not v_cache.is_contiguous()):
        raise L.KernelError(f"{what}: caches must be contiguous {dt} on the device of q")
    if (k_cache.data_ptr() | v_cache.data_ptr()) % 16 and dev >= 0:
        raise L.KernelError(f"{what}: caches must be 16-byte aligned")
    return P, H, page


def _out(what: str, out, q, shape, dev: int):
    if out is None:
        return q.new_empty(shape)
    if out.shape != shape or out.dtype != q.dtype or out.get_device() != dev or not out.is_contiguous():
        raise L.KernelError(f"{what}: out must be contiguous {q.dtype} {list(shape)} on the device of q")
    return out


def _apart(what: str, out, q, *others) -> None:
    own = out.data_ptr() == q.data_ptr() and q.is_contiguous()
    if _shared((out,), others if own else (q, *others)):
        raise L.KernelError(f"{what}: out shares memory with another argument")


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slots: torch.Tensor, pos: torch.Tensor, freqs: typing.Optional[torch.Tensor],
                  interleaved: bool = False, mscale: float = 1.0, q_weight: typing.Optional[torch.Tensor] = None,
                  k_weight: typing.Optional[torch.Tensor] = None, eps: float = 1e-5,
                  out: typing.Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rotary.rotary`` of a step's tokens with the turned keys and the values written into the cache: q [T, Hq, D],
    k and v [T, Hk, D] (any token and head strides), ``slots`` int32 [T] (outside the pool: neither key nor value is
    written), ``pos`` int64 [T]. Returns the turned queries [T, Hq, D]. ``freqs`` None and no weights: a plain append.
    One launch, no gradient. Tokens of one call must have different slots. ``out`` may be q itself, and shares no memory
    with anything else here."""
    pos, freqs, rot, T = check_args("rotary_append", q, k, pos, freqs, q_weight, k_weight, eps)
    qs, ks, dev = q.shape, k.shape, q.get_device()
    if len(qs) != 3 or v.shape != ks or v.dtype != q.dtype or v.get_device() != dev:
        raise L.KernelError(f"rotary_append: q [T, Hq, D], k and v [T, Hk, D] of one type, got {list(qs)}, {list(ks)}, "
                            f"{list(v.shape)}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_cache.requires_grad
                                    or v_cache.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        raise L.KernelError("rotary_append has no gradient: call it under torch.no_grad()")
    refuse_tangents("rotary_append", q, k, v, k_cache, v_cache, q_weight, k_weight)
    _, Hq, D = qs
    P, Hk, page = _pools("rotary_append", k_cache, v_cache, q, dev, D, ks[1])
    _ints("rotary_append", dev, ("slots", slots))
    if slots.dim() != 1 or slots.numel() != T:
        raise L.KernelError(f"rotary_append: slots {list(slots.shape)} for {T} tokens")
    out = _out("rotary_append", out, q, qs, dev)
    if T == 0 or q.is_meta:
        return out
    if dev >= 0:
        q, q_ts, q_hs = tokens_view(q)
        k, k_ts, k_hs = tokens_view(k)
        v, v_ts, v_hs = tokens_view(v)
        wq, wk, wt = kernel_weights(q_weight, k_weight)
        L.launch(L.lib().obst_rotary_fwd, q, "rotary_append", L.ROT_DESC.pack(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), 0, 0, out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            L.ptr(wq), L.ptr(wk), L.ptr(freqs), pos.data_ptr(), slots.data_ptr(), 0, 0, 0, q_ts, q_hs, k_ts, k_hs, v_ts,
            v_hs, 0, 0, 0, 0, T, P * page, Hq, Hk, D, rot, bool(interleaved), DTYPES[q.dtype], wt, 0, 0, page, mscale,
            eps))
        return out
    # ---- torch oracle
    _apart("rotary_append", out, q, k, v, k_cache, v_cache, slots, pos)
    _scatter_t(rotary_t(k, None if k_weight is None else k_weight.detach(), pos, freqs, interleaved, mscale, eps), v,
               k_cache, v_cache, slots)
    out.copy_(rotary_t(q, None if q_weight is None else q_weight.detach(), pos, freqs, interleaved, mscale, eps))
    return out


def append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    """keys and values [T, Hk, D] as they are into the cache at ``slots`` (as ``rotary_append`` writes them): for prompts
    whose turned keys their own attention has read"""
    ks, dev = k.shape, k.get_device()
    if len(ks) != 3 or v.shape != ks or v.dtype != k.dtype or v.get_device() != dev or ks[1] < 1 \
            or not 1 <= ks[2] <= MAX_DIM:
        raise L.KernelError(f"append: k and v [T, Hk, D] of one type, D up to {MAX_DIM}, got {list(ks)}, {list(v.shape)}")
    if dev >= 0 and k.dtype not in DTYPES:
        raise L.KernelError(f"append: bf16, fp16 or fp32 on the GPU, got {k.dtype}")
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise L.KernelError("append has no gradient: call it under torch.no_grad()")
    refuse_tangents("append", k, v, k_cache, v_cache)
    T, Hk, D = ks
    P, Hk, page = _pools("append", k_cache, v_cache, k, dev, D, Hk)
    _ints("append", dev, ("slots", slots))
    if slots.dim() != 1 or slots.numel() != T:
        raise L.KernelError(f"append: slots {list(slots.shape)} for {T} tokens")
    if T == 0 or k.is_meta:
        return
    if dev >= 0:
        k, k_ts, k_hs = tokens_view(k)
        v, v_ts, v_hs = tokens_view(v)
        L.launch(L.lib().obst_rotary_fwd, k, "append", L.ROT_DESC.pack(
            0, k.data_ptr(), v.data_ptr(), 0, 0, 0, k_cache.data_ptr(), v_cache.data_ptr(), 0, 0, 0, 0, slots.data_ptr(), 0,
            0, 0, 0, 0, k_ts, k_hs, v_ts, v_hs, 0, 0, 0, 0, T, P * page, 0, Hk, D, 0, 0, DTYPES[k.dtype], 0, 0, 0, page,
            1.0, 1.0))
        return
    _scatter_t(k, v, k_cache, v_cache, slots)


def _scatter_t(k, v, k_cache, v_cache, slots):
    P, _, page, _ = k_cache.shape
    live = (slots >= 0) & (slots < P * page)
    s = slots[live].long()
    k_cache[s // page, :, s % page] = k[live]
    v_cache[s // page, :, s % page // 8, :, s % 8] = v[live]


# ----------------------------------------------------------------------------------------------------------------
def paged_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
               scale: float, max_len: typing.Optional[int] = None, out: typing.Optional[torch.Tensor] = None
               ) -> torch.Tensor:
    """Attention of one new token per request over its pages: q [B, Hq, D] (batch and head strides free), caches as
    ``page_pools`` makes them with Hq a multiple of their heads (query heads h * G .. h * G + G - 1 read key head h),
    ``table`` int32 [B, W], ``lens`` int32 [B] the tokens that count, the new one among them:

        out[b, h] = softmax_j(scale * q[b, h] . k_j) @ v,  j < min(lens[b], max_len)
        0 for a request without tokens, or with -inf for every score

    ``max_len`` (default: what the table's width holds) is a bound on lens that the host knows; a close one spares a wide
    table some empty blocks and workspace. A page id outside the pool hides its tokens. What the cache holds behind a length
    is never looked at. Infinities and NaN among the values that count stay in their dims, as the formula has them (a weight
    too small for 32 bits is 0, and makes an infinite value NaN). ``out`` may be q itself, and shares no memory with anything
    else here. No gradient."""
    qs, dev = q.shape, q.get_device()
    if len(qs) != 3 or qs[1] < 1 or qs[2] < 1:
        raise L.KernelError(f"paged_attn: q must be [B, heads, D], got {list(qs)}")
    B, Hq, D = qs
    P, Hk, page = _pools("paged_attn", k_cache, v_cache, q, dev, D)
    if Hk < 1 or Hq % Hk:
        raise L.KernelError(f"paged_attn: {Hq} query heads over {Hk} key heads")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise L.KernelError("paged_attn has no gradient: call it under torch.no_grad()")
    refuse_tangents("paged_attn", q, k_cache, v_cache)
    W, ld = _table("paged_attn", table, B, dev)
    _ints("paged_attn", dev, ("lens", lens))
    if lens.dim() != 1 or lens.numel() != B:
        raise L.KernelError(f"paged_attn: lens {list(lens.shape)} for {B} requests")
    cap = W * page
    if max_len is not None:
        if max_len < 0:
            raise L.KernelError(f"paged_attn: max_len {max_len}")
        cap = min(cap, max_len)
    if cap > _MAX_LEN:
        raise L.KernelError(f"paged_attn: {cap} tokens a request (at most {_MAX_LEN}; max_len bounds a wide table)")
    out = _out("paged_attn", out, q, qs, dev)
    if B == 0 or q.is_meta:
        return out
    if dev >= 0:
        rows = Hk * (-(-Hq // Hk // 16))
        if D not in HEAD_DIMS or q.dtype not in (torch.bfloat16, torch.float16):
            raise L.KernelError(f"paged_attn: heads of {HEAD_DIMS} in bf16 or fp16 on the GPU, got {D} in {q.dtype}")
        if B > 65535 or rows > 65535:
            raise L.KernelError(f"paged_attn: {B} requests x {Hk} heads (at most 65535 each)")
        q_bs, q_hs, q_ds = q.stride()
        if q_ds != 1 or (q_bs | q_hs) % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            q_bs, q_hs = Hq * D, D
        nsplit, split, most = _splits(B, rows, cap)
        part = q.new_empty(B * Hq * nsplit * (D + 2), dtype=torch.float32) if nsplit > 1 else None
        L.launch(L.lib().obst_paged_attn, q, "paged_attn", L.PAGED_DESC.pack(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr(),
            L.ptr(part), q_bs, q_hs, B, Hq, Hk, D, P, cap, ld, page.bit_length() - 1, DTYPES[q.dtype], nsplit, split,
            most, scale))
        return out
    # ---- torch oracle
    _apart("paged_attn", out, q, k_cache, v_cache, table, lens)
    G = Hq // Hk
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        ids = table[b, :-(-n // page)].long()
        ok = (ids >= 0) & (ids < P)
        live = ok.repeat_interleave(page)[:n]
        ids = torch.where(ok, ids, 0)
        kk = k_cache[ids].transpose(1, 2).reshape(-1, Hk, D)[:n][live]
        vv = v_cache[ids].permute(0, 2, 4, 1, 3).reshape(-1, Hk, D)[:n][live]
        if kk.shape[0] == 0:
            out[b] = 0
            continue
        s = torch.einsum("hgd,jhd->hgj", raw._f(q[b]).reshape(Hk, G, D), raw._f(kk)) * scale
        o = torch.einsum("hgj,jhd->hgd", torch.softmax(s, -1), raw._f(vv))
        out[b] = o.masked_fill(s.amax(-1, keepdim=True) == float("-inf"), 0).reshape(Hq, D)
    return out


def _splits(B: int, rows: int, cap: int) -> typing.Tuple[int, int, int]:
    """(splits of the length, tokens a split, ``most``) for B requests of ``rows`` blocks each without a split.

    Up to 16 requests (``most`` > 0): the kernel sizes the splits from the lengths it finds, at least 256 tokens each
    and three blocks a CU from all of them, so no request has more than ``most`` splits and the table's width hardly
    matters (8 requests of 1 to 2000 tokens, 8 key heads: 12.3 us in a table of 2000, 14.7 in one of 131072; 4 of 1 to
    30000: 53 us, 59 in two blocks a CU, 57 in four). One request's splits are all alike: two blocks a CU (131072
    tokens, 4 key heads: 46.7 us with the join, 48.3 in three). A table so narrow that its splits are the shortest either
    way spares the kernel that sum, 0.6 us.

    More requests would start too many empty blocks that way (32 of 1 to 2000 in a table of 131072: 42 us, 33 by the
    width), so the width decides: four blocks a CU, 384 to 2048 tokens a split (64 of 6144, 8 key heads: 248 us, 275
    in splits of 512; 200 of 1 to 2000, 1 key head: 28 us, 31 in two blocks a CU), and longer splits where that makes
    more than 65536 blocks (1000 of 1 to 500 in a table of 131072: 201 us, 395 in splits of 2048; 256, one of them of
    120000: 209, 168). At most 1024 splits (csrc/kernels/paged.hip MAX_SPLITS)."""
    if B <= 16:
        blocks = 512 if B == 1 else 768
        most = max(1, blocks // rows) if cap * rows * B > blocks * 256 else 0
        split = max(256, -(-cap // 1024))
    else:
        most, split = 0, max(384, min(-(-cap * rows * B // 1024), 2048), -(-cap // max(1, 65536 // (B * rows))),
                             -(-cap // 1024))
    split = -(-split // 128) * 128
    n = max(1, -(-cap // split))
    return min(n, most) if most else n, split, most
