"""Inputs and 64-bit definitions shared by the rotary / paged-cache tests (written apart from the operators' oracles)."""
import math

import torch

from homebrewnlp_mtf_amd.ops import paged

U32 = 2.0 ** -24          # half a step of fp32, relative


def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def turn64(x, pos, freqs, inter, m, sign=1.0):
    """x [T, H, D] float64"""
    y = x.clone()
    R = 2 * freqs.numel()
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + R // 2)
        ang = pos.double() * freqs[i].double()
        c, s = (torch.cos(ang) * m)[:, None], (torch.sin(ang) * m * sign)[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def rotary64(x, w, pos, freqs, inter, m, eps):
    x = x.double().reshape(-1, *x.shape[-2:])
    if w is not None:
        x = x / ((x ** 2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return turn64(x, pos.reshape(-1), freqs, inter, m)


def rotary_grad64(x, w, g, pos, freqs, inter, m, eps):
    """(dx, dw, sum of |terms| of dw)"""
    g = turn64(g.double().reshape(-1, *g.shape[-2:]), pos.reshape(-1), freqs, inter, m, -1.0)
    if w is None:
        return g, None, None
    x = x.double().reshape(-1, *x.shape[-2:])
    s = ((x ** 2).mean(-1, keepdim=True) + eps).sqrt()
    h = g * w.double()
    dx = h / s - x * (h * x).mean(-1, keepdim=True) / s ** 3
    t = g * x / s
    return dx, t.sum((0, 1)), t.abs().sum((0, 1))


def attn64(q, kc, vc, table, lens, scale, cap=None):
    """(outputs, bound of the error that 32-bit sums and two-part weights leave) in float64, request by request"""
    B, Hq, D = q.shape
    P, Hk, page, _ = kc.shape
    G = Hq // Hk
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    err = torch.zeros_like(out)
    for b in range(B):
        n = min(max(int(lens[b]), 0), table.shape[1] * page, 2 ** 31 if cap is None else cap)
        toks = [(int(table[b, j // page]), j % page) for j in range(n)]
        toks = [t for t in toks if 0 <= t[0] < P]
        if not toks:
            continue
        p = torch.tensor([t[0] for t in toks], device=q.device)
        o = torch.tensor([t[1] for t in toks], device=q.device)
        k, v = kc[p, :, o].double(), vc[p, :, o // 8, :, o % 8].double()          # [n, Hk, D]
        for h in range(Hq):
            kh, vh, qh = k[:, h // G], v[:, h // G], q[b, h].double()
            s = (kh * qh).sum(-1) * scale
            w = torch.softmax(s, 0)
            out[b, h] = w @ vh
            # a score is off by D roundings of its products' sizes and two of its own; a weight by that, the two-part
            # form's 2^-17 and the exponential's few steps; the sums over n tokens by n roundings at most
            ds = (D + 4) * U32 * float(((kh.abs() * qh.abs()).sum(-1) * abs(scale)).max())
            err[b, h] = 2 * (2 * ds + 2.0 ** -17 + (len(toks) + 8) * U32) * (w @ vh.abs())
    return out, err


def make_cache(lens, page, Hk, D, dtype, device, seed=0, spare=2, W=None, garbage=float("nan")):
    """caches whose unused places hold `garbage`, a table with shuffled ids (-1 behind a request's pages)"""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    ids = torch.randperm(P, generator=g).tolist()
    W = W or max(1, max(need))
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    kc = torch.full((P, Hk, page, D), garbage)
    vc = torch.full((P, Hk, page // 8, D, 8), garbage)
    at = 0
    for b, n in enumerate(lens):
        for i in range(need[b]):
            p, m = ids[at], min(page, n - i * page)
            at += 1
            table[b, i] = p
            kc[p, :, :m] = torch.randn(Hk, m, D, generator=g)
            o = torch.arange(m)
            vc[p, :, o // 8, :, o % 8] = torch.randn(m, Hk, D, generator=g)
    return (kc.to(dtype).to(device), vc.to(dtype).to(device), table.to(device),
            torch.tensor(lens, dtype=torch.int32, device=device))


def plan_loop(cached, new, table, stack, nfree, page, T):
    """the block-table rules as a plain loop over Python lists: (slots, pos, start, lens, height, table)"""
    P, W = len(stack), len(table[0])
    table = [list(r) for r in table]
    top = min(max(nfree, 0), P)
    left, asked, at = top, 0, 0
    slots, pos, start, lens = [-1] * T, [0] * T, [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        start.append(at)
        have, want = math.ceil(c / page), math.ceil((c + n) / page)
        ok = want <= W and at + n <= T
        if ok:
            asked += want - have
            ok = want == have or asked <= top
        if ok:
            for i in range(have, want):
                left -= 1
                table[b][i] = stack[left]
        lens.append(c + n if ok else c)
        for i in range(n):
            if at + i < T:
                pos[at + i] = c + i
                if ok:
                    p = table[b][(c + i) // page]
                    slots[at + i] = p * page + (c + i) % page if 0 <= p < P else -1
        at += n
    return slots, pos, start + [at], lens, left, table


def past_31_bits(device):
    """a length that would pass 31 bits is refused, one that just fits is not"""
    def i32(*v):
        return torch.tensor(v, dtype=torch.int32, device=device)
    top = 2 ** 31 - 1
    for new, ok in ((9, True), (10, False)):
        cached, table, stack = i32(top - 9, 3), i32(0, 0, 0, 0, 0, 0).reshape(2, 3), i32(0)
        plan = paged.page_plan(cached, i32(new, 2), table, stack, i32(1), 2 ** 30, tokens=12)
        n = 2 ** 30 - 10                       # offset of the first new token in the second page, whose id is 0
        assert plan.lens.tolist() == [top if ok else top - 9, 5] and plan.nfree.tolist() == [1]
        assert plan.slots.tolist() == ([n + i for i in range(9)] if ok else [-1] * 10) + [3, 4] + [-1] * (10 - new)
        assert plan.start.tolist() == [0, new, new + 2]
