"""Cases and plain forms of the rotary / paged key-value cache operators (``homebrewnlp_mtf_amd.ops.rotary`` and
``homebrewnlp_mtf_amd.ops.paged``): per-head norm and rotary positions of queries and keys with their gradients, block
tables and slot maps from request lengths, the rotated keys and the values written into the pages of a cache, and the
attention of one new token per request over that cache.

``own`` chooses what ``run`` computes: the plain torch form (32 bits, angles in 64) or the framework's operators.

Layouts: keys [pages, kv heads, page, head dim]; values [pages, kv heads, page / 8, head dim, 8] (eight tokens of one
dimension side by side); a token's slot is ``page id * page + offset``; -1 marks a token that has no slot.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
DEV = "cuda"


# ----------------------------------------------------------------------------------------------------------------
# cases
def listed():
    return [
        # ---- rotary: queries and keys of a training step, forward and backward
        # a 1.3B step's attention layer (configs/gpt_neo_1.3b.json: 16 x 2048 tokens, 16 heads x 128), q and k inside
        # the interleaved k|q|v buffer, both normed
        dict(name="rotary_train_kqv", op="rotary", dtype="bf16", B=16, S=2048, Hq=16, Hk=16, D=128, rot=128,
             inter=0, norm=1, packed=1, theta=10000.0, factor=1.0, far=0),
        # the 125M configuration's heads (12 x 64) on an odd batch, interleaved pairs on half of each head, no norm
        dict(name="rotary_train_part", op="rotary", dtype="fp16", B=7, S=1023, Hq=12, Hk=12, D=64, rot=32,
             inter=1, norm=0, packed=0, theta=10000.0, factor=1.0, far=0),
        # few key heads, 96-wide heads, positions far out at a stretched base, in 32 bits
        dict(name="rotary_train_far32", op="rotary", dtype="fp32", B=3, S=1531, Hq=20, Hk=4, D=96, rot=96,
             inter=0, norm=1, packed=0, theta=500000.0, factor=8.0, far=120000),
        # ---- block tables and slot maps
        # one decode step of a served batch: one token each
        dict(name="plan_decode", op="plan", B=64, cached_lo=1, cached_hi=2047, new_lo=1, new_hi=1, page=16, W=128,
             short=0, mix=11),
        # a step that takes in prompts: ragged lengths, and a pool that runs out before the last requests
        dict(name="plan_prompts", op="plan", B=203, cached_lo=0, cached_hi=700, new_lo=0, new_hi=511, page=32, W=64,
             short=1, mix=12),
        # ---- rotated keys and values into the cache
        # one decode step of the server's default batch
        dict(name="append_decode", op="append", dtype="bf16", B=8, cached_lo=1, cached_hi=2047, new_lo=1, new_hi=1,
             Hq=16, Hk=16, D=128, rot=128, inter=0, norm=1, page=16, theta=10000.0, mix=21),
        # prompts of a batch, ragged, continuing cached ones
        dict(name="append_prompts", op="append", dtype="bf16", B=17, cached_lo=0, cached_hi=1500, new_lo=1,
             new_hi=1200, Hq=32, Hk=8, D=128, rot=64, inter=1, norm=0, page=64, theta=10000.0, mix=22),
        # ---- attention of one token per request over the cache
        # the server's default batch on the 1.3B shape, one slot of the batch empty
        dict(name="attn_serve8", op="attn", dtype="bf16", B=8, lo=0, hi=2048, Hq=16, Hk=16, D=128, page=16, mix=31),
        # a full batch with grouped queries and long contexts
        dict(name="attn_grouped_8k", op="attn", dtype="bf16", B=64, lo=4001, hi=8192, Hq=32, Hk=8, D=128, page=64,
             mix=32),
        # one request with a very long context
        dict(name="attn_one_131k", op="attn", dtype="fp16", B=1, lo=131071, hi=131071, Hq=32, Hk=4, D=128, page=128,
             mix=33),
        # 64 heads x 96 (configs/gpt_neo_20b_scale.json), each with its own keys, ragged
        dict(name="attn_heads64x96", op="attn", dtype="bf16", B=19, lo=1, hi=2048, Hq=64, Hk=64, D=96, page=32,
             mix=34),
        # the 125M heads at its short contexts: many small rows
        dict(name="attn_short_64", op="attn", dtype="bf16", B=150, lo=1, hi=130, Hq=12, Hk=12, D=64, page=16, mix=35),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    Hk = rng.choice([1, 2, 4, 8, 12, 16, 20])
    return Hk * rng.choice([1, 1, 2, 4, 8] if Hk <= 8 else [1]), Hk


def draw(rng):
    op = rng.choice(["rotary", "plan", "append", "attn", "attn"])
    mix = rng.randrange(1 << 30)
    if op == "plan":
        hi = rng.choice([1, 1, 4, 100, 1000])
        page = rng.choice([16, 32, 64, 128])
        return dict(op=op, B=_log(rng, 1, 2000 if hi < 100 else 300), cached_lo=0, cached_hi=_log(rng, 16, 8000),
                    new_lo=rng.choice([0, 1]), new_hi=hi, page=page, W=-(-9100 // page), short=rng.choice([0, 0, 1]),
                    mix=mix)
    Hq, Hk = _heads(rng)
    if op == "attn":
        D = rng.choice([32, 64, 96, 128, 128, 256])
        B = _log(rng, 1, 200)
        most = min(131072, max(64, int(1.2e9 / (4 * B * Hk * D))))
        hi = _log(rng, 17, most)
        return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=B, lo=rng.choice([0, 1, max(1, hi // 2)]), hi=hi,
                    Hq=Hq, Hk=Hk, D=D, page=rng.choice([16, 32, 64, 128]), mix=mix)
    D = rng.choice([32, 64, 96, 128, 256])
    c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), Hq=Hq, Hk=Hk, D=D, rot=D if rng.random() < 0.6 else D // 2,
             inter=rng.choice([0, 1]), norm=rng.choice([0, 1]), theta=rng.choice([10000.0, 500000.0]))
    if op == "append":
        hi = rng.choice([1, 1, 50, 900])
        c.update(B=_log(rng, 1, 200 if hi < 100 else 20), cached_lo=0, cached_hi=_log(rng, 16, 2000), new_lo=1,
                 new_hi=hi, page=rng.choice([16, 32, 64, 128]), mix=mix)
        return c
    S = _log(rng, 1, 4096)
    c.update(B=_log(rng, 1, max(1, min(32, int(6e7 / (S * (Hq + Hk) * D))))), S=S,
             packed=rng.choice([0, 1]) if c["dtype"] == "bf16" else 0, factor=rng.choice([1.0, 4.0]),
             far=rng.choice([0, 0, 100000]))
    if rng.random() < 0.2:
        c["dtype"] = "fp32"
    return c


def _between(c, lo, hi, n, salt):
    """n lengths of a case, both ends among them where there is room (the case's own, whatever the seed)"""
    r = random.Random(c["mix"] * 7 + salt)
    v = [r.randint(lo, hi) for _ in range(n)]
    v[r.randrange(n)] = hi
    if n > 1:
        i = r.randrange(n)
        v[i if v[i] != hi or lo == hi else (i + 1) % n] = lo
    return v


def _sizes(c):
    cached = _between(c, c["cached_lo"], c["cached_hi"], c["B"], 1)
    new = _between(c, c["new_lo"], c["new_hi"], c["B"], 2)
    return cached, new


def _cdiv(a, b):
    return -(-a // b)


# ----------------------------------------------------------------------------------------------------------------
# inputs
def _freqs(c):
    i = torch.arange(c["rot"] // 2, dtype=torch.float64, device=DEV)
    return c["theta"] ** (-2.0 * i / c["rot"]) / c.get("factor", 1.0)


def _weights(c, g, dt, s):
    s["wq"] = s["wk"] = None
    if c["norm"]:
        for n in ("wq", "wk"):
            s[n] = (1.0 + 0.1 * torch.randn(c["D"], device=DEV, generator=g)).to(dt)


def _table(c, held, seed, spare):
    """random page ids for requests that hold `held` tokens each: (table rows, unused ids), as lists"""
    page = c["page"]
    need = [_cdiv(n, page) for n in held]
    ids = list(range(sum(need) + spare))
    random.Random(seed * 31 + c["mix"]).shuffle(ids)
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n])
        at += n
    return rows, ids[at:]


def _rect(rows, W, fill=-1):
    return torch.tensor([r + [fill] * (W - len(r)) for r in rows], dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=DEV)
    s = {"case": c}
    if c["op"] == "plan":
        cached, new = _sizes(c)
        want = sum(_cdiv(a + b, c["page"]) - _cdiv(a, c["page"]) for a, b in zip(cached, new))
        rows, unused = _table(c, cached, seed, want + 5)
        n = want * 3 // 4 if c["short"] else want + 5
        P = sum(len(r) for r in rows) + len(unused)
        s.update(cached=torch.tensor(cached, **i32), new=torch.tensor(new, **i32), table=_rect(rows, c["W"]),
                 free=torch.tensor(unused + [0] * (P - len(unused)), **i32), nfree=torch.tensor([n], **i32),
                 tokens=_cdiv(sum(new) + 1, 64) * 64)
        if own:
            from homebrewnlp_mtf_amd.ops import paged
            buf = paged.plan_buffers(c["B"], s["tokens"], DEV)
            # run returns the first row of the height's buffer: [1], as the plain form has it
            s["out"] = buf._replace(nfree=buf.nfree.view(1, 1))
        return s
    dt = TYPES[c["dtype"]]
    D, Hq, Hk = c["D"], c["Hq"], c["Hk"]
    randn = lambda *n: torch.randn(*n, device=DEV, generator=g).to(dt)  # noqa: E731
    if c["op"] == "rotary":
        B, S = c["B"], c["S"]
        if c["packed"]:
            buf = randn(B, S, (2 * Hk + Hq) * D)
            q = buf[..., Hk * D:(Hk + Hq) * D].unflatten(-1, (Hq, D))
            k = buf[..., :Hk * D].unflatten(-1, (Hk, D))
        else:
            q, k = randn(B, S, Hq, D), randn(B, S, Hk, D)
        _weights(c, g, dt, s)
        s.update(q=q.detach(), k=k.detach(), gq=randn(B, S, Hq, D), gk=randn(B, S, Hk, D), freqs=_freqs(c),
                 mscale=1.0 if c["factor"] == 1.0 else 0.1 * math.log(c["factor"]) + 1.0,
                 pos=(torch.arange(S, device=DEV) + c["far"]).expand(B, S).contiguous())
        for n in ("q", "k", "wq", "wk"):
            if s[n] is not None:
                s[n].requires_grad_()
        return s
    if c["op"] == "append":
        cached, new = _sizes(c)
        rows, unused = _table(c, [a + b for a, b in zip(cached, new)], seed, 3)
        P, page = sum(len(r) for r in rows) + len(unused), c["page"]
        slots, pos = [], []
        for a, n, r in zip(cached, new, rows):
            pos += range(a, a + n)
            slots += [r[p // page] * page + p % page for p in range(a, a + n)]
        pad = 1 + (-len(slots) - 1) % 4          # a step's token buffer is rounded up: padding has no slot
        T = len(slots) + pad
        _weights(c, g, dt, s)
        s.update(q=randn(T, Hq, D), k=randn(T, Hk, D), v=randn(T, Hk, D), kc=randn(P, Hk, page, D),
                 vc=randn(P, Hk, page // 8, D, 8), slots=torch.tensor(slots + [-1] * pad, **i32),
                 pos=torch.tensor(pos + [0] * pad, dtype=torch.int64, device=DEV), freqs=_freqs(c), mscale=1.0)
        return s
    lens = _between(c, c["lo"], c["hi"], c["B"], 3)
    rows, unused = _table(c, lens, seed, 2)
    P, page = sum(len(r) for r in rows) + len(unused), c["page"]
    s.update(q=randn(c["B"], Hq, D), kc=randn(P, Hk, page, D), vc=randn(P, Hk, page // 8, D, 8),
             table=_rect(rows, max(1, _cdiv(c["hi"], page))), lens=torch.tensor(lens, **i32), scale=D ** -0.5)
    return s


# ----------------------------------------------------------------------------------------------------------------
# plain forms
def _pairs(x, rot, inter):
    """the two members of every rotated pair"""
    r = x[..., :rot]
    return (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])


def _join(a, b, x, rot, inter):
    r = torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _angles(s):
    a = s["pos"].to(torch.float64)[..., None] * s["freqs"]
    return ((torch.cos(a) * s["mscale"]).float()[..., None, :], (torch.sin(a) * s["mscale"]).float()[..., None, :])


def _normed(x, w):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r * w, r


def _rotated(x, w, cs, c):
    if w is not None:
        x, _ = _normed(x, w.float())
    a, b = _pairs(x, c["rot"], c["inter"])
    return _join(a * cs[0] - b * cs[1], b * cs[0] + a * cs[1], x, c["rot"], c["inter"])


def _rotated_back(x, w, g, cs, c):
    a, b = _pairs(g, c["rot"], c["inter"])
    g = _join(a * cs[0] + b * cs[1], b * cs[0] - a * cs[1], g, c["rot"], c["inter"])
    if w is None:
        return g, None
    w = w.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    dw = (g * n).flatten(0, -2).sum(0)
    g = g * w
    return r * (g - n * (g * n).mean(-1, keepdim=True)), dw


def _plain_rotary(s):
    c, out = s["case"], []
    dt, cs = TYPES[c["dtype"]], _angles(s)
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        out.append(_rotated(x.detach().float(), None if w is None else w.detach(), cs, c).to(dt))
    for x, w, g in ((s["q"], s["wq"], s["gq"]), (s["k"], s["wk"], s["gk"])):
        dx, dw = _rotated_back(x.detach().float(), None if w is None else w.detach(), g.float(), cs, c)
        out += [dx.to(dt)] + ([] if dw is None else [dw.to(dt)])
    return out


def _plain_plan(s):
    c = s["case"]
    page, W, T, B = c["page"], c["W"], s["tokens"], c["B"]
    free, table = s["free"].long(), s["table"]
    cached, new, avail = s["cached"].long(), s["new"].long(), s["nfree"].long()
    old, want = (cached + page - 1) // page, (cached + new + page - 1) // page
    end = new.cumsum(0)
    start = end - new
    wide = (want > W) | (end > T)
    need = torch.where(wide, 0, want - old)
    upto = need.cumsum(0)
    ok = ~wide & ((need == 0) | (upto <= avail))
    taken = torch.where(ok, need, 0)
    # new table entries
    col = torch.arange(W, device=DEV)
    fresh = ok[:, None] & (col >= old[:, None]) & (col < want[:, None])
    src = (avail - 1 - (upto - need)[:, None] - (col - old[:, None])).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[src].int(), table))
    # one slot and position per new token
    t = torch.arange(T, device=DEV)
    row = torch.searchsorted(end, t, right=True).clamp(max=B - 1)
    real = t < end[-1]
    pos = torch.where(real, cached[row] + t - start[row], 0)
    id_ = table[row, (pos // page).clamp(max=W - 1)].long()
    slot = torch.where(real & ok[row], id_ * page + pos % page, -1)
    return {"slots": slot.int(), "pos": pos, "start": torch.cat((start, end[-1:])).int(),
            "lens": torch.where(ok, cached + new, cached).int(), "nfree": (avail - taken.sum()).int(), "table": table}


def _plain_append(s):
    c = s["case"]
    page, dt = c["page"], TYPES[c["dtype"]]
    cs = _angles(s)
    qo = _rotated(s["q"].float(), s["wq"], cs, c).to(dt)
    k = _rotated(s["k"].float(), s["wk"], cs, c).to(dt)
    live = s["slots"] >= 0
    sl = s["slots"].long()[live]
    p, o = sl // page, sl % page
    s["kc"][p, :, o] = k[live]
    s["vc"][p, :, o // 8, :, o % 8] = s["v"][live]
    return [qo, s["kc"], s["vc"]]


def _plain_attn(s):
    c = s["case"]
    B, Hq, Hk, D, page = c["B"], c["Hq"], c["Hk"], c["D"], c["page"]
    W = s["table"].shape[1]
    n = W * page
    out = torch.empty(B, Hq, D, device=DEV, dtype=s["q"].dtype)
    step = max(1, int(2e9 / (n * Hk * D * 4)))     # requests per piece: at most 2 GB of gathered keys
    for b in range(0, B, step):
        e = min(B, b + step)
        id_ = s["table"][b:e].clamp(min=0).long()
        k = s["kc"][id_].float().permute(0, 2, 1, 3, 4).reshape(e - b, Hk, n, D)
        v = s["vc"][id_].float().permute(0, 2, 1, 3, 5, 4).reshape(e - b, Hk, n, D)
        live = (torch.arange(n, device=DEV) < s["lens"][b:e, None])[:, None, None]
        x = torch.matmul(s["q"][b:e].float().view(e - b, Hk, Hq // Hk, D) * s["scale"], k.transpose(-1, -2))
        x = x.masked_fill(~live, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
        den = x.sum(-1, keepdim=True)
        o = torch.matmul(x, v) / torch.where(den > 0, den, 1.0)
        out[b:e] = o.reshape(e - b, Hq, D).to(out.dtype)
    return out


# ----------------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rotary": _plain_rotary, "plan": _plain_plan, "append": _plain_append, "attn": _plain_attn}[c["op"]](s)
    from homebrewnlp_mtf_amd.ops import paged, rotary
    if c["op"] == "rotary":
        q, k, wq, wk = s["q"], s["k"], s["wq"], s["wk"]
        qo, ko = rotary.rotary(q, k, s["pos"], s["freqs"], interleaved=bool(c["inter"]), mscale=s["mscale"],
                               q_weight=wq, k_weight=wk, eps=EPS)
        if wq is None:
            return [qo.detach(), ko.detach(), *torch.autograd.grad((qo, ko), (q, k), (s["gq"], s["gk"]))]
        dq, dwq, dk, dwk = torch.autograd.grad((qo, ko), (q, wq, k, wk), (s["gq"], s["gk"]))
        return [qo.detach(), ko.detach(), dq, dwq, dk, dwk]
    if c["op"] == "plan":
        p = paged.page_plan(s["cached"], s["new"], s["table"], s["free"], s["nfree"], c["page"], out=s["out"])
        return {"slots": p.slots, "pos": p.pos, "start": p.start, "lens": p.lens, "nfree": p.nfree[0],
                "table": s["table"]}
    if c["op"] == "append":
        qo = paged.rotary_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["pos"], s["freqs"],
                                 interleaved=bool(c["inter"]), mscale=s["mscale"], q_weight=s["wq"],
                                 k_weight=s["wk"], eps=EPS)
        return [qo, s["kc"], s["vc"]]
    return paged.paged_attn(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["scale"])


# ----------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "plan":
        cached, new = _sizes(c)
        T = _cdiv(sum(new) + 1, 64) * 64
        pages = sum(_cdiv(a + b, c["page"]) - _cdiv(a, c["page"]) for a, b in zip(cached, new))
        return {"bytes": 4 * (2 * c["B"] + 2) + 8 * pages + 12 * T + 4 * (2 * c["B"] + 2), "flops": 8 * T}
    size = 4 if c["dtype"] == "fp32" else 2
    row = c["D"] * size
    if c["op"] == "rotary":
        T, H = c["B"] * c["S"], c["Hq"] + c["Hk"]
        # forward: in and out; backward: the gradient in and out, and the inputs again where they were normed
        return {"bytes": T * H * row * (5 if c["norm"] else 4) + 16 * T, "flops": T * H * c["D"] * (20 if c["norm"]
                                                                                               else 6)}
    if c["op"] == "append":
        T = sum(_sizes(c)[1])
        return {"bytes": T * (2 * c["Hq"] + 4 * c["Hk"]) * row + 12 * T, "flops": T * (c["Hq"] + c["Hk"]) * c["D"] * 6}
    n = sum(_between(c, c["lo"], c["hi"], c["B"], 3))
    return {"bytes": 2 * n * c["Hk"] * row + 2 * c["B"] * c["Hq"] * row + 4 * _cdiv(n, c["page"]),
            "flops": 4 * n * c["Hq"] * c["D"]}


# ----------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
def _exact_turn(x, w, pos, freqs, mscale, c, sign):
    """x [T, H, D] in 64 bits: the pairs as complex numbers, times mscale * exp(sign i angle)"""
    D, R = c["D"], c["rot"]
    if w is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / D + EPS) ** 0.5 * w
    turn = torch.polar(torch.full((), float(mscale), dtype=torch.float64, device=DEV).expand(pos.numel(), R // 2),
                       sign * torch.outer(pos.double(), freqs))[:, None, :]
    order = torch.arange(R, device=DEV)
    order = order.view(R // 2, 2) if c["inter"] else order.view(2, R // 2).t()
    z = torch.complex(x[..., order[:, 0]].contiguous(), x[..., order[:, 1]].contiguous()) * turn
    y = x.clone()
    y[..., order[:, 0]], y[..., order[:, 1]] = z.real, z.imag
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "plan":
        return _exact_plan(c, s)
    D, page = c["D"], c.get("page")
    if c["op"] == "rotary":
        pos, out = s["pos"].reshape(-1), []
        flat = lambda x: x.detach().reshape(-1, x.shape[-2], D).double()  # noqa: E731
        for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
            y = _exact_turn(flat(x), None if w is None else w.detach().double(), pos, s["freqs"], s["mscale"], c, 1)
            out.append(y.view(x.shape))
        for x, w, g in ((s["q"], s["wq"], s["gq"]), (s["k"], s["wk"], s["gk"])):
            gx = _exact_turn(flat(g), None, pos, s["freqs"], s["mscale"], c, -1)
            if w is None:
                out.append(gx.view(x.shape))
                continue
            x2, w = flat(x), w.detach().double()
            rms = ((x2 ** 2).sum(-1, keepdim=True) / D + EPS) ** 0.5
            wg = gx * w
            dx = wg / rms - x2 * (wg * x2).sum(-1, keepdim=True) / (D * rms ** 3)
            out += [dx.view(x.shape), torch.einsum("thd,thd->d", gx, x2 / rms)]
        return out
    if c["op"] == "append":
        w = [None if s[n] is None else s[n].double() for n in ("wq", "wk")]
        qo = _exact_turn(s["q"].double(), w[0], s["pos"], s["freqs"], s["mscale"], c, 1)
        k = _exact_turn(s["k"].double(), w[1], s["pos"], s["freqs"], s["mscale"], c, 1)
        kc, vc = s["kc"].double(), s["vc"].double()
        for t, sl in enumerate(s["slots"].tolist()):
            if sl >= 0:
                p, o = divmod(sl, page)
                kc[p, :, o] = k[t]
                vc[p, :, o // 8, :, o % 8] = s["v"][t].double()
        return [qo, kc, vc]
    out = torch.zeros(c["B"], c["Hq"], D, dtype=torch.float64, device=DEV)
    G = c["Hq"] // c["Hk"]
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        ids = s["table"][b, :_cdiv(n, page)].long()
        k = s["kc"][ids].double()                                    # [pages, kv heads, page, D]
        v = s["vc"][ids].double().transpose(-1, -2)                  # [pages, kv heads, page / 8, 8, D]
        for h in range(c["Hk"]):
            kh, vh = k[:, h].reshape(-1, D)[:n], v[:, h].reshape(-1, D)[:n]
            p = torch.softmax(s["q"][b, h * G:(h + 1) * G].double() @ kh.t().contiguous() * s["scale"], -1)
            out[b, h * G:(h + 1) * G] = p @ vh
    return out


def _exact_plan(c, s):
    page, W, T = c["page"], c["W"], s["tokens"]
    cached, new, table, free = s["cached"].tolist(), s["new"].tolist(), s["table"].tolist(), s["free"].tolist()
    left = top = int(s["nfree"])
    asked = at = 0
    slots, pos, start, lens = [-1] * T, [0] * T, [], []
    for b, (a, n) in enumerate(zip(cached, new)):
        start.append(at)
        have, want = _cdiv(a, page), _cdiv(a + n, page)
        good = want <= W and at + n <= T
        if good:
            asked += want - have
            good = want == have or asked <= top
        if good:
            for i in range(have, want):
                left -= 1
                table[b][i] = free[left]
        lens.append(a + n if good else a)
        for i in range(n):
            if at + i < T:
                pos[at + i] = a + i
                slots[at + i] = table[b][(a + i) // page] * page + (a + i) % page if good else -1
        at += n
    as_t = lambda x, dt=torch.int32: torch.tensor(x, dtype=dt, device=DEV)  # noqa: E731
    return {"slots": as_t(slots), "pos": as_t(pos, torch.int64), "start": as_t(start + [at]), "lens": as_t(lens),
            "nfree": as_t(left), "table": as_t(table)}
