"""Rotary and paged-cache HIP kernels against 64-bit definitions (tests/paged_cases.py), at the sizes, layouts and
lengths where they can go wrong; captured graphs; other streams."""
import random

import pytest
import torch

from homebrewnlp_mtf_amd.ops import _lib as L
from homebrewnlp_mtf_amd.ops import paged, rotary
from paged_cases import U32, attn64, half_step, make_cache, past_31_bits, plan_loop, rotary64, rotary_grad64
from test_rotary_paged_cpu import random_plan, run_plan

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def close_rows(y, ref, dtype, extra=0.0):
    """within half a step of the output type plus (32 + D) roundings of fp32 at the size of the row: a row is a chain of
    one sum over D, a reciprocal root, two products and a rotation"""
    ref = ref.reshape(y.shape)
    size = ref.abs().amax(-1, keepdim=True)
    tol = half_step(dtype) * ref.abs() + (32 + y.shape[-1]) * U32 * size + extra
    if dtype == HF:
        tol = tol + 2.0 ** -25                     # half a step of its subnormals
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((y.double() - ref).abs().max())}"


def near(y, ref, tol):
    """NaN exactly where the definition gives NaN (tokens that were never written), the rest within tol"""
    off = (y.double() - ref).abs()
    return bool(torch.equal(torch.isnan(y), torch.isnan(ref))) and bool(((off <= tol) | torch.isnan(ref)).all())


# (q heads, k heads, D, rot, token gap): vectorised and scalar layouts, tails, odd widths, one to many lanes a head
ROT = [(2, 1, 128, 128, 0), (16, 16, 128, 64, 0), (3, 5, 64, 64, 8), (12, 4, 96, 96, 0), (4, 4, 96, 48, 0),
       (1, 1, 256, 256, 0), (2, 2, 512, 256, 0), (5, 1, 32, 8, 0), (3, 2, 80, 32, 0), (2, 3, 33, 16, 0),
       (1, 2, 1, 0, 0), (2, 1, 6, 6, 1), (1, 1, 511, 510, 0), (40, 8, 128, 128, 0), (3, 1, 24, 16, 0),
       (7, 7, 64, 0, 0)]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("Hq,Hk,D,rot,gap", ROT)
def test_rotary_forward_backward(cuda, Hq, Hk, D, rot, gap, dtype, inter):
    g = gen(cuda, D * 7 + Hq)
    B, S = 3, 7
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g).to(dtype)  # noqa: E731
    buf = rnd(B, S, (Hq + Hk) * D + gap)
    k = buf[..., :Hk * D].unflatten(-1, (Hk, D)).detach().requires_grad_()
    q = buf[..., Hk * D:(Hk + Hq) * D].unflatten(-1, (Hq, D)).detach().requires_grad_()
    pos = torch.randint(-3, 130000, (B, S), device=cuda, generator=g)
    freqs = rotary.rotary_freqs(rot, device=cuda)[0] if rot else None
    f64 = freqs if rot else torch.zeros(0, dtype=torch.float64, device=cuda)
    for wq, wk in ((rnd(D) + 1, rnd(D) + 1), (None, rnd(D)), (None, None)):
        ws = [None if w is None else w.requires_grad_() for w in (wq, wk)]
        qo, ko = rotary.rotary(q, k, pos, freqs, interleaved=inter, mscale=1.2, q_weight=ws[0], k_weight=ws[1])
        gq, gk = rnd(B, S, Hq, D), rnd(B, S, Hk, D)
        leaves = [t for t in (q, k, *ws) if t is not None]
        grads = dict(zip(map(id, leaves), torch.autograd.grad((qo, ko), leaves, (gq, gk))))
        for x, w, y, gg in ((q, ws[0], qo, gq), (k, ws[1], ko, gk)):
            w64 = None if w is None else w.detach()
            close_rows(y.detach(), rotary64(x.detach(), w64, pos, f64, inter, 1.2, 1e-5), dtype)
            dx, dw, mag = rotary_grad64(x.detach(), w64, gg, pos, f64, inter, 1.2, 1e-5)
            # dx is a difference of h and its projection: roundings count at the size of the larger, |h| r
            r = 1.0 if w is None else ((x.detach().double() ** 2).mean(-1, keepdim=True) + 1e-5).rsqrt()
            h = gg.double().abs().amax(-1, keepdim=True) * 1.7 * (1.0 if w is None else float(w64.abs().max()))
            close_rows(grads[id(x)], dx, dtype, extra=(32 + D) * U32 * h * r * (1 + D ** 0.5))
            if w is not None:
                # every term off by D + 16 roundings; at most 100 additions in a row to one sum (2 in a lane, 6 over
                # lanes, 4 over waves, the rest over blocks)
                tol = half_step(dtype) * dw.abs() + (D + 116) * U32 * mag + (2.0 ** -25 if dtype == HF else 0)
                assert bool(((grads[id(w)].double() - dw).abs() <= tol).all())


def test_rotary_many_tokens(cuda):
    """more units than waves (the grid-stride loop) and weight sums over many blocks, twice: the same bits"""
    g = gen(cuda, 11)
    T, H, D = 20011, 4, 64
    q, k = (torch.randn(T, h, D, device=cuda, generator=g).to(BF).requires_grad_() for h in (H, 1))
    wq, wk = (torch.randn(D, device=cuda, generator=g).requires_grad_() for _ in range(2))
    gq, gk = torch.randn(T, H, D, device=cuda, generator=g).to(BF), torch.randn(T, 1, D, device=cuda, generator=g).to(BF)
    freqs, pos = rotary.rotary_freqs(D, device=cuda)[0], torch.arange(T, device=cuda)
    runs = []
    for _ in range(2):
        o = rotary.rotary(q, k, pos, freqs, q_weight=wq, k_weight=wk)
        runs.append([*o, *torch.autograd.grad(o, (q, k, wq, wk), (gq, gk))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    close_rows(runs[0][0].detach(), rotary64(q.detach(), wq.detach(), pos, freqs, False, 1.0, 1e-5), BF)
    _, dw, mag = rotary_grad64(q.detach(), wq.detach(), gq, pos, freqs, False, 1.0, 1e-5)
    # fp32 weights: additions in a row to one sum are at most T H / (lanes' heads, waves) + 6 + 4 + blocks
    assert bool(((runs[0][4].double() - dw).abs() <= (D + 16 + 1100) * U32 * mag + U32 * dw.abs()).all())


def test_rotary_layouts(cuda):
    """broadcast keys, expanded gradients, permuted and misaligned inputs, broadcast positions"""
    g = gen(cuda, 12)
    freqs = rotary.rotary_freqs(64, device=cuda)[0]
    pos = torch.arange(5, device=cuda)
    base = torch.randn(2, 4, 5, 64, device=cuda, generator=g).to(BF)
    odd = torch.randn(2 * 5 * 4 * 64 + 1, device=cuda, generator=g).to(BF)[1:].view(2, 5, 4, 64)
    for q in (base.transpose(1, 2), odd):
        k = torch.randn(1, 5, 2, 64, device=cuda, generator=g).to(BF).requires_grad_()
        qo, ko = rotary.rotary(q, k.expand(2, 5, 2, 64), pos, freqs)
        p2 = pos.expand(2, 5)
        close_rows(qo, rotary64(q, None, p2.reshape(-1), freqs, False, 1.0, 1e-5), BF)
        close_rows(ko.detach(), rotary64(k.detach().expand(2, 5, 2, 64), None, p2.reshape(-1), freqs, False, 1.0, 1e-5), BF)
        dk, = torch.autograd.grad(ko.float().sum(), k)          # an expanded (stride 0) gradient arrives
        ref = rotary_grad64(k.detach().cpu(), None, torch.ones(1, 5, 2, 64), pos.cpu(), freqs.cpu(), False, 1.0, 1e-5)
        # two equal bf16 rows are added: their sum in bf16 is exact
        assert bool(((dk.cpu().double() - 2 * ref[0].reshape(dk.shape)).abs()
                     <= 2 * (half_step(BF) * ref[0].abs() + 200 * U32).reshape(dk.shape)).all())


def test_rotary_main_grad(cuda):
    g = gen(cuda, 13)
    q, k = (torch.randn(9, 2, 64, device=cuda, generator=g).to(BF) for _ in range(2))
    freqs, pos = rotary.rotary_freqs(64, device=cuda)[0], torch.arange(9, device=cuda)
    a, b = (torch.rand(64, device=cuda, generator=g).to(BF).requires_grad_() for _ in range(2))
    for wq, wk in ((a, b), (a, a)):
        for w in (a, b):
            w.main_grad = torch.ones(64, device=cuda)
            w.master = w.detach().float() + 0.001          # the kernel reads the fp32 copy
        o = rotary.rotary(q, k, pos, freqs, q_weight=wq, k_weight=wk)
        (o[0].float().sum() + o[1].float().sum()).backward()
        one = torch.ones(9, 2, 64)
        ref = {id(w): 1.0 for w in (wq, wk)}
        tol = {id(w): 0.0 for w in (wq, wk)}
        for x, w in ((q, wq), (k, wk)):
            _, dw, mag = rotary_grad64(x.cpu(), w.master.cpu(), one, pos.cpu(), freqs.cpu(), False, 1.0, 1e-5)
            ref[id(w)] = ref[id(w)] + dw
            tol[id(w)] = tol[id(w)] + (64 + 120) * U32 * mag + 4 * U32 * (1 + dw.abs())
        for w in (wq, wk):
            assert w.grad is None
            assert bool(((w.main_grad.cpu().double() - ref[id(w)]).abs() <= tol[id(w)]).all())
        for w in (a, b):
            del w.main_grad, w.master


def test_rotary_refuses_types(cuda):
    x = torch.zeros(2, 1, 8, device=cuda, dtype=torch.float64)
    with pytest.raises(L.KernelError):
        rotary.rotary(x, x, torch.arange(2, device=cuda), None)
    y = x.float()
    with pytest.raises(L.KernelError):
        rotary.rotary(y, y, torch.arange(2), None)
    with pytest.raises(L.KernelError):
        rotary.rotary(y, y.cpu(), torch.arange(2, device=cuda), None)
    e = rotary.rotary(y[:0], y[:0], torch.arange(0, device=cuda), None)
    assert e[0].shape == (0, 1, 8)
    w = torch.ones(8, device=cuda, requires_grad=True)
    o = rotary.rotary(y[:0], y[:0], torch.arange(0, device=cuda), None, q_weight=w)
    assert torch.equal(torch.autograd.grad(o[0].sum(), w)[0], torch.zeros(8, device=cuda))


# ----------------------------------------------------------------------------------------------------------------
def test_plan_random(cuda):
    r = random.Random(14)
    for _ in range(60):
        c = random_plan(r)
        assert run_plan(cuda, *c) == tuple(plan_loop(*c)), c


@pytest.mark.parametrize("B,T,n", [(1, 40000, 39990), (1000, 1000, 1), (4099, 6000, 2), (257, 70000, 200), (3, 0, 0),
                                   (2, 70000, 5)])
def test_plan_sizes(cuda, B, T, n):
    r = random.Random(B)
    page, W = 16, -(-(n + 100) // 16)
    cached, new = [r.randint(0, 90) for _ in range(B)], [r.randint(0, n) for _ in range(B)]
    need = sum(-(-(c + m) // page) - -(-c // page) for c, m in zip(cached, new))
    P = need + 7
    stack = list(range(P))
    r.shuffle(stack)
    table = [[r.randrange(P) for _ in range(W)] for _ in range(B)]
    for height in (P, need * 2 // 3):
        c = (cached, new, table, stack, height, page, T)
        assert run_plan(cuda, *c) == tuple(plan_loop(*c))


def test_plan_strided_table_and_overflow(cuda):
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    wide = torch.full((3, 9), -7, dtype=torch.int32, device=cuda)
    table = wide[:, 2:6]
    big = 2 ** 31 - 1
    p = paged.page_plan(i([big, 0, 3]), i([big, 20, big]), table, i([5, 4, 3, 2, 1, 0]), i([6]), 16, tokens=50)
    # 2^31 tokens pass the table's width, and all tokens behind them the buffer
    assert p.lens.tolist() == [big, 0, 3] and int(p.nfree) == 6 and p.slots.tolist() == [-1] * 50
    assert p.start.tolist() == [0, big, big, big] and bool((wide == -7).all())
    p = paged.page_plan(i([0, 0, 3]), i([0, 20, 1]), table, i([5, 4, 3, 2, 1, 0]), i([6]), 16, tokens=50)
    assert wide[1, 2:4].tolist() == [0, 1] and bool((wide[:, :2] == -7).all()) and bool((wide[:, 6:] == -7).all())
    assert p.lens.tolist() == [0, 20, 4] and int(p.nfree) == 4


def test_plan_refuses_lengths_past_31_bits(cuda):
    past_31_bits(cuda)


def test_release_more_pages_than_31_bits(cuda):
    """1024 rows of 2^21 + 1 pages each: the stack takes what it has room for, what lies behind it stays"""
    B, W, P = 1024, 2 ** 21 + 1, 1000
    table = torch.zeros(B, W, dtype=torch.int32, device=cuda)
    table[0, :P] = torch.arange(P, device=cuda).int() + 7
    room = torch.full((P + 64,), -5, dtype=torch.int32, device=cuda)
    lens = torch.full((B,), W, dtype=torch.int32, device=cuda)
    nfree = torch.tensor([10], dtype=torch.int32, device=cuda)
    paged.page_release(torch.ones(B, dtype=torch.bool, device=cuda), lens, table, room[:P], nfree, 1)
    assert nfree.tolist() == [P] and bool((lens == 0).all())
    assert room.tolist() == [-5] * 10 + [i + 7 for i in range(P - 10)] + [-5] * 64


def test_release(cuda):
    r = random.Random(15)
    for B in (1, 7, 1024, 2500):
        W, page, P = 6, 16, B * 4
        lens = [r.choice([0, r.randint(1, W * page), 10 ** 9, -5]) for _ in range(B)]
        table = [[r.randrange(P) for _ in range(W)] for _ in range(B)]
        done = [r.random() < 0.6 for _ in range(B)]
        out = []
        for dev in ("cpu", cuda):
            i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
            a = (torch.tensor(done, device=dev), i(lens), i(table), i([-1] * P), i([B // 2]))
            paged.page_release(*a, page)
            out.append([t.tolist() for t in a[1:]])
        assert out[0] == out[1]


# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("Hq,Hk,D,rot,page,inter,norm", [
    (2, 2, 128, 128, 16, False, True), (8, 1, 64, 32, 32, True, False), (3, 3, 96, 96, 64, False, True),
    (20, 4, 256, 256, 128, True, True), (2, 1, 32, 0, 256, False, False), (1, 1, 33, 8, 16, False, True),
    (32, 8, 128, 64, 64, True, False), (4, 2, 512, 512, 16, False, True)])
@pytest.mark.parametrize("T", [1, 37, 300, 1500])
def test_append(cuda, T, Hq, Hk, D, rot, page, inter, norm, dtype):
    g = gen(cuda, T + D)
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g).to(dtype)  # noqa: E731
    buf = rnd(T, (Hq + 2 * Hk) * D)
    q = buf[:, :Hq * D].unflatten(1, (Hq, D))
    k = buf[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
    v = buf[:, (Hq + Hk) * D:].unflatten(1, (Hk, D))
    P = -(-T // page) + 3
    kc, vc = paged.page_pools(P, page, Hk, D, dtype, cuda)
    kc.fill_(3)
    vc.fill_(3)
    r = random.Random(T)
    # runs of neighbouring slots from any offset, as prompts have them, single ones, none, and slots outside the pool
    at, slots = r.randrange(page), []
    while len(slots) < T:
        n = r.choice([1, 3, 40])
        slots += range(at, at + n)
        at += n + r.choice([0, 0, 5])
    slots = [s if s < P * page else -1 for s in slots[:T]]
    for i in range(0, T, 11):
        slots[i] = r.choice([-1, P * page, 2 ** 31 - 1, -2 ** 31])
    st = torch.tensor(slots, dtype=torch.int32, device=cuda)
    pos = torch.randint(0, 130000, (T,), device=cuda, generator=g)
    freqs = rotary.rotary_freqs(rot, device=cuda)[0] if rot else None
    f64 = freqs if rot else torch.zeros(0, dtype=torch.float64, device=cuda)
    w = [rnd(D) + 1 if norm else None for _ in range(2)]
    qo = paged.rotary_append(q, k, v, kc, vc, st, pos, freqs, interleaved=inter, mscale=1.1, q_weight=w[0], k_weight=w[1])
    close_rows(qo, rotary64(q, w[0], pos, f64, inter, 1.1, 1e-5), dtype)
    live = (st >= 0) & (st < P * page)
    s = st[live].long()
    kd, vd = kc.permute(0, 2, 1, 3).reshape(P * page, Hk, D), vc.permute(0, 2, 4, 1, 3).reshape(P * page, Hk, D)
    close_rows(kd[s], rotary64(k, w[1], pos, f64, inter, 1.1, 1e-5)[live], dtype)
    assert torch.equal(vd[s], v[live])
    rest = torch.ones(P * page, dtype=torch.bool, device=cuda)
    rest[s] = False
    assert bool((kd[rest] == 3).all()) and bool((vd[rest] == 3).all())


# ----------------------------------------------------------------------------------------------------------------
ATTN = [  # Hq, Hk, D, page, lens
    (16, 16, 128, 16, [0, 1, 15, 16, 17, 31, 32, 33, 500]),
    (32, 8, 128, 64, [129, 0, 1000, 64, 2049]),
    (2, 1, 64, 32, [1, 300, 257, 256, 255]),
    (12, 12, 64, 16, [7]),
    (64, 64, 96, 32, [40, 3]),
    (5, 1, 96, 128, [700, 0]),
    (40, 2, 128, 16, [100, 513]),            # 20 query heads a key head: two groups of columns
    (17, 1, 32, 256, [1000]),
    (8, 4, 256, 64, [65, 320, 1]),
    (1, 1, 32, 16, [0, 0]),
    (32, 2, 256, 32, [70, 0, 300]),          # the most shared memory a block takes: 16 heads of 256
    (4, 1, 128, 128, [20000]),               # many splits
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,Hk,D,page,lens", ATTN)
def test_attn(cuda, Hq, Hk, D, page, lens, dtype):
    kc, vc, table, ln = make_cache(lens, page, Hk, D, dtype, cuda, seed=D + Hq, W=-(-max(lens + [1]) // page) + 1)
    q = torch.randn(len(lens), Hq, D, device=cuda, generator=gen(cuda, 3)).to(dtype)
    ref, err = attn64(q, kc, vc, table, ln, D ** -0.5)
    tol = half_step(dtype) * ref.abs() + err
    for kw in ({}, {"max_len": max(lens)}):
        o = paged.paged_attn(q, kc, vc, table, ln, D ** -0.5, **kw)
        assert near(o, ref, tol)
        for b, n in enumerate(lens):
            assert n or bool((o[b] == 0).all())


@pytest.mark.parametrize("Hq,Hk,lens,W", [
    (8, 2, [3000], 2000),                                    # one request in a table of 32000 tokens
    (8, 8, [1, 9000, 0, 17, 300, 128, 129, 2], 4096),        # a long one among short ones: splits sized by the kernel
    (4, 1, [700] * 15 + [20000], 4096),
    (4, 1, [700] * 16 + [20000], 4096),                      # one request more: sized by the width
    (64, 64, [1500, 5], 1024),
    (600, 600, [400, 0, 1000], 512),                         # more heads than blocks asked for: no split
])
def test_attn_wide_tables(cuda, Hq, Hk, lens, W):
    """a table much wider than its requests, and lengths that differ much"""
    D, page = 64, 16
    kc, vc, table, ln = make_cache(lens, page, Hk, D, BF, cuda, seed=Hq, W=W)
    q = torch.randn(len(lens), Hq, D, device=cuda, generator=gen(cuda, 3)).to(BF)
    ref, err = attn64(q, kc, vc, table, ln, D ** -0.5)
    tol = half_step(BF) * ref.abs() + err
    a = paged.paged_attn(q, kc, vc, table, ln, D ** -0.5)
    assert near(a, ref, tol) and near(paged.paged_attn(q, kc, vc, table, ln, D ** -0.5, max_len=max(lens)), ref, tol)
    assert torch.equal(a, paged.paged_attn(q, kc, vc, table, ln, D ** -0.5))


def test_attn_hidden_ids_bounds_strides(cuda):
    lens = [70, 33, 16, 200, 500]
    kc, vc, table, ln = make_cache(lens, 16, 2, 64, BF, cuda, seed=5)
    P = kc.shape[0]
    table[0, 2] = P
    table[1, 0] = -1
    table[2, 0] = 2 ** 31 - 1
    table[3, 12] = -2 ** 31
    table[4, ::2] = P + 5
    buf = torch.randn(5, 4 * 64 * 2, device=cuda, generator=gen(cuda, 6)).to(BF)
    q = buf[:, 128:128 + 256].unflatten(1, (4, 64))
    wide = torch.full((5, table.shape[1] + 7), -9, dtype=torch.int32, device=cuda)
    wide[:, 3:3 + table.shape[1]] = table
    for cap in (None, 100, 16, 0, 10 ** 9):
        ref, err = attn64(q, kc, vc, table, ln, 0.2, cap=cap)
        o = paged.paged_attn(q, kc, vc, wide[:, 3:3 + table.shape[1]], ln, 0.2, max_len=cap)
        assert near(o, ref, half_step(BF) * ref.abs() + err)
        assert bool((o[2] == 0).all())
    # lengths past the table, negative ones; queries of other strides and alignment
    far = torch.tensor([2 ** 31 - 1, -4, 16, 200, 500], dtype=torch.int32, device=cuda)
    odd = torch.empty(5 * 256 + 1, dtype=BF, device=cuda)[1:].view(5, 4, 64).copy_(q)
    for qq in (odd, q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(1, 2).contiguous().transpose(1, 2)):
        ref, err = attn64(qq, kc, vc, table, far, 0.2)
        o = paged.paged_attn(qq, kc, vc, table, far, 0.2)
        assert near(o, ref, half_step(BF) * ref.abs() + err)
        assert bool((o[1] == 0).all())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_attn_extreme_scores(cuda, dtype):
    """one key far above the rest, equal scores, scores that grow along the length, scale 0, -inf and NaN keys"""
    lens = [300, 300, 300]
    kc, vc, table, ln = make_cache(lens, 32, 1, 64, dtype, cuda, seed=9)
    q = torch.ones(3, 2, 64, device=cuda, dtype=dtype)
    for j in range(300):
        p, o = int(table[1, j // 32]), j % 32
        kc[p, 0, o] = 0.25
        p = int(table[2, j // 32])
        kc[p, 0, o] = j / 16
    kc[int(table[0, 4]), 0, 3] = 60
    for scale in (1.0, 0.0, -0.5):
        ref, err = attn64(q, kc, vc, table, ln, scale)
        o = paged.paged_attn(q, kc, vc, table, ln, scale)
        assert near(o, ref, half_step(dtype) * ref.abs() + err)
    kc[int(table[0, 1]), 0, 0] = float("-inf")           # hidden by its own score
    kc[int(table[1, 1]), 0, 0] = float("nan")
    o = paged.paged_attn(q, kc, vc, table, ln, 1.0)
    assert bool(torch.isfinite(o[0]).all()) and bool(torch.isnan(o[1]).all()) and bool(torch.isfinite(o[2]).all())


def test_attn_offsets_past_32_bits(cuda):
    """a pool of more than 2^31 elements: pages behind that offset"""
    P, page, Hk, D = 66000, 256, 1, 128
    kc, vc = paged.page_pools(P, page, Hk, D, BF, cuda)
    g = gen(cuda, 21)
    ids = [65999, 65537, 1]
    for i in ids:
        kc[i] = torch.randn(Hk, page, D, device=cuda, generator=g).to(BF)
        vc[i] = torch.randn(Hk, page // 8, D, 8, device=cuda, generator=g).to(BF)
    table = torch.tensor([ids], dtype=torch.int32, device=cuda)
    ln = torch.tensor([600], dtype=torch.int32, device=cuda)
    q, k, v = (torch.randn(1, h, D, device=cuda, generator=g).to(BF) for h in (2, 1, 1))
    slot = torch.tensor([65537 * page + 255], dtype=torch.int32, device=cuda)
    with torch.no_grad():
        qo = paged.rotary_append(q, k, v, kc, vc, slot, torch.zeros(1, dtype=torch.int64, device=cuda), None)
    assert torch.equal(kc[65537, :, 255], k[0]) and torch.equal(vc[65537, :, 31, :, 7], v[0]) and torch.equal(qo, q)
    ref, err = attn64(q, kc, vc, table, ln, D ** -0.5)
    o = paged.paged_attn(q, kc, vc, table, ln, D ** -0.5)
    assert near(o, ref, half_step(BF) * ref.abs() + err)


def test_paged_refusals_gpu(cuda):
    """what only the kernels cannot do (the rest is refused on the CPU too): types, head widths, places, alignment"""
    kc, vc, table, ln = make_cache([5, 9], 16, 2, 32, BF, cuda)
    q = torch.zeros(2, 4, 32, dtype=BF, device=cuda)
    ok = dict(q=q, k_cache=kc, v_cache=vc, table=table, lens=ln, scale=1.0)
    paged.paged_attn(**ok)
    odd = torch.empty(kc.numel() + 1, dtype=BF, device=cuda)[1:].view(kc.shape)
    k48, v48 = paged.page_pools(3, 16, 2, 48, BF, cuda)
    for bad in (dict(q=q.float(), k_cache=kc.float(), v_cache=vc.float()), dict(k_cache=odd), dict(table=table.cpu()),
                dict(lens=ln.cpu()), dict(k_cache=kc.cpu()), dict(out=torch.empty(2, 4, 32, dtype=BF)),
                dict(q=torch.zeros(2, 4, 48, dtype=BF, device=cuda), k_cache=k48, v_cache=v48),
                dict(q=q[:1].expand(70000, 4, 32), table=table[:1].repeat(70000, 1), lens=ln[:1].repeat(70000))):
        with pytest.raises(L.KernelError):
            paged.paged_attn(**{**ok, **bad})
    one = torch.zeros(2, dtype=torch.int32, device=cuda)
    with pytest.raises(L.KernelError):
        paged.rotary_append(q, q[:, :2], q[:, :2], odd, vc, one, one.long(), None)
    with pytest.raises(L.KernelError):
        paged.append(q[:, :2].double(), q[:, :2].double(), kc.double(), vc.double(), one)
    with pytest.raises(L.KernelError):
        paged.page_plan(one, one.cpu(), table, one, one[:1], 16, tokens=2)
    with pytest.raises(L.KernelError):
        paged.page_release(torch.ones(2, dtype=torch.bool), one, table, one, one[:1], 16)


# ----------------------------------------------------------------------------------------------------------------
def test_step_graph_and_streams(cuda):
    """decode steps -- plan, append, attend, lengths carried on -- as two captured graphs and eagerly on another stream:
    the same caches and outputs, replay after replay"""
    B, Hq, Hk, D, page, P, W = 5, 8, 2, 64, 16, 60, 12
    f = rotary.rotary_freqs(D, device=cuda)[0]
    first = [3, 0, 40, 15, 100]

    def fresh(seed):
        g = gen(cuda, 30)
        kc, vc = paged.page_pools(P, page, Hk, D, BF, cuda)
        kc.copy_(torch.randn(kc.shape, device=cuda, generator=g))
        vc.copy_(torch.randn(vc.shape, device=cuda, generator=g))
        s = dict(kc=kc, vc=vc, table=torch.full((B, W), -1, dtype=torch.int32, device=cuda),
                 lens=torch.zeros(B, dtype=torch.int32, device=cuda), stack=torch.arange(P, dtype=torch.int32, device=cuda),
                 nfree=torch.tensor([P], dtype=torch.int32, device=cuda), new=torch.ones(B, dtype=torch.int32, device=cuda),
                 x=torch.zeros(B, (Hq + 2 * Hk) * D, dtype=BF, device=cuda))
        p = paged.page_plan(s["lens"], torch.tensor(first, dtype=torch.int32, device=cuda), s["table"], s["stack"],
                            s["nfree"], page, tokens=sum(first))
        s["lens"].copy_(p.lens)
        s["nfree"].copy_(p.nfree)
        return s

    def step(s):
        q, k, v = s["x"].unflatten(1, (-1, D)).split((Hq, Hk, Hk), 1)
        p = paged.page_plan(s["lens"], s["new"], s["table"], s["stack"], s["nfree"], page, tokens=B)
        q = paged.rotary_append(q, k, v, s["kc"], s["vc"], p.slots, p.pos, f)
        o = paged.paged_attn(q, s["kc"], s["vc"], s["table"], p.lens, D ** -0.5)
        s["lens"].copy_(p.lens)
        s["nfree"].copy_(p.nfree)
        return o

    with torch.no_grad():
        xs = [torch.randn(B, (Hq + 2 * Hk) * D, device=cuda, generator=gen(cuda, 40 + i)).to(BF) for i in range(40)]
        a, b1, b2 = fresh(0), fresh(0), fresh(0)
        graphs = []
        for s in (b1, b2):
            step(fresh(0))                                   # first-use work outside the capture
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                out = step(s)
            graphs.append((gr, s, out))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for x in xs:
            with torch.cuda.stream(side):
                a["x"].copy_(x)
                want = step(a)
            for gr, s, out in graphs:
                s["x"].copy_(x)
                gr.replay()
            torch.cuda.synchronize()
            for gr, s, out in graphs:
                assert torch.equal(out, want) and torch.equal(s["lens"], a["lens"]) and torch.equal(s["nfree"], a["nfree"])
                assert torch.equal(s["kc"], a["kc"]) and torch.equal(s["vc"], a["vc"])
    assert a["lens"].tolist() == [n + 40 for n in first]


def test_rotary_backward_in_a_graph(cuda):
    """forward and backward captured (weight sums included), replayed with new inputs against the eager result"""
    g = gen(cuda, 50)
    T, H, D = 100, 4, 64
    f, pos = rotary.rotary_freqs(D, device=cuda)[0], torch.arange(T, device=cuda)
    q, k, gq, gk = (torch.randn(T, H, D, device=cuda, generator=g).to(BF) for _ in range(4))
    w = [torch.randn(D, device=cuda, generator=g).to(BF) for _ in range(2)]

    def run(q, k, gq, gk):
        leaves = [t.detach().requires_grad_() for t in (q, k, *w)]
        o = rotary.rotary(leaves[0], leaves[1], pos, f, q_weight=leaves[2], k_weight=leaves[3])
        return [t.detach() for t in o] + list(torch.autograd.grad(o, leaves, (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(q, k, gq, gk)
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = run(q, k, gq, gk)
    for i in range(4):
        for t in (q, k, gq, gk):
            t.copy_(torch.randn(T, H, D, device=cuda, generator=g))
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, run(q, k, gq, gk)))


# ----------------------------------------------------------------------------------------------------------------
def test_odd_weights_and_single_rows(cuda):
    """norm weights of two types and in 64 bits; a table of one row with a stride of no meaning"""
    g = gen(cuda, 61)
    q, k = torch.randn(6, 2, 64, device=cuda, generator=g).to(BF), torch.randn(6, 1, 64, device=cuda, generator=g).to(BF)
    freqs, pos = rotary.rotary_freqs(64, device=cuda)[0], torch.arange(6, device=cuda)
    one = torch.ones(6, 2, 64, device=cuda)
    for a, b in ((torch.float64, torch.float64), (F32, BF), (BF, torch.float64)):
        wq, wk = ((torch.rand(64, device=cuda, generator=g) + 0.5).to(t).requires_grad_() for t in (a, b))
        o = rotary.rotary(q, k, pos, freqs, q_weight=wq, k_weight=wk)
        close_rows(o[0].detach(), rotary64(q, wq.detach(), pos, freqs, False, 1.0, 1e-5), BF)
        dq, dk = torch.autograd.grad(o[0].float().sum() + o[1].float().sum(), (wq, wk))
        assert dq.dtype == a and dk.dtype == b
        # weights in 64 bits are read in 32: one more rounding of each term
        _, dw, mag = rotary_grad64(q, wq.detach(), one, pos, freqs, False, 1.0, 1e-5)
        assert bool(((dq.double() - dw).abs() <= half_step(a) * dw.abs() + (64 + 117) * U32 * mag).all())
    kc, vc, table, ln = make_cache([40], 16, 1, 64, BF, cuda, seed=8)
    row = torch.empty(1, 2 ** 33, dtype=torch.int32, device="meta").stride()[0]
    odd = torch.as_strided(table, (1, 3), (row, 1))
    qq = q[:1]
    ref, err = attn64(qq, kc, vc, table, ln, 0.125)
    assert near(paged.paged_attn(qq, kc, vc, odd, ln, 0.125), ref, half_step(BF) * ref.abs() + err)


def test_plain_append_gpu(cuda):
    g = gen(cuda, 60)
    for D, Hk, page, dtype in ((128, 4, 16, BF), (33, 1, 32, HF), (64, 3, 64, F32)):
        k, v = (torch.randn(50, Hk, D, device=cuda, generator=g).to(dtype) for _ in range(2))
        slots = torch.arange(3, 53, dtype=torch.int32, device=cuda)
        slots[7] = -1
        kc, vc = paged.page_pools(5, page, Hk, D, dtype, cuda)
        kc.zero_()
        vc.zero_()
        cpu = [t.cpu() for t in (kc, vc)]
        paged.append(k, v, kc, vc, slots)
        paged.append(k.cpu(), v.cpu(), *cpu, slots.cpu())
        assert torch.equal(kc.cpu(), cpu[0]) and torch.equal(vc.cpu(), cpu[1])


def _model(cuda, **kw):
    from homebrewnlp_mtf_amd.config import ModelParameter
    from homebrewnlp_mtf_amd.models.model import Model
    from homebrewnlp_mtf_amd.parallel import state as pstate
    pstate.set_mesh(pstate.Mesh())
    torch.manual_seed(0)
    cfg = dict(model_mode="gpt", use_video=False, use_language=True, heads=2, features_per_head=64, depth=2,
               sequence_length=96, train_batch_size=3, vocab_size=256, calculation_dtype="bfloat16",
               storage_dtype="bfloat16", block_config=[
                   {"layer": ["norm-shift-scale", "attention-dot_product-context-rotary-qk_norm"], "skip": True},
                   {"layer": ["norm-shift-scale", "feed_forward-in:gelu"], "skip": True}],
               memory_reduction_strategy="none", **kw)
    p = ModelParameter(cfg)
    return Model(p, cuda), p


def test_model_paged_decoding_gpu(cuda):
    """paged caches: the replayed decode graph gives the eager steps' tokens exactly, over requests of several sizes (the
    pool grows, the graph is taken anew); the steps' logits are the full recompute's but for bf16 roundings, as those of
    dense caches of the same model are"""
    from homebrewnlp_mtf_amd.run.infer import Sampler
    m, p = _model(cuda, kv_page_size=16)
    rows = torch.arange(3, device=cuda)
    for seed, start, end in ((1, [3, 7, 1], [16, 30, 9]), (2, [60, 2, 90], [96, 40, 96]), (3, [5, 5, 5], [20, 20, 20])):
        x = torch.randint(0, 256, (3, 96, 1), generator=torch.Generator().manual_seed(seed)).to(cuda)
        got = []
        for graphs in (True, False, True):
            p.decode_hip_graphs = graphs
            s = Sampler(m, p, cuda)
            got.append(s.sample(x, start, 0.0, end))
            assert s.kv_cache
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
        full = m.logits(got[0])[:, :, 0]
        pos = torch.tensor(start, device=cuda)
        for page in (16, 0):
            p.kv_page_size = page
            step = m.prefill(got[0], pos - 1)
            for i in range(10):
                cur = (pos + i - 1).clamp(max=95)
                if i:
                    step = m.decode(got[0][rows, cur].unsqueeze(1), cur)
                ref = full[rows, cur]
                # two layers of about ten bf16 roundings each, every one off by 2^-8 of what it rounds at most
                assert bool(((step[:, 0, 0] - ref).norm(dim=-1) <= 20 * 2.0 ** -8 * ref.norm(dim=-1)).all())
            m.end_decode()
        p.kv_page_size = 16
    x = torch.randint(0, 256, (3, 96, 1), device=cuda)
    bad, _ = _model(cuda)
    bad.params.kv_page_size = 16
    bad.dtype = torch.float32
    with pytest.raises(ValueError):
        bad.prefill(x, torch.tensor([1, 1, 1], device=cuda))


def test_model_rotary_training_gpu(cuda):
    """one training step's gradients on the GPU point where the CPU oracle's do (bf16 activations through two layers)"""
    from homebrewnlp_mtf_amd.models.model import Model
    m, p = _model(cuda, rotary_fraction=0.5)
    c = Model(p, "cpu")
    c.store.master.copy_(m.store.master)
    if c.store.compute.data_ptr() != c.store.master.data_ptr():
        c.store.compute.copy_(c.store.master)
    t = torch.randint(0, 256, (3, 97, 1), generator=torch.Generator().manual_seed(3))
    for mm, dev in ((m, cuda), (c, "cpu")):
        mm.store.grad.zero_()
        mm(token_x=t[:, :-1].contiguous().to(dev), token_y=t[:, 1:].contiguous().to(dev))["loss"].backward()
    names = [n for n in m.store.order if "qk_norm" in n]
    assert len(names) == 4
    for n in names:
        sp = m.store.specs[n]
        a, b = (mm.store.grad[sp.offset:sp.offset + sp.numel].cpu() for mm in (m, c))
        assert torch.nn.functional.cosine_similarity(a, b, dim=0) > 0.97, n
    cos = torch.nn.functional.cosine_similarity(m.store.grad.cpu(), c.store.grad, dim=0)
    assert cos > 0.97, cos


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype,D,rot", [(BF, 128, 64), (HF, 96, 48), (F32, 64, 32), (BF, 128, 0), (BF, 33, 8), (BF, 24, 16),
                                         (BF, 80, 16)])
def test_dims_that_do_not_turn_are_untouched(cuda, dtype, D, rot, inter):
    """infinities and NaN beside the rotated dims, in either direction, and in keys that are appended as they are"""
    g = gen(cuda, 70)
    q, k = (torch.randn(5, h, D, device=cuda, generator=g).to(dtype) for h in (3, 1))
    q[:, :, rot::2] = float("inf")
    k[1, :, -1] = float("nan")
    k[2, :, rot] = float("-inf")
    freqs = rotary.rotary_freqs(rot, device=cuda)[0] if rot else None
    f64 = freqs if rot else torch.zeros(0, dtype=torch.float64, device=cuda)
    pos = torch.arange(5, device=cuda) * 1000
    q.requires_grad_()
    qo, ko = rotary.rotary(q, k, pos, freqs, interleaved=inter, mscale=1.3)
    for x, y in ((q.detach(), qo.detach()), (k, ko)):
        assert torch.equal(torch.nan_to_num(y[..., rot:]), torch.nan_to_num(x[..., rot:]))
        assert torch.equal(torch.isnan(y), torch.isnan(x))
        if rot:
            close_rows(y[..., :rot].contiguous(), rotary64(x, None, pos, f64, inter, 1.3, 1e-5)[..., :rot], dtype)
    dq, = torch.autograd.grad(qo, q, q.detach())
    assert torch.equal(dq[..., rot:], q.detach()[..., rot:]) and bool(torch.isfinite(dq[..., :rot]).all())
    slots = torch.arange(5, dtype=torch.int32, device=cuda) + 2
    kc, vc = paged.page_pools(1, 16, 1, D, dtype, cuda)
    paged.append(k, k, kc, vc, slots)
    assert torch.equal(torch.nan_to_num(kc[0, :, 2:7].transpose(0, 1)), torch.nan_to_num(k))
    assert torch.equal(torch.isnan(kc[0, :, 2:7].transpose(0, 1)), torch.isnan(k))
