"""Rotary and paged-cache operators on the CPU: the oracles against 64-bit definitions, gradients against the formula
and against differences, frequencies, and every refusal."""
import math
import random

import pytest
import torch

from homebrewnlp_mtf_amd.ops import _lib as L
from homebrewnlp_mtf_amd.ops import paged, rotary
from paged_cases import U32, attn64, half_step, make_cache, past_31_bits, plan_loop, rotary64, rotary_grad64


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_rotary_oracle(dtype, inter):
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(2, 5, 3, 12, generator=g).to(dtype), torch.randn(2, 5, 1, 12, generator=g).to(dtype)
    pos = torch.randint(-5, 130000, (2, 5), generator=g)
    freqs, _ = rotary.rotary_freqs(8)
    w = torch.rand(12, generator=g).to(dtype) + 0.5
    qo, ko = rotary.rotary(q, k, pos, freqs, interleaved=inter, mscale=1.3, q_weight=w)
    for x, y, ww in ((q, qo, w), (k, ko, None)):
        ref = rotary64(x, ww, pos, freqs, inter, 1.3, 1e-5).reshape(x.shape)
        size = ref.abs().amax(-1, keepdim=True)
        tol = half_step(dtype) * ref.abs() + (32 + 12) * min(U32, half_step(dtype)) * size
        assert y.dtype == dtype and bool(((y.double() - ref).abs() <= tol + 1e-15).all())


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, False)])
def test_rotary_gradients(norms, inter):
    g = torch.Generator().manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, gq, gk = rnd(3, 2, 10), rnd(3, 1, 10), rnd(3, 2, 10), rnd(3, 1, 10)
    ws = [rnd(10) if n else None for n in norms]
    pos = torch.tensor([0, 7, 100000])
    freqs, _ = rotary.rotary_freqs(6, scaling={"type": "linear", "factor": 2})
    leaves = [t.requires_grad_() for t in (q, k, *ws) if t is not None]

    def f(q, k, *w):
        w = list(w)
        wq, wk = (w.pop(0) if n else None for n in norms)
        return rotary.rotary(q, k, pos, freqs, interleaved=inter, mscale=0.7, q_weight=wq, k_weight=wk)
    assert torch.autograd.gradcheck(f, tuple(leaves), eps=1e-6, atol=1e-7, rtol=1e-6)
    grads = list(torch.autograd.grad(f(*leaves), leaves, (gq, gk)))
    for x, w, gg, d in ((q, ws[0], gq, grads[0]), (k, ws[1], gk, grads[1])):
        dx, dw, _ = rotary_grad64(x.detach(), None if w is None else w.detach(), gg, pos, freqs, inter, 0.7, 1e-5)
        assert torch.allclose(d, dx.reshape(d.shape), rtol=1e-12, atol=1e-13)
        if dw is not None:
            got = grads[2 if w is ws[0] else len(grads) - 1]
            assert torch.allclose(got, dw, rtol=1e-12, atol=1e-12)


def test_rotary_main_grad_and_shared_weight():
    """model parameters accumulate into their flat fp32 gradient; one parameter for q and k gets both parts"""
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(4, 2, 8, generator=g), torch.randn(4, 2, 8, generator=g)
    freqs, _ = rotary.rotary_freqs(8)
    pos = torch.arange(4)
    a, b = torch.rand(8, generator=g).requires_grad_(), torch.rand(8, generator=g).requires_grad_()
    both = torch.rand(8, generator=g).requires_grad_()
    for wq, wk in ((a, b), (both, both)):
        ref = torch.autograd.grad(sum(o.pow(2).sum() for o in rotary.rotary(q, k, pos, freqs, q_weight=wq, k_weight=wk)),
                                  [wq] if wq is wk else [wq, wk])
        for w in (wq, wk):
            w.main_grad = torch.ones(8)
        sum(o.pow(2).sum() for o in rotary.rotary(q, k, pos, freqs, q_weight=wq, k_weight=wk)).backward()
        for w, r in zip([wq] if wq is wk else [wq, wk], ref):
            assert w.grad is None and torch.allclose(w.main_grad - 1, r, rtol=1e-5, atol=1e-5)
            del w.main_grad


def test_rotary_freqs():
    f, m = rotary.rotary_freqs(8, 10000.0)
    assert m == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    lin, _ = rotary.rotary_freqs(8, scaling={"type": "linear", "factor": 4})
    assert torch.allclose(lin, f / 4)
    base, _ = rotary.rotary_freqs(8, scaling={"type": "base", "factor": 4})
    assert base[0] == 1.0 and math.isclose(float(base[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    f, _ = rotary.rotary_freqs(64)
    ramp, m = rotary.rotary_freqs(64, scaling={"type": "ramp", "factor": 8, "length": 2048})
    turns = f * 2048 / (2 * math.pi)
    assert torch.equal(ramp[turns > 40], f[turns > 40]) and torch.allclose(ramp[turns < 0.7], f[turns < 0.7] / 8)
    assert bool((ramp <= f).all()) and bool((ramp >= f / 8 * (1 - 1e-12)).all())
    assert math.isclose(m, 0.1 * math.log(8) + 1)
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, theta=0.0),
                dict(rot_dim=8, scaling={"type": "other", "factor": 2}),
                dict(rot_dim=8, scaling={"type": "linear", "factor": 0.5}),
                dict(rot_dim=8, scaling={"type": "linear", "factor": 2, "len": 1}),
                dict(rot_dim=2, scaling={"type": "base", "factor": 2}),
                dict(rot_dim=8, scaling={"type": "ramp", "factor": 2, "fast": 1, "slow": 2})):
        with pytest.raises(ValueError):
            rotary.rotary_freqs(**bad)


def test_rotary_refusals():
    q, k = torch.zeros(3, 2, 8), torch.zeros(3, 1, 8)
    pos, (f, _) = torch.arange(3), rotary.rotary_freqs(8)
    ok = dict(q=q, k=k, pos=pos, freqs=f)
    rotary.rotary(**ok)
    rotary.rotary(**{**ok, "freqs": None})
    for bad in (dict(q=q[0]), dict(k=k[:2]), dict(k=torch.zeros(3, 1, 6)), dict(k=k.double()), dict(pos=pos.int()),
                dict(pos=torch.arange(4)), dict(freqs=f.float()), dict(freqs=torch.ones(5, dtype=torch.float64)),
                dict(freqs=f.view(2, 2)), dict(q_weight=torch.ones(7)), dict(k_weight=torch.ones(8, dtype=torch.int32)),
                dict(eps=0.0), dict(q=torch.zeros(3, 0, 8)),
                dict(q=torch.zeros(3, 1, 514), k=torch.zeros(3, 1, 514))):
        with pytest.raises(L.KernelError):
            rotary.rotary(**{**ok, **bad})
    e = rotary.rotary(q[:0], k[:0], pos[:0], f)
    assert e[0].shape == (0, 2, 8)
    qq = q.clone().requires_grad_()
    with pytest.raises(L.KernelError):
        torch.autograd.grad(rotary.rotary(qq, k, pos, f)[0].sum(), qq, create_graph=True)
    # no tokens: zero gradients
    z = q[:0].clone().requires_grad_()
    w = torch.ones(8, requires_grad=True)
    o = rotary.rotary(z, k[:0], pos[:0], f, q_weight=w)
    assert torch.equal(torch.autograd.grad(o[0].sum(), w)[0], torch.zeros(8))


# ----------------------------------------------------------------------------------------------------------------
def run_plan(dev, cached, new, table, stack, nfree, page, T):
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t = i(table)
    p = paged.page_plan(i(cached), i(new), t, i(stack), i([nfree]), page, tokens=T)
    return (p.slots.tolist(), p.pos.tolist(), p.start.tolist(), p.lens.tolist(), int(p.nfree), t.tolist())


def random_plan(r):
    B, page, W = r.randint(1, 40), r.choice([1, 7, 16, 32]), r.randint(1, 9)
    cached = [r.choice([0, r.randint(0, W * page), -3]) for _ in range(B)]
    new = [r.choice([0, 1, 1, r.randint(0, 3 * page), -2]) for _ in range(B)]
    P = r.randint(1, 60)
    stack = [r.randint(0, P - 1) for _ in range(P)]
    table = [[r.choice([r.randint(0, P - 1), -1, P, 2 ** 31 - 1]) for _ in range(W)] for _ in range(B)]
    T = max(0, sum(max(n, 0) for n in new) + r.randint(-8, 8))
    return cached, new, table, stack, r.randint(-1, P + 1), page, T


def test_plan_oracle():
    r = random.Random(4)
    for _ in range(60):
        c = random_plan(r)
        assert run_plan("cpu", *c) == tuple(plan_loop(*c)), c


def test_plan_refuses_lengths_past_31_bits():
    past_31_bits("cpu")


def test_plan_and_release_refusals():
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    ok = dict(cached=i(0, 1), new=i(1, 1), table=torch.zeros(2, 3, dtype=torch.int32), stack=i(0, 1, 2), nfree=i(3),
              page=16, tokens=4)
    paged.page_plan(**ok)
    b = paged.plan_buffers(2, 4, "cpu")
    paged.page_plan(**{**ok, "out": b})
    shared = i(0, 1)
    for bad in (dict(cached=i(0)), dict(new=torch.ones(2)), dict(table=torch.zeros(2, 3)), dict(tokens=None),
                dict(table=torch.zeros(3, 2, dtype=torch.int32).t()), dict(table=torch.zeros(3, 3, dtype=torch.int32)),
                dict(table=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)), dict(nfree=i(1, 2)), dict(page=0),
                dict(stack=i()), dict(page=2 ** 30), dict(out=b, tokens=5), dict(out=b._replace(pos=b.pos.int())),
                dict(out=b._replace(lens=shared), cached=shared), dict(cached=torch.arange(4, dtype=torch.int32)[::2])):
        with pytest.raises(L.KernelError):
            paged.page_plan(**{**ok, **bad})
    nf = i(3)
    with pytest.raises(L.KernelError):
        paged.page_plan(**{**ok, "out": b._replace(nfree=nf), "nfree": nf})
    done = torch.tensor([True, False])
    rel = dict(done=done, lens=i(20, 1), table=torch.tensor([[2, 1, 0], [0, 0, 0]], dtype=torch.int32),
               stack=i(9, 9, 9), nfree=i(1), page=16)
    paged.page_release(**rel)
    assert rel["stack"].tolist() == [9, 2, 1] and rel["nfree"].tolist() == [3] and rel["lens"].tolist() == [0, 1]
    for bad in (dict(done=done.int()), dict(done=done[:1]), dict(lens=i(1, 1).long()), dict(page=0), dict(nfree=i())):
        with pytest.raises(L.KernelError):
            paged.page_release(**{**rel, **bad})


def test_plan_release_cycle():
    """pages taken step by step and given back: the stack ends as full as it began, no page is held twice"""
    r = random.Random(5)
    B, W, P, page = 6, 5, 17, 16
    lens, table = torch.zeros(B, dtype=torch.int32), torch.full((B, W), -1, dtype=torch.int32)
    stack, nfree = torch.arange(P, dtype=torch.int32), torch.tensor([P], dtype=torch.int32)
    for _ in range(60):
        new = torch.tensor([r.choice([0, 1, 9, 30]) for _ in range(B)], dtype=torch.int32)
        p = paged.page_plan(lens, new, table, stack, nfree, page, tokens=200)
        lens, nfree = p.lens, p.nfree
        held = [int(table[b, i]) for b in range(B) for i in range(-(-int(lens[b]) // page))]
        free = stack[:int(nfree)].tolist()
        assert sorted(held + free) == list(range(P))
        live = p.slots[p.slots >= 0].tolist()
        assert len(set(live)) == len(live)
        paged.page_release(torch.tensor([r.random() < 0.2 for _ in range(B)]), lens, table, stack, nfree, page)
    paged.page_release(torch.ones(B, dtype=torch.bool), lens, table, stack, nfree, page)
    assert sorted(stack[:int(nfree)].tolist()) == list(range(P))


# ----------------------------------------------------------------------------------------------------------------
def test_append_oracle_and_refusals():
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(5, h, 32, generator=g) for h in (4, 2, 2))
    kc, vc = paged.page_pools(3, 16, 2, 32, torch.float32, "cpu")
    kc.fill_(7)
    vc.fill_(7)
    slots, pos = torch.tensor([47, -1, 0, 48, 17], dtype=torch.int32), torch.tensor([3, 9, 0, 1, 70000])
    f, _ = rotary.rotary_freqs(32)
    w = torch.rand(32, generator=g)
    args = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, slots=slots, pos=pos, freqs=f)
    qo = paged.rotary_append(**args, k_weight=w)
    assert torch.allclose(qo.double(), rotary64(q, None, pos, f, False, 1.0, 1e-5), atol=1e-5)
    kr = rotary64(k, w, pos, f, False, 1.0, 1e-5)
    touched = torch.zeros(48, dtype=torch.bool)
    for t in (0, 2, 4):
        p, o = divmod(int(slots[t]), 16)
        touched[int(slots[t])] = True
        assert torch.allclose(kc[p, :, o].double(), kr[t], atol=1e-5)
        assert torch.equal(vc[p, :, o // 8, :, o % 8], v[t])
    assert bool((kc.permute(0, 2, 1, 3).reshape(48, 2, 32)[~touched] == 7).all())
    assert bool((vc.permute(0, 2, 4, 1, 3).reshape(48, 2, 32)[~touched] == 7).all())
    plain = paged.rotary_append(**{**args, "freqs": None})
    assert torch.equal(plain, q) and torch.equal(kc[0, :, 0], k[2])
    for bad in (dict(v=v[:4]), dict(v=v.double()), dict(slots=slots.long()), dict(slots=slots[:4]), dict(k=k[:, :1]),
                dict(k_cache=kc.double()), dict(v_cache=vc[:2]), dict(k_cache=kc[:, :1]), dict(pos=pos[:4]),
                dict(k_cache=kc.transpose(0, 1)), dict(q=q.clone().requires_grad_()), dict(out=q[:3]),
                dict(k_weight=w.clone().requires_grad_()), dict(v_cache=vc.clone().requires_grad_()),
                dict(q=q.unsqueeze(0), k=k.unsqueeze(0), v=v.unsqueeze(0))):
        with pytest.raises(L.KernelError):
            paged.rotary_append(**{**args, **bad})
    with pytest.raises(L.KernelError):
        paged.page_pools(3, 24, 2, 32, torch.float32, "cpu")
    with pytest.raises(L.KernelError):
        paged.page_pools(2 ** 28, 16, 2, 32, torch.float32, "meta")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attn_oracle(dtype):
    lens = [0, 1, 16, 17, 50]
    kc, vc, table, ln = make_cache(lens, 16, 2, 32, dtype, "cpu")
    q = torch.randn(5, 6, 32, generator=torch.Generator().manual_seed(7)).to(dtype)
    o = paged.paged_attn(q, kc, vc, table, ln, 0.3)
    ref, err = attn64(q, kc, vc, table, ln, 0.3)
    assert bool(((o.double() - ref).abs() <= half_step(dtype) * ref.abs() + err).all())
    assert bool((o[0] == 0).all())
    # ids outside the pool hide their tokens; a bound cuts
    table[4, 1] = kc.shape[0]
    table[2, 0] = -1
    o = paged.paged_attn(q, kc, vc, table, ln, 0.3, max_len=40)
    ref, err = attn64(q, kc, vc, table, ln, 0.3, cap=40)
    assert bool(((o.double() - ref).abs() <= half_step(dtype) * ref.abs() + err).all()) and bool((o[2] == 0).all())


def test_attn_refusals():
    kc, vc, table, ln = make_cache([5, 9], 16, 2, 32, torch.bfloat16, "cpu")
    q = torch.zeros(2, 4, 32, dtype=torch.bfloat16)
    ok = dict(q=q, k_cache=kc, v_cache=vc, table=table, lens=ln, scale=1.0)
    paged.paged_attn(**ok)
    for bad in (dict(q=q[0]), dict(q=q.float()), dict(q=q[:, :3]), dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
                dict(table=table.long()), dict(table=table[:1]), dict(lens=ln.long()), dict(lens=ln[:1]),
                dict(max_len=-1), dict(out=torch.zeros(2, 4, 32)), dict(v_cache=vc.flatten(2)),
                dict(k_cache=kc.transpose(1, 2)), dict(q=q.clone().requires_grad_())):
        with pytest.raises(L.KernelError):
            paged.paged_attn(**{**ok, **bad})
    wide = torch.zeros(1, 2 ** 22 + 1, dtype=torch.int32)                     # pages of 256: more than 2^30 tokens
    big = dict(q=q[:1], k_cache=torch.zeros(1, 2, 256, 32, dtype=torch.bfloat16), table=wide, lens=ln[:1], scale=1.0,
               v_cache=torch.zeros(1, 2, 32, 32, 8, dtype=torch.bfloat16))
    with pytest.raises(L.KernelError):
        paged.paged_attn(**big)
    paged.paged_attn(**big, max_len=300)
    assert paged.paged_attn(**{**ok, "q": q[:0], "table": table[:0], "lens": ln[:0]}).shape == (0, 4, 32)


def test_step_by_step_matches_dense():
    """prompts, then decode steps, through plan -> append -> attend against attention over plain dense keys"""
    g = torch.Generator().manual_seed(8)
    B, Hq, Hk, D, page = 3, 4, 2, 32, 16
    f, _ = rotary.rotary_freqs(D)
    kc, vc = paged.page_pools(12, page, Hk, D, torch.float32, "cpu")
    lens, table = torch.zeros(B, dtype=torch.int32), torch.full((B, 4), -1, dtype=torch.int32)
    stack, nfree = torch.randperm(12, generator=g).int(), torch.tensor([12], dtype=torch.int32)
    ks, vs = [[] for _ in range(B)], [[] for _ in range(B)]
    for step in range(20):
        new = torch.tensor([13, 0, 30] if step == 0 else [1, 1, 1], dtype=torch.int32)
        T = int(new.sum()) + 2
        q, k, v = (torch.randn(T, h, D, generator=g) for h in (Hq, Hk, Hk))
        p = paged.page_plan(lens, new, table, stack, nfree, page, tokens=T)
        qo = paged.rotary_append(q, k, v, kc, vc, p.slots, p.pos, f)
        lens, nfree = p.lens, p.nfree
        kr = rotary64(k, None, p.pos, f, False, 1.0, 1e-5)
        for b in range(B):
            for t in range(int(p.start[b]), int(p.start[b + 1])):
                ks[b].append(kr[t])
                vs[b].append(v[t].double())
        if step == 0:
            continue
        o = paged.paged_attn(qo[:B].contiguous(), kc, vc, table, lens, D ** -0.5)
        for b in range(B):
            kk, vv = torch.stack(ks[b]).repeat_interleave(2, 1), torch.stack(vs[b]).repeat_interleave(2, 1)
            s = torch.softmax(torch.einsum("hd,jhd->hj", qo[b].double(), kk) * D ** -0.5, -1)
            assert torch.allclose(o[b].double(), torch.einsum("hj,jhd->hd", s, vv), atol=1e-5)


def test_plain_append():
    g = torch.Generator().manual_seed(9)
    k, v = torch.randn(4, 2, 32, generator=g), torch.randn(4, 2, 32, generator=g)
    slots = torch.tensor([5, -1, 31, 32], dtype=torch.int32)
    pools = [paged.page_pools(2, 16, 2, 32, torch.float32, "cpu") for _ in range(2)]
    for kc, vc in pools:
        kc.zero_()
        vc.zero_()
    paged.append(k, v, *pools[0], slots)
    paged.rotary_append(k, k, v, *pools[1], slots, torch.zeros(4, dtype=torch.int64), None)
    assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1])
    for bad in (dict(k=k[:3]), dict(v=v.double()), dict(slots=slots.long()), dict(slots=slots[:3]), dict(k=k[0]),
                dict(k_cache=pools[0][0].double()), dict(k=k.clone().requires_grad_())):
        with pytest.raises(L.KernelError):
            paged.append(**{**dict(k=k, v=v, k_cache=pools[0][0], v_cache=pools[0][1], slots=slots), **bad})


# ----------------------------------------------------------------------------------------------------------------
def _params(**kw):
    from homebrewnlp_mtf_amd.config import ModelParameter
    cfg = dict(model_mode="gpt", use_video=False, use_language=True, heads=2, features_per_head=8, depth=2,
               sequence_length=16, train_batch_size=3, vocab_size=64, intermediate_feed_forward_multiplier=2,
               memory_reduction_strategy="none", calculation_dtype="float32", learning_rate=0.01,
               optimizer="adam-learning_rate",
               block_config=[{"layer": ["norm-shift-scale", "attention-dot_product-context-rotary-qk_norm"], "skip": True},
                             {"layer": ["norm-shift-scale", "feed_forward-in:gelu"], "skip": True}])
    cfg.update(kw)
    return ModelParameter(cfg)


ROTARY = dict(rotary_fraction=0.5, rotary_interleaved=True, rotary_scaling={"type": "ramp", "factor": 4.0, "length": 8})


@pytest.mark.parametrize("strategy", ["none", "revnet"])
@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("extras", ["-rotary-qk_norm", "-rotary", "-qk_norm", ""])
def test_model_decodes_like_full_recompute(extras, page, strategy, monkeypatch):
    """rotary / qk_norm attention under dense and paged caches: the tokens of the full recompute, rows of different
    lengths, one of them done from the start, twice with one model (buffers of another request)"""
    from homebrewnlp_mtf_amd.models.model import Model
    from homebrewnlp_mtf_amd.parallel import state as pstate
    from homebrewnlp_mtf_amd.run.infer import Sampler
    pstate.set_mesh(pstate.Mesh())
    torch.manual_seed(0)
    p = _params(kv_page_size=page, memory_reduction_strategy=strategy, sequence_length=40, **ROTARY, block_config=[
        {"layer": ["norm-shift-scale", "attention-dot_product-context" + extras], "skip": True},
        {"layer": ["norm-shift-scale", "feed_forward-in:gelu"], "skip": True}])
    m = Model(p, "cpu")
    calls = []
    real = paged.paged_attn
    monkeypatch.setattr(paged, "paged_attn", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    for seed, start, end in ((4, [3, 7, 1], [16, 40, 9]), (5, [30, 2, 40], [40, 8, 12])):
        x = torch.randint(0, 64, (3, 40, 1), generator=torch.Generator().manual_seed(seed))
        for temp in (0.0, [0.0, 1.0, 3.0]):
            cached, full = Sampler(m, p, "cpu"), Sampler(m, p, "cpu")
            full.kv_cache = False
            a = cached.sample(x, start, temp, end)
            assert cached.kv_cache and bool(calls) == bool(page)
            assert torch.equal(a, full.sample(x, start, temp, end))
    assert m.builder.kv is None


def test_model_rotary_positions_matter_and_train():
    """the rotation changes the logits, and one step's gradients match differences (fp64 model)"""
    from homebrewnlp_mtf_amd.models.model import Model
    from homebrewnlp_mtf_amd.parallel import state as pstate
    pstate.set_mesh(pstate.Mesh())
    torch.manual_seed(0)
    p = _params(**ROTARY)
    m = Model(p, "cpu", dtype=torch.float64)
    names = [n for n in m.store.order if "qk_norm" in n]
    assert len(names) == 4 and all(m.store.specs[n].full_shape == [8] for n in names)
    g = torch.Generator().manual_seed(1)
    t = torch.randint(0, 64, (3, 17, 1), generator=g)
    batch = {"token_x": t[:, :-1].contiguous(), "token_y": t[:, 1:].contiguous()}
    base = m.logits(batch["token_x"])
    m.params.rotary_theta = m.builder.params.rotary_theta = 50.0
    assert not torch.allclose(base, m.logits(batch["token_x"]))
    with pytest.raises(ValueError):
        Model(_params(block_config=[{"layer": ["attention-dot_product-embedded-absolute-rotary"]}]), "cpu")
    for bad in (dict(kv_page_size=24), dict(rotary_fraction=0.0), dict(rotary_fraction=1.5)):
        with pytest.raises(ValueError):
            _params(**bad)


def test_trainer_steps_with_rotary_attention():
    """gradients of the qk_norm weights through a whole training step against differences of the loss"""
    from homebrewnlp_mtf_amd.parallel import state as pstate
    from homebrewnlp_mtf_amd.run.trainer import Trainer
    pstate.set_mesh(pstate.Mesh())
    torch.manual_seed(0)
    tr = Trainer(_params(**ROTARY), "cpu")
    st = tr.store if hasattr(tr, "store") else tr.model.store
    g = torch.Generator().manual_seed(2)
    t = torch.randint(0, 64, (3, 17, 1), generator=g)
    batch = {"token_x": t[:, :-1].contiguous(), "token_y": t[:, 1:].contiguous()}

    def loss():
        return tr.model(**batch)["loss"]
    name = next(n for n in st.order if "qk_norm" in n)
    out = loss()
    st.zero_grad() if hasattr(st, "zero_grad") else st.grad.zero_()
    out.backward()
    sp = st.specs[name]
    grad = st.grad[sp.offset:sp.offset + sp.numel].clone()
    assert float(grad.abs().max()) > 0
    for i in (0, 5):
        vals = []
        for d in (1e-2, -1e-2):
            for buf in {st.master.data_ptr(): st.master, st.compute.data_ptr(): st.compute}.values():
                buf[sp.offset + i] += d
            with torch.no_grad():
                vals.append(float(loss()))
            for buf in {st.master.data_ptr(): st.master, st.compute.data_ptr(): st.compute}.values():
                buf[sp.offset + i] -= d
        # central difference: third derivatives times 1e-4 / 6, and two fp32 losses (~4, half a step 2.4e-7) over 2e-2
        assert abs((vals[0] - vals[1]) / 2e-2 - float(grad[i])) < 1e-4 + 0.02 * abs(float(grad[i]))


def test_splits_cover_every_length():
    rng = random.Random(3)
    for B in (1, 3, 8, 16, 17, 200, 60000):
        for rows in (1, 4, 20, 64, 1000):
            for cap in (0, 1, 16, 255, 256, 257, 2048, 4097, 131072, 2 ** 21 + 1, 2 ** 30):
                n, split, most = paged._splits(B, rows, cap)
                assert 1 <= n <= 1024 and split % 128 == 0
                if not most:
                    assert (n - 1) * split < max(cap, 1) <= n * split
                    continue
                # the kernel's own size for these lengths: no request needs more than n
                for lens in ([cap] * B, [cap] + [0] * (B - 1), [rng.randint(0, cap) for _ in range(B)]):
                    units = sum(-(-x // 128) for x in lens)
                    s = max(split, min(-(-units // most), 2 ** 23) * 128)
                    assert s < 2 ** 31 and all(-(-x // s) <= n for x in lens)
