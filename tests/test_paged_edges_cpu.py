"""Rotary and paged-cache operators on the CPU: calls at the edge of what they take."""
import math
import pathlib
import random
import re

import pytest
import torch
from torch.autograd import forward_ad

from homebrewnlp_mtf_amd.ops import _lib as L
from homebrewnlp_mtf_amd.ops import paged, rotary
from test_rotary_paged_cpu import ROTARY, _params

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "csrc" / "kernels"


@pytest.mark.parametrize("source,name,packed", [("rotary.hip", "RotDesc", L.ROT_DESC), ("paged.hip", "PlanDesc", L.PLAN_DESC),
                                                ("paged.hip", "PagedDesc", L.PAGED_DESC)])
def test_packed_descriptors_are_as_long_as_the_structs(source, name, packed):
    """the launch reads the whole struct: its padded size, which the source asserts"""
    size = int(re.search(rf"static_assert\(sizeof\({name}\) == (\d+)\)", (KERNELS / source).read_text()).group(1))
    assert packed.size == size and size % 8 == 0


def release_loop(done, lens, table, stack, nfree, page):
    """the rules of page_release over Python lists"""
    lens, stack, P = list(lens), list(stack), len(stack)
    at = min(max(nfree, 0), P)
    for b, d in enumerate(done):
        if not d:
            continue
        for i in range(min(-(-max(lens[b], 0) // page), len(table[b]))):
            if 0 <= table[b][i] < P and at < P:
                stack[at] = table[b][i]
                at += 1
        lens[b] = 0
    return lens, stack, [at]


def release_cases(dev, sizes):
    r = random.Random(16)
    for B, W, P in sizes:
        lens = [r.choice([0, r.randint(1, W * 16), 10 ** 9, -5]) for _ in range(B)]
        table = [[r.choice([r.randrange(P), r.randrange(P), -1, P, 2 ** 31 - 1, -2 ** 31]) for _ in range(W)] for _ in range(B)]
        done = [r.random() < 0.6 for _ in range(B)]
        i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        a = (torch.tensor(done, device=dev), i(lens), i(table), i([-1] * P), i([P // 3]))
        paged.page_release(*a, 16)
        assert [a[1].tolist(), a[3].tolist(), a[4].tolist()] == list(release_loop(done, lens, table, [-1] * P, P // 3, 16))


def test_release_leaves_out_ids_outside_the_pool():
    """an id that is no page would be handed out again, and its tokens lost"""
    release_cases("cpu", [(1, 1, 1), (5, 6, 20), (40, 3, 500)])


def plan_refuses_shared_memory(dev):
    """every buffer that the plan writes, each over the end of every other one: refused, nothing written"""
    B, W, T, P = 3, 4, 6, 12
    room = torch.zeros(256, dtype=torch.int32, device=dev)
    sizes = dict(table=B * W, slots=T, pos=2 * T, start=B + 1, lens=B, nfree_out=1, cached=B, new=B, stack=P, nfree=1)
    apart, at = {}, 0
    for n, m in sizes.items():
        apart[n] = at
        at += m + m % 2

    def call(first):
        room.fill_(0)
        v = {n: room[first[n]:first[n] + m] for n, m in sizes.items()}
        v["new"].fill_(2)
        v["stack"].copy_(torch.arange(P))
        v["nfree"].fill_(P)
        out = paged.PagePlan(v["slots"], v["pos"].view(torch.int64), v["start"], v["lens"], v["nfree_out"])
        before = room.clone()
        try:
            return paged.page_plan(v["cached"], v["new"], v["table"].view(B, W), v["stack"], v["nfree"], 16, out=out)
        finally:
            if first is not apart:
                assert torch.equal(room, before)
    assert call(apart).lens.tolist() == [2] * B
    written = ("table", "slots", "pos", "start", "lens", "nfree_out")
    for w in written:
        for x in sizes:
            if x == w:
                continue
            # the last place of w over the first of x (pos by its 8 bytes)
            to = apart[x] - sizes[w] + (2 if w == "pos" else 1)
            if w == "pos":
                to -= to % 2
            if to >= 0:
                with pytest.raises(L.KernelError):
                    call({**apart, w: to})
            with pytest.raises(L.KernelError):
                call({**apart, w: apart[x]})


def test_plan_refuses_shared_memory():
    plan_refuses_shared_memory("cpu")


def outputs_in_place_and_shared(dev):
    """queries turned, and attended, in their own place; an output over any other part of a call's memory is refused"""
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(5)
    B, Hq, Hk, D, page = 4, 4, 2, 32, 16
    room = torch.randn(4 * B * Hq * D, generator=g).to(dt).to(dev)
    n = B * Hq * D
    q = room[n:2 * n].view(B, Hq, D)
    k, v = (torch.randn(B, Hk, D, generator=g).to(dt).to(dev) for _ in range(2))
    kc, vc = paged.page_pools(4, page, Hk, D, dt, dev)
    kc.normal_()
    vc.normal_()
    i32 = dict(dtype=torch.int32, device=dev)
    slots, pos = torch.arange(B, device=dev).mul(page).int(), torch.arange(B, device=dev) * 100
    table, lens = torch.arange(4, **i32).view(B, 1), torch.tensor([16, 3, 0, 9], **i32)
    f = rotary.rotary_freqs(D, device=dev)[0]
    calls = (lambda q, out=None, k=k, v=v, kc=kc, vc=vc: paged.rotary_append(q, k, v, kc, vc, slots, pos, f, out=out),
             lambda q, out=None, kc=kc, vc=vc: paged.paged_attn(q, kc, vc, table, lens, 0.2, out=out))
    for call in calls:
        want = call(q.clone())
        own = q.clone()
        assert call(own, out=own).data_ptr() == own.data_ptr() and torch.equal(own, want)
        before = room.clone()
        for shift in (8, D, Hq * D, n - 8):
            for at in (n - shift, n + shift):
                with pytest.raises(L.KernelError):
                    call(q, out=room[at:at + n].view(B, Hq, D))
        with pytest.raises(L.KernelError):                 # the queries' place, in another order
            call(q.view(Hq, B, D).transpose(0, 1), out=q)
        assert torch.equal(room, before)
        assert torch.equal(call(q, out=room[:n].view(B, Hq, D)), want)          # beside each other
        room.copy_(before)
        for cache in (kc, vc):
            with pytest.raises(L.KernelError):
                call(q, out=cache.view(-1)[:n].view(B, Hq, D))
    for x in ("k", "v"):
        with pytest.raises(L.KernelError):
            calls[0](q, out=room[2 * n:3 * n].view(B, Hq, D), **{x: room[2 * n + 8:2 * n + 8 + B * Hk * D].view(B, Hk, D)})


def test_outputs_in_place_and_shared():
    outputs_in_place_and_shared("cpu")


def tangents(dev):
    """forward-mode derivatives: what has none says so"""
    g = torch.Generator().manual_seed(6)
    f = rotary.rotary_freqs(32, device=dev)[0]
    kc, vc = paged.page_pools(2, 16, 1, 32, torch.bfloat16, dev)
    kc.zero_()
    vc.zero_()
    x, t, w = (torch.randn(*s, generator=g).to(torch.bfloat16).to(dev) for s in ((3, 1, 32), (3, 1, 32), (32,)))
    i32 = dict(dtype=torch.int32, device=dev)
    slots, pos = torch.arange(3, **i32), torch.arange(3, device=dev)
    table, lens = torch.zeros(3, 1, **i32), torch.ones(3, **i32)
    with torch.no_grad(), forward_ad.dual_level():
        d, dw = forward_ad.make_dual(x, t), forward_ad.make_dual(w, w)
        dk, dv = forward_ad.make_dual(kc, kc.clone()), forward_ad.make_dual(vc, vc.clone())
        calls = [lambda: paged.rotary_append(d, x, x, kc, vc, slots, pos, f), lambda: paged.rotary_append(x, d, x, kc, vc, slots, pos, f),
                 lambda: paged.rotary_append(x, x, d, kc, vc, slots, pos, f),
                 lambda: paged.rotary_append(x, x, x, kc, vc, slots, pos, f, k_weight=dw),
                 lambda: paged.append(d, x, kc, vc, slots), lambda: paged.append(x, d, kc, vc, slots),
                 lambda: paged.append(x, x, dk, vc, slots), lambda: paged.paged_attn(d, kc, vc, table, lens, 1.0),
                 lambda: paged.paged_attn(x, kc, dv, table, lens, 1.0)]
        if x.is_cuda:
            calls += [lambda: rotary.rotary(d, x, pos, f), lambda: rotary.rotary(x, d, pos, f),
                      lambda: rotary.rotary(x, x, pos, f, q_weight=dw)]
        else:
            o = rotary.rotary(d, x, pos, f)[0]
            assert torch.equal(forward_ad.unpack_dual(o).tangent, rotary.rotary(t, x, pos, f)[0])
        for call in calls:
            with pytest.raises(L.KernelError):
                call()
        assert not bool(kc.any()) and not bool(vc.any())
        rotary.rotary(x, x, pos, f, q_weight=w)                       # none of them has a tangent
        paged.rotary_append(x, x, x, kc, vc, slots, pos, f)
        paged.paged_attn(x, kc, vc, table, lens, 1.0)


def test_tangents():
    tangents("cpu")


@pytest.mark.parametrize("theta", [500.0, 10000.0, 500000.0])
@pytest.mark.parametrize("rot,length,fast,slow", [(64, 2048, 32, 1), (128, 4096, 32, 1), (8, 32768, 32, 1), (16, 10 ** 6, 32, 1),
                                                  (64, 4, 32, 1), (64, 2, 2, 0.5), (32, 6, 8, 2), (8, 100, 4, 3.9)])
def test_ramp_keeps_and_divides_as_it_says(rot, length, fast, slow, theta):
    """every pair by its own turns over the trained length: as it was above `fast`, divided below `slow`, in between on
    a line over the pair's index that spans the two (their whole pairs around it)"""
    s = 8.0
    f, _ = rotary.rotary_freqs(rot, theta)
    r, m = rotary.rotary_freqs(rot, theta, {"type": "ramp", "factor": s, "length": length, "fast": fast, "slow": slow})
    assert math.isclose(m, 0.1 * math.log(s) + 1)
    turns = f * length / (2 * math.pi)
    part = (r / f - 1) / (1 / s - 1)                     # 0: kept, 1: divided
    assert bool((part >= -1e-12).all()) and bool((part <= 1 + 1e-12).all())
    assert bool((part[turns < slow] > 1 - 1e-9).all()) and bool((part[turns > fast] < 1e-9).all())
    step = part.diff()
    assert bool((step > -1e-9).all())
    # the line: equal steps between the pairs that are on it
    on = (part > 1e-9) & (part < 1 - 1e-9)
    both = on[1:] & on[:-1]
    if int(both.sum()) > 1:
        assert float(step[both].max() - step[both].min()) < 1e-9
    # the slowest pair is divided in full only where it turns less than the pair after it, at most `slow` times
    if float(turns[-1]) > slow * theta ** (2 / rot):
        assert float(part[-1]) < 1 - 1e-9


def test_eps_that_vanishes_in_32_bits():
    """added in 32 bits, it is 0: rows of zeros would be 0 times infinity. 64 bits hold it"""
    f = rotary.rotary_freqs(8)[0]
    pos = torch.arange(2)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x, w = torch.zeros(2, 1, 8, dtype=dtype), torch.ones(8, dtype=dtype)
        kc, vc = paged.page_pools(1, 16, 1, 8, dtype, "cpu")
        for eps in (1e-50, 1e-39, math.inf, math.nan, 1e39, -1.0):
            with pytest.raises(L.KernelError):
                rotary.rotary(x, x, pos, f, q_weight=w, eps=eps)
            with pytest.raises(L.KernelError):
                paged.rotary_append(x, x, x, kc, vc, pos.int(), pos, f, k_weight=w, eps=eps)
        for eps in (2.0 ** -126, 1e-30, 1e-5, 1e38):
            assert not bool(rotary.rotary(x, x, pos, f, q_weight=w, eps=eps)[0].any())
    x = torch.zeros(2, 1, 8, dtype=torch.float64)
    assert not bool(rotary.rotary(x, x, pos, f, q_weight=torch.ones(8), eps=1e-50)[0].any())


def scores_of_minus_infinity(dev):
    """a request all of whose scores are -inf has no weights: 0, as one without tokens; some of them hide their keys"""
    g = torch.Generator().manual_seed(8)
    kc, vc = paged.page_pools(4, 16, 1, 32, torch.bfloat16, dev)
    kc.copy_(torch.randn(kc.shape, generator=g))
    vc.copy_(torch.randn(vc.shape, generator=g))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    lens = torch.tensor([20, 20], dtype=torch.int32, device=dev)
    q = torch.ones(2, 3, 32, dtype=torch.bfloat16, device=dev)
    kc[:2, :, :, 5] = -math.inf
    kc[2, :, :, 5] = -math.inf                 # the second request's keys 16 to 19 are left
    o = paged.paged_attn(q, kc, vc, table, lens, 0.1)
    w = torch.softmax(0.1 * kc[3, 0, :4].double().sum(-1), 0)
    ref = (w[:, None] * vc[3, 0, 0, :, :4].double().t()).sum(0)
    assert not bool(o[0].any())
    # a score of 32 products within (32 + 4) roundings of its size, twice; half a step of bf16
    err = 2 * 36 * 2.0 ** -24 * float(0.1 * kc[3, 0, :4].double().abs().sum(-1).max()) + 2.0 ** -20
    assert bool(((o[1].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + err * vc[3].double().abs().max()).all())


def test_scores_of_minus_infinity():
    scores_of_minus_infinity("cpu")


# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("extras", ["-rotary", ""])
def test_decoding_outside_the_context(extras):
    """a position before or behind the context: paged caches give what dense ones do, and hold what they held"""
    from homebrewnlp_mtf_amd.models.model import Model
    from homebrewnlp_mtf_amd.parallel import state as pstate
    pstate.set_mesh(pstate.Mesh())
    torch.manual_seed(0)
    p = _params(sequence_length=40, **ROTARY, block_config=[
        {"layer": ["norm-shift-scale", "attention-dot_product-context" + extras], "skip": True}])
    m = Model(p, "cpu")
    x = torch.randint(0, 64, (3, 40, 1), generator=torch.Generator().manual_seed(1))
    for pos in (40, 47, 48, 10 ** 6, -1, -17, -10 ** 6):
        out = []
        for page in (0, 16):
            p.kv_page_size = page
            m.prefill(x, torch.tensor([39, 39, 5]))          # rows 0 and 1 hold the whole context
            out.append([m.decode(x[:, :1], torch.tensor([pos, pos, at])) for at in (6, 7)])
            m.end_decode()
        for a, b in zip(*out):
            assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)       # fp32, sums in another order


@pytest.mark.parametrize("extras", ["-rotary-qk_norm", "-rotary", "-qk_norm"])
@pytest.mark.parametrize("strategy", ["none", "checkpoint", "revnet", "momentum"])
def test_training_gradients(strategy, extras):
    """every strategy's gradients -- recomputed blocks, reconstructed streams -- against differences of the loss, along
    random directions of each weight that lies before or in the turned attention"""
    from homebrewnlp_mtf_amd.parallel import state as pstate
    from homebrewnlp_mtf_amd.run.trainer import Trainer
    pstate.set_mesh(pstate.Mesh())
    torch.manual_seed(0)
    tr = Trainer(_params(memory_reduction_strategy=strategy, **ROTARY, block_config=[
        {"layer": ["norm-shift-scale", "attention-dot_product-context" + extras], "skip": True},
        {"layer": ["norm-shift-scale", "feed_forward-in:gelu"], "skip": True}]), "cpu")
    st = tr.model.store
    t = torch.randint(0, 64, (3, 17, 1), generator=torch.Generator().manual_seed(2))
    batch = {"token_x": t[:, :-1].contiguous(), "token_y": t[:, 1:].contiguous()}
    st.zero_grad()
    tr.model(**batch)["loss"].backward()
    grads = st.grad.clone()
    names = [n for n in st.order if "qk_norm" in n or "attention" in n]
    assert len(names) >= 4 and ("qk_norm" not in extras or sum("qk_norm" in n for n in names) == 4)
    g = torch.Generator().manual_seed(3)
    bufs = {b.data_ptr(): b for b in (st.master, st.compute)}.values()
    for name in names:
        sp = st.specs[name]
        grad = grads[sp.offset:sp.offset + sp.numel]
        d = torch.sign(grad) + 0.5 * torch.randn(sp.numel, generator=g)     # a direction in which the loss moves
        d *= 3e-2 / d.norm()
        vals = []
        for sign in (1, -2, 1):
            for b in bufs:
                b[sp.offset:sp.offset + sp.numel] += sign * d
            with torch.no_grad():
                vals.append(float(tr.model(**batch)["loss"]))
        got, want = float(grad @ d), (vals[0] - vals[1]) / 2
        # the losses (~4) are fp32 sums, each off by some half steps of 2.4e-7; the difference's third order, of a step
        # of 3e-2, is 1e-3 of it
        assert got > 0 and abs(got - want) < 4e-6 + 0.02 * abs(want), (name, got, want)
