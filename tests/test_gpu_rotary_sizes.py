"""Rotary kernels at the sizes of a training step, every output and gradient against the 64-bit definition."""
import pytest
import torch

from homebrewnlp_mtf_amd.ops import paged, rotary
from paged_cases import U32, half_step, rotary64, rotary_grad64
from test_gpu_rotary_paged import ROT

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rows_within(y, ref, dtype, extra=0.0):
    """half a step of the output type plus (32 + D) roundings of fp32 at the size of the row (a sum over D, a reciprocal
    root, two products, a rotation); NaN is never within"""
    ref = ref.reshape(y.shape)
    assert bool(torch.isfinite(ref).all())
    tol = half_step(dtype) * ref.abs() + (32 + y.shape[-1]) * U32 * ref.abs().amax(-1, keepdim=True) + extra
    if dtype == HF:
        tol = tol + 2.0 ** -25                     # half a step of its subnormals
    ok = (y.double() - ref).abs() <= tol
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off"


def check(dev, lead, Hq, Hk, D, rot, dtype, inter, norms, gap=0, few=False, seed=0):
    g = torch.Generator(device=dev).manual_seed(D * 7 + Hq + seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(dtype)  # noqa: E731
    buf = rnd(*lead, (Hq + Hk) * D + gap)
    k = buf[..., :Hk * D].unflatten(-1, (Hk, D)).detach().requires_grad_()
    q = buf[..., Hk * D:(Hk + Hq) * D].unflatten(-1, (Hq, D)).detach().requires_grad_()
    pos = torch.randint(-3, 130000, lead, device=dev, generator=g)
    f64 = torch.zeros(0, dtype=torch.float64, device=dev)
    freqs = rotary.rotary_freqs(rot, device=dev)[0] if rot else None
    f64 = freqs if rot else f64
    ws = [(rnd(D) + 1).requires_grad_() if n else None for n in norms]
    qo, ko = rotary.rotary(q, k, pos, freqs, interleaved=inter, mscale=1.2, q_weight=ws[0], k_weight=ws[1])
    gq, gk = rnd(*lead, Hq, D), rnd(*lead, Hk, D)
    if few:                 # only these tokens have a gradient: each one's share of the weights' sums shows
        on = torch.zeros(*lead, 1, 1, dtype=torch.bool, device=dev)
        n = on.numel()
        on.view(-1)[[0, 1, n // 2, n - 2, n - 1]] = True
        gq, gk = gq * on, gk * on
    leaves = [t for t in (q, k, *ws) if t is not None]
    grads = dict(zip(map(id, leaves), torch.autograd.grad((qo, ko), leaves, (gq, gk))))
    for x, w, y, gg in ((q, ws[0], qo, gq), (k, ws[1], ko, gk)):
        w64 = None if w is None else w.detach()
        rows_within(y.detach(), rotary64(x.detach(), w64, pos, f64, inter, 1.2, 1e-5), dtype)
        dx, dw, mag = rotary_grad64(x.detach(), w64, gg, pos, f64, inter, 1.2, 1e-5)
        # dx is a difference of h and its projection: roundings count at the size of the larger, |h| r
        r = 1.0 if w is None else ((x.detach().double() ** 2).mean(-1, keepdim=True) + 1e-5).rsqrt()
        h = gg.double().abs().amax(-1, keepdim=True) * 1.7 * (1.0 if w is None else float(w64.abs().max()))
        rows_within(grads[id(x)], dx, dtype, extra=(32 + D) * U32 * h * r * (1 + D ** 0.5))
        if w is not None:
            # every term off by D + 16 roundings; at most 100 additions in a row to one sum (a lane's units, 6 over
            # lanes, 4 over waves; the blocks' are added in 64 bits)
            tol = half_step(dtype) * dw.abs() + (D + 116) * U32 * mag + (2.0 ** -25 if dtype == HF else 0)
            assert bool(((grads[id(w)].double() - dw).abs() <= tol).all())


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("Hq,Hk,D,rot,gap", ROT)
def test_small(cuda, Hq, Hk, D, rot, gap, dtype, inter):
    for norms in ((True, True), (False, True), (False, False)):
        check(cuda, (3, 7), Hq, Hk, D, rot, dtype, inter, norms, gap)


# one token's heads fill at most half of a wave (2 + 1 x 64), or not; heads of several passes, units that mix q and k
# and end short (12 + 5), a wave of four heads in 32 bits (20 + 4 x 96), one element a lane (3 + 2 x 33)
SIZES = [(2, 1, 64, 64, BF), (2, 1, 64, 32, HF), (1, 4, 32, 32, F32), (16, 16, 128, 128, BF), (12, 5, 64, 32, HF),
         (20, 4, 96, 96, F32), (40, 1, 128, 64, BF), (3, 2, 33, 16, BF)]


@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, False)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T", [1024, 1031, 5003])
@pytest.mark.parametrize("Hq,Hk,D,rot,dtype", SIZES)
def test_training_sizes(cuda, Hq, Hk, D, rot, dtype, T, inter, norms):
    check(cuda, (T,), Hq, Hk, D, rot, dtype, inter, norms)
    if any(norms):
        check(cuda, (T,), Hq, Hk, D, rot, dtype, inter, norms, few=True)


@pytest.mark.parametrize("Hq,Hk,D,rot,dtype", [(16, 16, 128, 128, BF), (2, 1, 64, 64, BF), (12, 12, 64, 32, HF)])
def test_more_units_than_waves(cuda, Hq, Hk, D, rot, dtype):
    for norms in ((True, True), (False, False)):
        check(cuda, (20011,), Hq, Hk, D, rot, dtype, False, norms, few=any(norms))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("Hq,Hk,D,rot,inter,norm", [(2, 1, 64, 64, False, True), (32, 8, 128, 64, True, False),
                                                    (12, 12, 64, 32, False, True), (20, 4, 96, 96, False, True),
                                                    (3, 2, 33, 8, True, True)])
@pytest.mark.parametrize("T", [5, 1031, 5003])
def test_append_sizes(cuda, T, Hq, Hk, D, rot, inter, norm, dtype):
    g = torch.Generator(device=cuda).manual_seed(T + D)
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g).to(dtype)  # noqa: E731
    q, k, v, page = rnd(T, Hq, D), rnd(T, Hk, D), rnd(T, Hk, D), 16
    P = -(-T // page) + 2
    kc, vc = paged.page_pools(P, page, Hk, D, dtype, cuda)
    kc.fill_(3)
    slots = (torch.arange(T, device=cuda) + 5).int()          # one run from inside a column of eight
    slots[T // 2:] += 9
    pos = torch.randint(0, 130000, (T,), device=cuda, generator=g)
    freqs = rotary.rotary_freqs(rot, device=cuda)[0]
    w = [rnd(D) + 1 if norm else None for _ in range(2)]
    qo = paged.rotary_append(q, k, v, kc, vc, slots, pos, freqs, interleaved=inter, mscale=1.1, q_weight=w[0], k_weight=w[1])
    rows_within(qo, rotary64(q, w[0], pos, freqs, inter, 1.1, 1e-5), dtype)
    s = slots.long()
    rows_within(kc.permute(0, 2, 1, 3).reshape(P * page, Hk, D)[s], rotary64(k, w[1], pos, freqs, inter, 1.1, 1e-5), dtype)
    assert torch.equal(vc.permute(0, 2, 4, 1, 3).reshape(P * page, Hk, D)[s], v)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("Hq,D", [(1, 64), (16, 64), (3, 34)])
def test_far_positions(cuda, Hq, D, inter):
    """angles formed in 64 bits, off by three roundings of 2^-53 of the turns made, the definition's by one"""
    g = torch.Generator(device=cuda).manual_seed(D)
    pos = torch.tensor([0, 1, 10 ** 6, 10 ** 7 + 1, 150000001, -150000001, 2 ** 31 - 1, -2 ** 31, 10 ** 11 + 7], device=cuda)
    q = torch.randn(pos.numel(), Hq, D, device=cuda, generator=g)
    freqs = rotary.rotary_freqs(D, device=cuda)[0]
    y = rotary.rotary(q, q, pos, freqs, interleaved=inter)[0]
    ref = rotary64(q, None, pos, freqs, inter, 1.0, 1e-5)
    angle = 4 * 2.0 ** -53 * pos.double().abs()[:, None, None]                 # the fastest pair's, in radians
    tol = ((32 + D) * U32 + angle) * 2 ** 0.5 * ref.abs().amax(-1, keepdim=True)
    assert bool(((y.double() - ref).abs() <= tol).all())
