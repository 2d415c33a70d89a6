"""Softmax weights of the paged attention against 64-bit results: weights far below the largest, weights that nearly
cancel."""
import math

import pytest
import torch

from homebrewnlp_mtf_amd.ops import paged
from paged_cases import U32, attn64, half_step, make_cache

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def one_request(scores, values, dtype, dev, page=16, D=32):
    """caches of one request whose key j has the score scores[j] against a query of ones in dim 0, and the value
    values[j] in every dim"""
    n = len(scores)
    P = -(-n // page)
    k = torch.zeros(P * page, D, dtype=torch.float64, device=dev)
    v = torch.zeros(P * page, D, dtype=torch.float64, device=dev)
    k[:n, 0] = scores
    v[:n] = values[:, None]
    kc = k.to(dtype).view(P, 1, page, D)
    vc = v.to(dtype).view(P, 1, page // 8, 8, D).transpose(-1, -2).contiguous()
    q = torch.zeros(1, 1, D, dtype=dtype, device=dev)
    q[..., 0] = 1
    table = torch.arange(P, dtype=torch.int32, device=dev)[None]
    return q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("peak", [0.0, 1.0])
@pytest.mark.parametrize("spread", [0.0, 0.5])
@pytest.mark.parametrize("n,gap", [(300, 8), (300, 14), (2048, 16), (2048, 19.5), (131072, 12), (131072, 16),
                                   (131072, 17.5), (131072, 20), (20011, 22)])
def test_small_weights(cuda, n, gap, spread, peak, dtype):
    """one key `gap` nats above all others: each of the others hardly counts, together they do"""
    g = torch.Generator(device=cuda).manual_seed(n)
    s = (torch.randn(n, device=cuda, generator=g, dtype=torch.float64) * spread).to(dtype).double()
    s[n // 3] = gap
    v = torch.ones(n, device=cuda, dtype=torch.float64)
    v[n // 3] = peak
    ref = float(torch.softmax(s, 0) @ v)
    o = paged.paged_attn(*one_request(s, v, dtype, cuda), 1.0)
    # in roundings of fp32: a score's product with the scale, the scale itself and the difference from the maximum are off
    # by three of its size in powers of two, the exponential by a few; sums of n weights run over at most n / 16 + 64
    # additions in a row (8 of every 128 tokens in a lane, then the lanes, waves and splits). Numerator and denominator
    # each. Two summands of fp16 keep 22 bits, and nothing below 2^-40 of the largest weight. Outputs of fp16 under 2^-14
    # (7.0e-6 at 2048 keys and 19.5 nats) are multiples of 2^-24: half of that
    size = max(float(s.abs().max()), gap) * 2 / math.log(2)
    rel = 2 * (3 * size + 8 + n / 16 + 64) * U32 + (2.0 ** -22 if dtype == HF else 0.0)
    tol = ref * (half_step(dtype) + rel) + (n * 2.0 ** -40 + 2.0 ** -25 if dtype == HF else 0.0)
    assert bool(((o.double() - ref).abs() <= tol).all()), (float(o[0, 0, 0]), ref)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", [2, 600])
def test_weights_that_cancel(cuda, n, dtype):
    """values a and -b in turn, with weights x and 1 where x a is nearly b: what is left of them shows the bits that the
    weights have (16 bits: up to 2^-17 of x a; an output of 8 bits sees that only where nothing else is left)"""
    H, D, page = 64, 32, 16
    g = torch.Generator(device=cuda).manual_seed(n)
    s = (-1.5 + 1.45 * torch.rand(H, device=cuda, generator=g)).to(dtype).double()
    x = s.exp()
    steps = 2.0 ** (7 if dtype == BF else 10)
    b = torch.arange(steps, 2 * steps, device=cuda, dtype=torch.float64) / steps       # every value in [1, 2)
    a = ((b / x[:, None]) * steps / 2).round() / steps * 2                             # the nearest in [1, 16), coarser
    a = a.to(dtype).double()
    left = (x[:, None] * a - b).abs()
    i = left.argmin(1, keepdim=True)
    a, b = a.gather(1, i), b[i]
    P = -(-n // page)
    j = torch.arange(P * page, device=cuda) % 2
    kc = torch.zeros(P, H, page, D, device=cuda, dtype=dtype)
    kc[..., 0] = j.to(dtype).view(P, 1, page)
    v = torch.where(j[None] == 1, a, -b).to(dtype)                                     # [H, tokens]
    vc = v.view(H, P, page // 8, 1, 8).transpose(0, 1).expand(P, H, page // 8, D, 8).contiguous()
    q = torch.zeros(1, H, D, device=cuda, dtype=dtype)
    q[0, :, 0] = s.to(dtype)
    table = torch.arange(P, dtype=torch.int32, device=cuda)[None]
    o = paged.paged_attn(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device=cuda), 1.0)[0].double()
    x = x[:, None]
    ref = (x * a - b) / (1 + x)
    # in roundings of fp32: the score's product and the scale by one each of 1.5 / ln 2, the exponential by two, its
    # summands by one, each product's sum by one of b: of x a, which is b. The sum of weights by n / 16 + 64 of its own
    tol = (half_step(dtype) + (n / 16 + 64) * U32) * ref.abs() + (2 * 1.5 + 4) * U32 * b / (1 + x)
    assert bool(((o - ref).abs() <= tol).all()), float(((o - ref).abs() / tol).max())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,Hq,Hk,D", [(1, 1, 1, 32), (45, 2, 1, 64), (300, 4, 2, 128), (5000, 3, 1, 96), (700, 2, 2, 256)])
def test_infinite_values(cuda, n, Hq, Hk, D, dtype):
    """infinities among the values that count: infinite where the definition is, NaN where it is (both signs, or a NaN),
    the other dims as ever"""
    kc, vc, table, ln = make_cache([n, 7], 16, Hk, D, dtype, cuda, seed=n)
    q = torch.randn(2, Hq, D, device=cuda, generator=torch.Generator(device=cuda).manual_seed(n)).to(dtype)
    scale = D ** -0.5

    def put(j, dim, x):
        vc[int(table[0, j // 16]), :, j % 16 // 8, dim, j % 8] = x
    put(0, 0, math.inf)
    put(n - 1, 1, -math.inf)
    put(n // 2, 2, math.nan)
    put(n // 3, 3, math.inf)
    put(n - 1, 3, -math.inf)
    for j in range(0, n, 3):
        put(j, 5, math.inf)
    # the key of the largest weight: its second summand is 0
    s = torch.stack([(kc[table[0].long(), h // (Hq // Hk)].reshape(-1, D)[:n].double() @ q[0, h].double())
                     for h in range(Hq)])
    put(int(s[0].argmax()), 6, -math.inf)
    ref, err = attn64(q, kc, vc, table, ln, scale)
    o = paged.paged_attn(q, kc, vc, table, ln, scale)
    fine = torch.isfinite(ref)
    assert bool(fine[1].all()) and bool(fine[0, :, 7:].all()) and not bool(fine[0, :, 0].any())
    assert torch.equal(torch.nan_to_num(o.double()[~fine], nan=7.0), torch.nan_to_num(ref[~fine], nan=7.0))
    assert bool(((o.double() - ref).abs()[fine] <= (half_step(dtype) * ref.abs() + err)[fine]).all())
