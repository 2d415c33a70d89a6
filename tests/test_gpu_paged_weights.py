"""Softmax weights of the paged attention against 64-bit results: weights far below the largest, weights that nearly
cancel."""
import math

import pytest
import torch

from homebrewnlp_mtf_amd.ops import paged
from paged_cases import U32, half_step

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
