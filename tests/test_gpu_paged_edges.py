"""Paged-cache kernels: calls at the edge of what they take."""
import pytest
import torch

from homebrewnlp_mtf_amd.ops import paged
from test_paged_edges_cpu import (outputs_in_place_and_shared, plan_refuses_shared_memory, release_cases,
                                  scores_of_minus_infinity, tangents)
from test_rotary_paged_cpu import _params

pytestmark = pytest.mark.gpu


def test_release_leaves_out_ids_outside_the_pool(cuda):
    release_cases(cuda, [(1, 1, 1), (5, 6, 20), (40, 130, 500), (1500, 64, 100000), (2500, 3, 300), (3, 1000, 2000)])


def test_release_row_without_ids(cuda):
    """rows that hold no page at all beside full ones"""
    table = torch.full((3, 200), -1, dtype=torch.int32, device=cuda)
    table[1] = torch.arange(200, device=cuda).int()
    stack = torch.full((200,), -5, dtype=torch.int32, device=cuda)
    lens, nfree = torch.full((3,), 3200, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    paged.page_release(torch.ones(3, dtype=torch.bool, device=cuda), lens, table, stack, nfree, 16)
    assert stack.tolist() == list(range(200)) and nfree.tolist() == [200] and lens.tolist() == [0, 0, 0]


def test_plan_refuses_shared_memory(cuda):
    plan_refuses_shared_memory(cuda)


def test_outputs_in_place_and_shared(cuda):
    outputs_in_place_and_shared(cuda)


def test_tangents(cuda):
    tangents(cuda)


def test_decoding_outside_the_context(cuda):
    """positions before and behind the context, eager and replayed: as dense caches, nothing kept and nothing read outside"""
    from test_gpu_rotary_paged import _model
    m, p = _model(cuda, kv_page_size=16)
    x = torch.randint(0, 256, (3, 96, 1), generator=torch.Generator().manual_seed(1)).to(cuda)
    steps = [torch.tensor(v, device=cuda) for v in ([96, 4, 50], [97, 5, -1], [10 ** 6, 6, -10 ** 6], [111, 7, 112])]
    out = []
    for page, graphs in ((0, False), (16, False), (16, True)):
        p.kv_page_size, p.decode_hip_graphs = page, graphs
        m.prefill(x, torch.tensor([95, 3, 95], device=cuda))
        out.append(torch.stack([m.decode(x[:, :1], s).clone() for s in steps]))
        m.end_decode()
    assert torch.equal(out[1], out[2])
    # two layers of about ten bf16 roundings each, every one off by 2^-8 of what it rounds at most
    a, b = out[0].flatten(2), out[1].flatten(2)
    assert bool(((a - b).norm(dim=-1) <= 20 * 2.0 ** -8 * a.norm(dim=-1)).all())


@pytest.mark.parametrize("strategy", ["checkpoint", "revnet", "momentum"])
def test_training_strategies(cuda, strategy):
    """gradients of recomputed and reconstructed blocks point where the CPU's do (bf16 activations through two layers)"""
    from homebrewnlp_mtf_amd.models.model import Model
    p = _params(calculation_dtype="bfloat16", storage_dtype="bfloat16", memory_reduction_strategy=strategy,
                features_per_head=64, sequence_length=96, vocab_size=256, rotary_fraction=0.5)
    grads = []
    t = torch.randint(0, 256, (3, 97, 1), generator=torch.Generator().manual_seed(3))
    for dev in (cuda, torch.device("cpu")):
        torch.manual_seed(0)
        m = Model(p, dev)
        if grads:
            m.store.master.copy_(master)
            if m.store.compute.data_ptr() != m.store.master.data_ptr():
                m.store.compute.copy_(master)
        master = m.store.master
        m.store.zero_grad()
        m(token_x=t[:, :-1].contiguous().to(dev), token_y=t[:, 1:].contiguous().to(dev))["loss"].backward()
        grads.append(m.store.grad.cpu())
    cos = torch.nn.functional.cosine_similarity
    assert cos(*grads, dim=0) > 0.97
    for n in [n for n in m.store.order if "qk_norm" in n]:
        sp = m.store.specs[n]
        assert cos(*(g[sp.offset:sp.offset + sp.numel] for g in grads), dim=0) > 0.97, n


def test_scores_of_minus_infinity(cuda):
    scores_of_minus_infinity(cuda)
