"""Captured training steps replayed back to back, at product sizes that take the GEMM's tile queue."""
import pytest
import torch

from homebrewnlp_mtf_amd.config import ModelParameter
from homebrewnlp_mtf_amd.ops import _lib as L
from homebrewnlp_mtf_amd.ops import raw
from homebrewnlp_mtf_amd.parallel import state as pstate
from homebrewnlp_mtf_amd.run.trainer import Trainer

pytestmark = pytest.mark.gpu

CFG = dict(model_mode="gpt", use_video=False, use_language=True, heads=16, features_per_head=128, depth=2,
           sequence_length=2048, train_batch_size=8, vocab_size=2048, intermediate_feed_forward_multiplier=2,
           memory_reduction_strategy="none", calculation_dtype="bfloat16", learning_rate=1e-4, embedding_stddev=0.02,
           learning_rate_config={"linear_warmup": {"final_step": 10}},
           optimizer="adaptive_clip:0.003-sm3-momentum:0.9:1:1-learning_rate")


@pytest.mark.parametrize("extras", ["", "-rotary", "-rotary-qk_norm"])
def test_back_to_back_replays_match_eager(cuda, extras):
    """no read-back, no kernel of the caller's between the replays: the weights are the eager run's, bit for bit"""
    pstate.set_mesh(pstate.Mesh())
    cfg = dict(CFG, block_config=[{"layer": ["norm-shift-scale", "attention-dot_product-context" + extras], "skip": True},
                                  {"layer": ["norm-shift-scale", "feed_forward-in:gelu"], "skip": True}])
    g = torch.Generator(device=cuda).manual_seed(1)
    toks = [torch.randint(0, 2048, (8, 2049, 1), device=cuda, generator=g) for _ in range(4)]
    batches = [{"token_x": t[:, :-1].contiguous(), "token_y": t[:, 1:].contiguous()} for t in toks]
    weights = []
    for graphs, watched in ((False, False), (True, False), (True, True)):
        torch.manual_seed(0)
        t = Trainer(ModelParameter(dict(cfg, use_hip_graphs=graphs)), cuda)
        queued = L.lib().obst_gemm4w_queue_calls()
        for i in range(12):
            loss = t.step(batches[i % 4])["loss"]
            if watched:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert L.lib().obst_gemm4w_queue_calls() > queued
        weights.append((t.store.master.clone(), float(loss)))
        t.close()
    assert weights[0][1] == weights[1][1] == weights[2][1], [w[1] for w in weights]
    assert all(torch.equal(weights[0][0], w[0]) for w in weights[1:])


def test_zero_at_any_alignment(cuda):
    for n in (0, 1, 3, 15, 16, 17, 31, 64, 4097, 1 << 20, (1 << 26) + 5):
        for at in (0, 1, 8, 15):
            t = torch.full((n + 48,), 7, dtype=torch.uint8, device=cuda)
            raw.zero_(t[at:at + n])
            assert not bool(t[at:at + n].any()) and bool((t[:at] == 7).all()) and bool((t[at + n:] == 7).all())


def test_zero_and_queued_products_in_a_graph(cuda):
    """a buffer zeroed, added to, and multiplied through the tile queue: every replay the eager result, with and without
    work and synchronisation in between"""
    g = torch.Generator(device=cuda).manual_seed(2)
    x, w = (torch.randn(n, 2048, device=cuda, generator=g).bfloat16() for n in (16384, 2048))
    acc = torch.empty(16384, 2048, device=cuda)

    def step():
        raw.zero_(acc)
        acc.add_(x)
        y = torch.empty(16384, 2048, dtype=torch.bfloat16, device=cuda)
        raw.gemm(raw.Operand(x, 0, 2048), raw.Operand(w, 0, 2048), raw.Operand(y, 0, 2048), 16384, 2048, 2048)
        return y
    queued = L.lib().obst_gemm4w_queue_calls()
    want = step()
    assert L.lib().obst_gemm4w_queue_calls() == queued + 1
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for i in range(12):
        y.fill_(float("nan"))
        if i % 3 == 1:
            torch.cuda.synchronize()
        for _ in range(1 + i % 2):
            graph.replay()
        if i % 3 == 2:
            torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(acc, x.float())
