"""Rotary / qk_norm attention on two CPU ranks (gloo) against one: heads split over TP, batches over DP."""
import pytest
import torch

from homebrewnlp_mtf_amd.config import ModelParameter
from homebrewnlp_mtf_amd.models.model import Model
from homebrewnlp_mtf_amd.parallel import state as pstate
from test_distributed import CFG, _gather_tp, _run, _single


@pytest.mark.parametrize("mode,extras", [("tp", "-rotary"), ("dp", "-rotary-qk_norm")])
def test_two_ranks_match_one(mode, extras):
    cfg = dict(CFG, rotary_fraction=0.5, block_config=[
        {"layer": ["norm-shift-scale", "attention-dot_product-context" + extras], "skip": True},
        {"layer": ["norm-shift-scale-group", "feed_forward-in:gelu"], "skip": True}])
    tr, losses = _single(cfg)
    ranks = _run(mode, cfg)
    for r in ranks:
        mean = sum(x["losses"][0] for x in ranks) / 2 if mode == "dp" else r["losses"][0]
        assert abs(mean - losses[0]) < 1e-5 * abs(losses[0])     # fp32 sums over another split of heads or batch
    for name, spec in tr.store.specs.items():
        want = tr.store.master[spec.offset:spec.offset + spec.numel].view(spec.full_shape)
        assert torch.allclose(_gather_tp(ranks, name, spec.full_shape, 2 if mode == "tp" else 1), want, atol=1e-4), name


def test_qk_norm_refuses_tp(monkeypatch):
    cfg = dict(CFG, block_config=[{"layer": ["attention-dot_product-context-qk_norm"]}])
    monkeypatch.setattr(pstate, "tp_size", lambda: 2)
    with pytest.raises(NotImplementedError):
        Model(ModelParameter(cfg), "cpu", tp_rank=0, tp_size=2)
