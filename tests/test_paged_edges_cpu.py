"""Rotary and paged-cache operators on the CPU: calls at the edge of what they take."""
import pathlib
import random
import re

import pytest
import torch

from homebrewnlp_mtf_amd.ops import _lib as L
from homebrewnlp_mtf_amd.ops import paged

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
