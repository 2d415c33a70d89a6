"""Paged-cache kernels: calls at the edge of what they take."""
import pytest
import torch

from homebrewnlp_mtf_amd.ops import paged
from test_paged_edges_cpu import outputs_in_place_and_shared, plan_refuses_shared_memory, release_cases, tangents

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
