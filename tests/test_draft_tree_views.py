"""Strided inputs of the draft-tree wrappers: what a view's rows are taken as, and which views are refused.  The tests of
a view touch no device, so CPU tensors stand in (device index -1)."""
import pytest
import torch

from rapidllm_b200 import ops
from rapidllm_b200._lib import RlError

CPU = -1


@pytest.mark.parametrize("make,shape", [
    (lambda: torch.zeros(1, 1, 512).expand(4, 1, 512), (4, 1, 512)),                 # one row for all sequences
    (lambda: torch.zeros(1, 1, 512).expand(1, 5, 512), (1, 5, 512)),                 # for all nodes
    (lambda: torch.zeros(1, 1, 512).expand(4, 5, 512), (4, 5, 512)),
    (lambda: torch.zeros(4, 1, 512).expand(4, 5, 512), (4, 5, 512)),
    (lambda: torch.zeros(1, 5, 512).expand(4, 5, 512), (4, 5, 512)),
    (lambda: torch.zeros(24, 256).expand(2, 8, 24, 256), (2, 8, 24, 256)),
    (lambda: torch.zeros(1, 1, 1, 256).expand(2, 8, 4, 256), (2, 8, 4, 256)),        # one head for all heads
    (lambda: torch.zeros(600).as_strided((1, 5, 512), (600, 4, 1)), (1, 5, 512)),    # rows that overlap
])
def test_rows_that_share_memory_are_refused(make, shape):
    with pytest.raises(RlError):
        ops._rows(make(), shape, CPU, "x")


@pytest.mark.parametrize("make,shape,row", [
    (lambda: torch.zeros(4, 5, 512), (4, 5, 512), 512),
    (lambda: torch.zeros(4, 5, 700)[..., 100:612], (4, 5, 512), 700),                # columns of a projection
    (lambda: torch.zeros(4, 1, 700)[..., :512], (4, 1, 512), 700),
    (lambda: torch.zeros(1, 1, 512).expand(1, 1, 512), (1, 1, 512), 512),
    (lambda: torch.zeros(2, 3, 4, 256), (2, 3, 4, 256), 1024),
    (lambda: torch.zeros(2, 0, 4, 256), (2, 0, 4, 256), 1024),
    (lambda: torch.zeros(0, 3, 512), (0, 3, 512), 512),
])
def test_distance_of_rows(make, shape, row):
    t = make()
    assert ops._rows(t, shape, CPU, "x") == (t.data_ptr(), row)


@pytest.mark.parametrize("make,shape", [
    (lambda: torch.zeros(24, 256).expand(2, 8, 24, 256), (2, 8, 24, 256)),           # a gate per channel
    (lambda: torch.zeros(1, 8, 24, 256).expand(2, 8, 24, 256), (2, 8, 24, 256)),
    (lambda: torch.zeros(2, 8, 1, 256).expand(2, 8, 24, 256), (2, 8, 24, 256)),      # one for all heads
    (lambda: torch.zeros(2, 1, 1, 256).expand(2, 1, 24, 256), (2, 1, 24, 256)),
    (lambda: torch.zeros(1, 1, 1, 256).expand(3, 1, 1, 256), (3, 1, 1, 256)),
    (lambda: torch.zeros(2, 8, 24, 1).expand(2, 8, 24, 256), (2, 8, 24, 256)),       # one per head
    (lambda: torch.zeros(2, 24, 8, 256).transpose(1, 2), (2, 8, 24, 256)),           # heads outside of the rows
    (lambda: torch.zeros(2, 8, 24), (2, 8, 24, 256)),
])
def test_gates_that_share_memory_are_refused(make, shape):
    with pytest.raises(RlError):
        ops._gate(make(), shape, CPU)


@pytest.mark.parametrize("make,row,head", [
    (lambda: torch.zeros(2, 8, 24, 256), 24 * 256, 256),
    (lambda: torch.zeros(2, 8, 24, 512)[..., 256:], 24 * 512, 512),                  # where the projection left it
    (lambda: torch.zeros(2, 8, 1, 256), 256, 256),
    (lambda: torch.zeros(1, 1, 24, 512)[..., :256], 24 * 512, 512),
])
def test_distances_of_a_gate(make, row, head):
    t = make()
    assert ops._gate(t, t.shape, CPU) == (t.data_ptr(), row, head)
