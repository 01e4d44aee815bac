"""GPU: what the operators at a packed step's ends keep of their values' bits beside rows and matrices of other sizes, through the
C ABI on device tensors, against their 64-bit definitions."""

from __future__ import annotations

import math

import pytest
import torch

import ends_reference as R
from test_gpu_step_ends import K, Loss, gen, randn  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e-12, 1e-9, 1e-6, 1e3])
def test_float32_gradients_beside_a_row_of_zeroes(K, size):  # noqa: F811
    """A counted row of zeroes adds nothing to dweight, and takes no bits of the others' hidden states either."""
    g = gen(70)
    weight = randn(g, 700, 96, scale=0.2 / max(size, 1.0))
    hidden = randn(g, 90, 96, scale=size)
    hidden[31] = 0
    targets = torch.randint(0, 700, (90,), generator=g, device="cuda")
    dloss = torch.exp2(-torch.arange(90, device="cuda") % 7).float() / 90
    Loss(K, hidden, weight, targets).check(dloss)


def test_float32_gradients_of_zeroes_alone(K):  # noqa: F811
    g = gen(71)
    weight = randn(g, 300, 40)
    targets = torch.randint(0, 300, (70,), generator=g, device="cuda")
    p = Loss(K, torch.zeros(70, 40, device="cuda"), weight, targets)
    p.check(torch.full((70,), 0.1, device="cuda"))
    assert bool((p.backward(torch.full((70,), 0.1, device="cuda"))[1] == 0).all())
