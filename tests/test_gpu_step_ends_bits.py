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


@pytest.mark.parametrize(("size", "spread"), [(0.1, 10), (0.1, 14), (1e-3, 12), (1e-6, 10), (1e3, 14), (1.0, 20)])
@pytest.mark.parametrize("zeroes", [False, True])
def test_float16_gradients_of_light_rows(K, size, spread, zeroes):  # noqa: F811
    """A row sure of its target, of the largest dloss, reaches hardly any other token; a light one with small hidden states keeps its
    bits in dweight's rows of those; so it does beside a row of zeroes."""
    g = gen(72)
    weight = randn(g, 600, 64, scale=0.25).half()
    targets = torch.tensor([3, 8, 9], device="cuda")
    sure = 40.0 * weight[3].float() / weight[3].float().square().sum()
    hidden = torch.stack([sure, torch.zeros_like(sure) if zeroes else sure, torch.zeros_like(sure)]).half()
    hidden[2] = randn(g, 64, scale=size).half()
    if not zeroes:
        targets[1] = 3
    if size > 1:
        weight[:, 32:] = 0  # the light row's large values reach no logit
        hidden[:, :32] = hidden[:, :32].clamp(-30, 30)
        hidden[2, :32] = 0
    # (the light row's part of dweight, about dloss / 600 times its hidden states, is no subnormal of float16)
    dloss = torch.tensor([1.0, 0.5, 2.0 ** -spread], device="cuda") * (2.0 ** spread * min(2.0 / size, 1e5))
    p = Loss(K, hidden, weight, targets)
    _, lse = p.forward()
    # (dhidden, of the heavy rows, is more than float16 holds)
    R.assert_within(p.backward(dloss)[1], R.light_rows(hidden, weight, targets, lse, dloss)["dweight"], "dweight")


def test_float16_gradients_of_unequal_rows(K):  # noqa: F811
    """Hidden states of every size, with dloss of every size, padding between them."""
    g = gen(73)
    weight = randn(g, 900, 72, scale=0.2).half()
    size = torch.exp2(-torch.arange(150, device="cuda") % 13).float()[:, None]
    hidden = (randn(g, 150, 72) * size).half()
    hidden[40] = 0
    targets = torch.randint(-200, 900, (150,), generator=g, device="cuda")
    dloss = torch.exp2(-torch.arange(150, device="cuda") % 11).float()
    p = Loss(K, hidden, weight, targets, softcap=9.0)
    _, lse = p.forward()
    got, want = p.backward(dloss), R.light_rows(hidden, weight, targets, lse, dloss, softcap=9.0)
    R.assert_within(got[0], want["dhidden"], "dhidden")
    R.assert_within(got[1], want["dweight"], "dweight")
