"""GPU: the packed-layer operators at the ends of their ranges, within the bounds of packed_reference."""

from __future__ import annotations

import pytest
import torch

import packed_reference as R
from test_gpu_packed_layers import K, gen, norm_backward, norm_forward, randn  # noqa: F401  (K: the fixture)

pytestmark = pytest.mark.gpu


# ---- norms ----


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize(("size", "eps"), [(1e14, 1e-6), (1e-14, 0.0)])
@pytest.mark.parametrize("placement", [0, 1, 2])
@pytest.mark.parametrize("dim", [2048, 1001, 20000])
def test_norm_gradients_of_very_large_and_small_rows(K, dtype, size, eps, placement, dim):  # noqa: F811
    """Rows whose inverse root mean square, cubed, is no float32: the gradients are as good as those of ordinary rows (a row
    kernel of 16-byte vectors, one of single elements, and the one for rows of any length)."""
    g, dt, rows = gen(70), R.DTYPES[dtype], 9
    x, y = (randn(g, rows, dim, scale=size).to(dt) for _ in range(2))
    post, pre = (1 + randn(g, dim, scale=0.2) if there else None for there in (placement != 0, placement != 1))
    gate = randn(g, dim)
    dh, dn = (randn(g, rows, dim, scale=0.1).to(dt) for _ in range(2))
    # upstream gradients of the sizes that make h's two uses alike
    dh, dn = (dh / size).to(dt), dn if placement != 1 else None
    shape = K.ResidualNorm(K.DTYPES[dtype], rows, dim, placement, 1, 0, eps, 0.5)
    h, n = norm_forward(K, shape, x, y, gate, post, pre)
    want = R.residual_norm(x, y, gate, post, pre, placement, eps, False, 0.5)
    R.assert_within(h, want["h"], "h")
    if n is not None:
        R.assert_within(n, want["n"], "n")
    got = norm_backward(K, shape, h, y, gate, post, pre, dh, dn)
    want = R.residual_norm(h, y, gate, post, pre, placement, eps, False, 0.5, dh=dh, dn=dn)
    assert got.keys() == want.keys()
    for name in want:
        R.assert_within(got[name], want[name], name)
