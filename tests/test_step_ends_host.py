"""The operators at a packed step's ends and its update without a GPU: refused calls, and the 64-bit definitions that the GPU
tests compare with against differences."""

from __future__ import annotations

import math
import shutil
from pathlib import Path

import numpy as np
import pytest
import torch

import ends_reference as R
import test_dpp_hazards as H

LIBRARY = Path(__file__).resolve().parents[1] / "etalii_dllm_amd" / "libdllm_hip.so"
needs_library = pytest.mark.skipif(not LIBRARY.exists(), reason="libdllm_hip.so not built")

# pointers that pass the null and alignment checks; the calls below are refused before anything is read or launched
P = 4096


@pytest.fixture(scope="module")
def K():
    from etalii_dllm_amd import kernels

    return kernels


EMBEDDING = dict(dtype=1, tokens=10, vocabulary=100, dim=16, accumulate=0, scale=1.0, stride=0)


@needs_library
@pytest.mark.parametrize(("change", "message"), [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 27), "tokens"),
    (dict(vocabulary=0), "vocabulary"), (dict(vocabulary=1 << 31), "vocabulary"), (dict(dim=0), "dim"), (dict(dim=(1 << 20) + 1), "dim"),
    (dict(tokens=1 << 26, dim=1 << 20), "2.40"), (dict(stride=15), "stride"), (dict(stride=-16), "stride"),
    (dict(stride=1 << 32), "stride"), (dict(scale=math.inf), "scale"),
    (dict(scale=math.nan), "scale"), (dict(scale=2.0 ** 61), "scale"),
])
def test_embedding_refuses_shapes(K, change, message):
    shape = K.TokenEmbedding(**{**EMBEDDING, **change})
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_token_embedding(shape, P, P, P, None))
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_token_embedding_backward(shape, P, P, P, P, 1 << 60, None))
    assert K.lib.dllm_hip_token_embedding_backward_workspace(shape) == 0


@needs_library
def test_embedding_refuses_pointers_and_workspaces(K):
    shape = K.TokenEmbedding(**EMBEDDING)
    for i, bad in [(0, None), (1, None), (2, None), (0, P + 1), (1, P + 4), (2, P + 1)]:
        args = [P] * 3
        args[i] = bad
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_token_embedding(shape, *args, None))
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_token_embedding_backward(shape, args[1], args[0], args[2], P, 1 << 60, None))
    need = K.lib.dllm_hip_token_embedding_backward_workspace(shape)
    assert need > 0
    for ws, size in ((P, need - 1), (None, need), (P + 8, need)):
        with pytest.raises(ValueError, match="workspace"):
            K.check(K.lib.dllm_hip_token_embedding_backward(shape, P, P, P, ws, size, None))
    for name, args in (("", 4), ("_backward", 4)):
        with pytest.raises(ValueError, match="null shape"):
            K.check(getattr(K.lib, f"dllm_hip_token_embedding{name}")(None, *[P] * 3, *([None] if not name else [P, 0, None])))
    none = K.TokenEmbedding(**{**EMBEDDING, "tokens": 0, "accumulate": 1})  # nothing to do: no pointer is looked at
    K.check(K.lib.dllm_hip_token_embedding(none, None, None, None, None))
    K.check(K.lib.dllm_hip_token_embedding_backward(none, None, None, None, None, 0, None))


LOSS = dict(dtype=1, rows=10, vocabulary=100, dim=16, accumulate=0, scale=1.0, softcap=0.0, hidden_stride=0, dhidden_stride=0)


@needs_library
@pytest.mark.parametrize(("change", "message"), [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "rows"), (dict(rows=1 << 27), "rows"),
    (dict(vocabulary=0), "vocabulary"), (dict(vocabulary=1 << 31), "vocabulary"), (dict(dim=0), "dim"), (dict(dim=(1 << 16) + 1), "dim"),
    (dict(rows=1 << 26, vocabulary=1 << 30), "2.48"), (dict(hidden_stride=15), "stride"), (dict(dhidden_stride=-1), "stride"),
    (dict(hidden_stride=1 << 32), "stride"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
    (dict(scale=1e-40), "scale"), (dict(softcap=-1.0), "softcap"), (dict(softcap=math.nan), "softcap"), (dict(softcap=1e-30), "softcap"),
    (dict(softcap=1e30), "softcap"),
])
def test_loss_refuses_shapes(K, change, message):
    shape = K.VocabularyLoss(**{**LOSS, **change})
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_vocabulary_loss(shape, *[P] * 6, 1 << 60, None))
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_vocabulary_loss_backward(shape, *[P] * 8, 1 << 60, None))
    assert K.lib.dllm_hip_vocabulary_loss_workspace(shape) == K.lib.dllm_hip_vocabulary_loss_backward_workspace(shape) == 0


@needs_library
def test_loss_refuses_pointers_and_workspaces(K):
    shape = K.VocabularyLoss(**LOSS)
    for i, bad in [(0, None), (1, None), (2, None), (0, P + 1), (1, P + 1), (2, P + 4), (3, P + 2), (4, P + 2)]:
        args = [P] * 6  # hidden weight targets loss lse workspace
        args[i] = bad
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_vocabulary_loss(shape, *args, 1 << 60, None))
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (4, None), (0, P + 1), (1, P + 1), (2, P + 4), (3, P + 2), (4, P + 1), (5, P + 1),
                   (6, P + 1)]:
        args = [P] * 8  # hidden weight targets lse dloss dhidden dweight workspace
        args[i] = bad
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_vocabulary_loss_backward(shape, *args, 1 << 60, None))
    for call, n in (("vocabulary_loss", 5), ("vocabulary_loss_backward", 7)):
        need = getattr(K.lib, f"dllm_hip_{call}_workspace")(shape)
        assert need > 0
        for ws, size in ((P, need - 1), (None, need), (P + 8, need)):
            with pytest.raises(ValueError, match="workspace"):
                K.check(getattr(K.lib, f"dllm_hip_{call}")(shape, *[P] * n, ws, size, None))
        with pytest.raises(ValueError, match="null shape"):
            K.check(getattr(K.lib, f"dllm_hip_{call}")(None, *[P] * n, P, 0, None))
    # nothing to do: no rows, or no results
    none = K.VocabularyLoss(**{**LOSS, "rows": 0, "accumulate": 1})
    K.check(K.lib.dllm_hip_vocabulary_loss(none, *[None] * 6, 0, None))
    K.check(K.lib.dllm_hip_vocabulary_loss_backward(none, *[None] * 8, 0, None))
    K.check(K.lib.dllm_hip_vocabulary_loss(shape, P, P, P, None, None, None, 0, None))
    K.check(K.lib.dllm_hip_vocabulary_loss_backward(shape, P, P, P, P, P, None, None, None, 0, None))


UPDATE = dict(dtype=1, batch=2, rows=10, cols=20, steps=5, eps=1e-7, scale=1.0, x_stride=0, x_batch_stride=0, out_stride=0, out_batch_stride=0)


@needs_library
@pytest.mark.parametrize(("change", "message"), [
    (dict(dtype=3), "dtype"), (dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(rows=0), "rows"), (dict(cols=0), "cols"),
    (dict(rows=65537), "rows"), (dict(cols=65537), "cols"), (dict(steps=-1), "steps"), (dict(steps=65), "steps"), (dict(eps=-1e-9), "eps"),
    (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(scale=math.nan), "scale"), (dict(scale=1e39), "scale"),
    (dict(x_stride=19), "row stride"), (dict(out_stride=-1), "row stride"), (dict(x_stride=1 << 62), "row stride"),
    (dict(x_batch_stride=199), "batch stride"), (dict(x_batch_stride=1 << 47), "batch stride"), (dict(out_stride=30, out_batch_stride=289), "batch stride"),
    (dict(batch=65535, rows=65536, cols=65536), "too many"),
])
def test_orthogonalize_refuses_shapes(K, change, message):
    shape = K.Orthogonalize(**{**UPDATE, **change})
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_orthogonalize(shape, None, P, 2 * P, P, 1 << 60, None))
    assert K.lib.dllm_hip_orthogonalize_workspace(shape) == 0


@needs_library
def test_orthogonalize_refuses_pointers_workspaces_and_coefficients(K):
    shape = K.Orthogonalize(**UPDATE)
    for i, bad in [(0, None), (1, None), (0, P + 1), (1, P + 1)]:
        args = [P, 2 * P]
        args[i] = bad
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_orthogonalize(shape, None, *args, P, 1 << 60, None))
    need = K.lib.dllm_hip_orthogonalize_workspace(shape)
    for ws, size in ((P, need - 1), (None, need), (P + 8, need)):
        with pytest.raises(ValueError, match="workspace"):
            K.check(K.lib.dllm_hip_orthogonalize(shape, None, P, 2 * P, ws, size, None))
    for bad in (math.nan, math.inf, 1e39):
        host = (K.C.c_double * 15)(*[1.0] * 14, bad)
        with pytest.raises(ValueError, match="coefficients"):
            K.check(K.lib.dllm_hip_orthogonalize(shape, host, P, 2 * P, P, 1 << 60, None))
    with pytest.raises(ValueError, match="in place"):
        K.check(K.lib.dllm_hip_orthogonalize(K.Orthogonalize(**{**UPDATE, "x_stride": 32}), None, P, P, P, 1 << 60, None))
    with pytest.raises(ValueError, match="null shape"):
        K.check(K.lib.dllm_hip_orthogonalize(None, None, P, P, P, 0, None))
    K.check(K.lib.dllm_hip_orthogonalize(K.Orthogonalize(**{**UPDATE, "batch": 0}), None, None, None, None, 0, None))


@needs_library
def test_array_functions_refuse(K):
    table, x = np.zeros((5, 4), np.float32), np.zeros((3, 4), np.float32)
    ids = np.zeros(3, np.int64)
    for call in (lambda: K.token_embedding(table, [0, 5]), lambda: K.token_embedding(table[0], ids), lambda: K.token_embedding(table, ids[None]),
                 lambda: K.token_embedding(table.astype(np.float64), ids), lambda: K.token_embedding_backward([0, 1, 5], x, 5),
                 lambda: K.token_embedding_backward(ids[:2], x, 5), lambda: K.token_embedding_backward(ids, x, 5, dtable=table[:4]),
                 lambda: K.token_embedding_backward(ids, x, 5, dtable=table.astype(np.float16)), lambda: K.vocabulary_loss(x, table, [0, 1, 5]),
                 lambda: K.vocabulary_loss(x, table[:, :3], ids), lambda: K.vocabulary_loss(x, table, ids[:2]),
                 lambda: K.vocabulary_loss(x.astype(np.float16), table, ids), lambda: K.vocabulary_loss(x, table, ids, softcap=-1.0),
                 lambda: K.vocabulary_loss_backward(x, table, ids, np.zeros(2), np.zeros(3)),
                 lambda: K.vocabulary_loss_backward(x, table, ids, np.zeros(3), np.zeros(3), dweight=x), lambda: K.orthogonalize(ids),
                 lambda: K.orthogonalize(x, 2, [(1, 2, 3)]), lambda: K.orthogonalize(np.zeros((2, 0), np.float32))):
        with pytest.raises(ValueError):
            call()


# ---- the definitions ----


def test_loss_definition_against_differences():
    g = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    h, w, dloss = rand(6, 5), rand(9, 5), rand(6)
    targets = torch.tensor([0, 8, -1, 3, 9, 3])
    for options in (dict(), dict(scale=0.3), dict(softcap=1.5), dict(scale=2.0, softcap=0.7)):
        lse = R.loss(h, w, targets, **options)["lse"][0]
        got = R.loss_backward(h, w, targets, lse, dloss, **options)
        value = lambda a, b: float((R.loss(a, b, targets, **options)["loss"][0] * dloss).sum())  # noqa: B023, E731
        for name, at, f in (("dhidden", h, lambda v: value(v, w)), ("dweight", w, lambda v: value(h, v))):  # noqa: B023
            d = rand(*at.shape)
            assert abs(R.finite_difference(f, at, d) - float((got[name][0] * d).sum())) < 1e-6
    old = rand(9, 5)
    added = R.loss_backward(h, w, targets, lse, dloss, old=old, **options)["dweight"][0]
    assert torch.allclose(added - old, got["dweight"][0], atol=1e-12)


def test_embedding_definition_against_differences():
    g = torch.Generator().manual_seed(2)
    table, dout = torch.randn(7, 3, generator=g, dtype=torch.float64), torch.randn(10, 3, generator=g, dtype=torch.float64)
    tokens = torch.tensor([0, 6, 6, -1, 7, 3, 3, 3, 0, 1])
    got = R.embedding_backward(tokens, dout, 7, 1.7)[0]
    d = torch.randn(7, 3, generator=g, dtype=torch.float64)
    f = lambda t: float((R.embedding(t, tokens, 1.7)[0] * dout).sum())  # noqa: E731
    assert abs(R.finite_difference(f, table, d) - float((got * d).sum())) < 1e-6


def test_orthogonalize_definition():
    """Singular vectors stay, singular values go through the polynomial; either side's products give the same."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 11, generator=g, dtype=torch.float64)
    u, s, v = torch.linalg.svd(x, full_matrices=False)
    s = s / (torch.linalg.norm(x) + 1e-7)
    for _ in range(5):
        a, b, c = R.QUINTIC
        s = a * s + b * s ** 3 + c * s ** 5
    assert (R.orthogonalize(x) - (u * s) @ v).abs().max() < 1e-12
    assert (R.orthogonalize(x.T) - R.orthogonalize(x).T).abs().max() < 1e-12
    rounded = R.orthogonalize(x, rounding=R.halves(1)) - R.orthogonalize(x)
    assert 1e-6 < rounded.abs().max() < 1e-2 and (R.orthogonalize(x, rounding=R.halves(2)) - R.orthogonalize(x)).abs().max() < 1e-5


@needs_library
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize(("rows", "vocabulary", "dim"), [
    (8192, 12287, 2304), (8192, 12287, 8192), (8192, 151936, 1536), (131072, 151936, 4096), (131072, 300, 4096), (100, 12287, 65536),
    (3000, 700, 65536), (16384, 256000, 2304), (1, 1, 1), (1, 2 ** 31 - 1, 8), (64, 2 ** 30, 65536)])
def test_loss_workspace_is_what_is_said_of_it(K, dtype, rows, vocabulary, dim):
    """256 MB of softmax, or a unit of 8192 (float32: 2048) of the vocabulary; half as much again at most of packed weights, by its
    own rule; 384 MB of dhidden's parts; rows of hidden and of float32."""
    size = 4 if dtype == 0 else 2
    need = K.lib.dllm_hip_vocabulary_loss_backward_workspace(K.VocabularyLoss(**{**LOSS, "dtype": dtype, "rows": rows, "vocabulary": vocabulary, "dim": dim}))
    unit, padded = 2048 if dtype == 0 else 8192, (dim + 31) // 32 * 32
    softmax = max(2 ** 28, rows * unit * size) + 64 * rows * size
    weight = max(2 ** 29, unit * padded * size)
    others = rows * padded * (2 * size + 4 + 4 + 1) + 8 * padded + rows * 64 + 5 * vocabulary + 2 ** 23
    assert 0 < need <= softmax + weight + 3 * 2 ** 27 + others, need


@pytest.mark.skipif(not Path(H.B.HIPCC).exists() and shutil.which("hipcc") is None, reason="hipcc not available")
@pytest.mark.parametrize("source", ["vocabulary_loss.hip", "orthogonalize.hip"])
def test_tiled_products_copies_respect_their_wait_states(tmp_path, source):
    """The tiled products' copies to LDS are inline statements whose base is in scalar registers."""
    asm = H._device_asm(tmp_path, source)
    copies = asm.count("global_load_lds_dwordx4")
    checked, bad = H.sgpr_base_hazards(asm)
    assert not bad, f"{len(bad)} SGPR-base hazards, e.g. {bad[:3]}"
    assert checked >= copies // 2 > 0
