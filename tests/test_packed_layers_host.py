"""The packed-layer operators without a GPU: refused calls, and the 64-bit definitions that the GPU tests compare with
against differences."""

from __future__ import annotations

from pathlib import Path

import numpy as np
import pytest
import torch

import packed_reference as R

LIBRARY = Path(__file__).resolve().parents[1] / "etalii_dllm_amd" / "libdllm_hip.so"
needs_library = pytest.mark.skipif(not LIBRARY.exists(), reason="libdllm_hip.so not built")

# pointers that pass the null and alignment checks; the calls below are refused before anything is read or launched
P = 4096


@pytest.fixture(scope="module")
def K():
    from etalii_dllm_amd import kernels

    return kernels


ATTENTION = dict(dtype=1, tokens=10, documents=1, heads=4, kv_heads=2, head_dim=64, causal=1, window=0, scale=0.125,
                 softcap=0.0, q_stride=0, k_stride=0, v_stride=0, out_stride=0)


@needs_library
@pytest.mark.parametrize(("change", "message"), [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "tokens"),
    (dict(documents=-1), "documents"), (dict(documents=1 << 31), "documents"), (dict(heads=3), "multiple of kv heads"),
    (dict(kv_heads=0), "multiple of kv heads"), (dict(heads=0), "multiple of kv heads"), (dict(heads=65536), "65535"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=257), "head_dim"), (dict(window=-1), "window"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(softcap=float("inf")), "softcap"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"), (dict(q_stride=255), "stride"),
    (dict(k_stride=127), "stride"), (dict(v_stride=-128), "stride"), (dict(out_stride=1), "stride"),
    (dict(tokens=(1 << 31) - 1, documents=(1 << 31) - 1), "too many"),
])
def test_attention_refuses_shapes(K, change, message):
    shape = K.DocumentAttention(**{**ATTENTION, **change})
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_document_attention(shape, *[P] * 9, 1 << 60, None))
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_document_attention_backward(shape, *[P] * 13, 1 << 60, None))
    if message != "too many":
        assert K.lib.dllm_hip_document_attention_backward_workspace(shape) == 0


@needs_library
def test_attention_refuses_pointers_and_workspaces(K):
    shape = K.DocumentAttention(**ATTENTION)
    forward = [P] * 9  # q k v offsets prefix slopes out lse workspace
    for i, bad in [(0, None), (1, None), (2, None), (3, None), (6, None), (0, P + 1), (2, P + 1), (3, P + 4), (4, P + 4),
                   (5, P + 2), (6, P + 1), (7, P + 2)]:
        args = list(forward)
        args[i] = bad
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_document_attention(shape, *args, 1 << 60, None))
    backward = [P] * 13  # q k v offsets prefix slopes out lse dout dq dk dv workspace
    for i, bad in [(6, None), (7, None), (8, None), (9, None), (10, None), (11, None), (8, P + 1), (11, P + 1)]:
        args = list(backward)
        args[i] = bad
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_document_attention_backward(shape, *args, 1 << 60, None))
    need = K.lib.dllm_hip_document_attention_backward_workspace(shape)
    assert need > 0
    for args, size in ((backward, need - 1), ([*backward[:12], None], need), ([*backward[:12], P + 8], need)):
        with pytest.raises(ValueError, match="workspace"):
            K.check(K.lib.dllm_hip_document_attention_backward(shape, *args, size, None))
    with pytest.raises(ValueError, match="null shape"):
        K.check(K.lib.dllm_hip_document_attention(None, *forward, 0, None))
    # nothing to do: no pointer is looked at
    for none in (dict(tokens=0), dict(documents=0)):
        shape = K.DocumentAttention(**{**ATTENTION, **none})
        K.check(K.lib.dllm_hip_document_attention(shape, *[None] * 9, 0, None))
        K.check(K.lib.dllm_hip_document_attention_backward(shape, *[None] * 13, 0, None))


ROPE = dict(dtype=0, tokens=3, q_heads=2, k_heads=1, head_dim=16, pairs=8, axes=3, interleaved=0, inverse=0, q_stride=0,
            k_stride=0, q_out_stride=0, k_out_stride=0)


@needs_library
@pytest.mark.parametrize(("change", "message"), [
    (dict(dtype=4), "dtype"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "tokens"), (dict(q_heads=-1), "head"),
    (dict(k_heads=65536), "head"), (dict(pairs=9), "pairs"), (dict(pairs=257, head_dim=1024), "pairs"),
    (dict(pairs=-1), "pairs"), (dict(head_dim=0, pairs=0), "head_dim"), (dict(axes=0), "axes"), (dict(axes=256), "axes"),
    (dict(q_stride=31), "stride"), (dict(k_out_stride=15), "stride"),
    (dict(q_heads=65535, head_dim=65536), "elements"),
])
def test_rope_axes_refuses_shapes(K, change, message):
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_rope_axes(K.RopeAxes(**{**ROPE, **change}), *[P] * 7, None))


@needs_library
def test_rope_axes_refuses_pointers(K):
    shape = K.RopeAxes(**ROPE)
    for i, bad, message in [(0, None, "null"), (1, None, "null"), (2, None, "null"), (3, None, "null"), (4, None, "null"),
                            (5, None, "null"), (6, None, "null"), (0, P + 2, "aligned"), (6, P + 2, "aligned"),
                            (2, P + 4, "aligned"), (3, P + 4, "aligned")]:
        args = [P] * 7  # q k positions inv_freq pair_axis q_out k_out
        args[i] = bad
        with pytest.raises(ValueError, match=message):
            K.check(K.lib.dllm_hip_rope_axes(shape, *args, None))
    with pytest.raises(ValueError, match="in place"):
        K.check(K.lib.dllm_hip_rope_axes(K.RopeAxes(**{**ROPE, "q_stride": 64}), P, 2 * P, P, P, P, P, 3 * P, None))
    K.check(K.lib.dllm_hip_rope_axes(K.RopeAxes(**{**ROPE, "tokens": 0}), *[None] * 7, None))


NORM = dict(dtype=2, rows=3, dim=16, norm_placement=2, gate=1, unit_offset=0, eps=1e-6, residual_scale=1.0)


@needs_library
@pytest.mark.parametrize(("change", "message"), [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(dim=0), "dim"),
    (dict(dim=(1 << 20) + 1), "dim"), (dict(norm_placement=3), "norm_placement"), (dict(norm_placement=-1), "norm_placement"),
    (dict(gate=3), "gate"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
])
def test_residual_norm_refuses_shapes(K, change, message):
    shape = K.ResidualNorm(**{**NORM, **change})
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_residual_norm(shape, *[P] * 7, None))
    with pytest.raises(ValueError, match=message):
        K.check(K.lib.dllm_hip_residual_norm_backward(shape, *[P] * 13, 1 << 60, None))
    assert K.lib.dllm_hip_residual_norm_backward_workspace(shape) == 0


@needs_library
def test_residual_norm_refuses_pointers_and_workspaces(K):
    shape = K.ResidualNorm(**NORM)
    for i, bad in [(0, None), (1, None), (2, None), (5, None), (6, None), (0, P + 1), (2, P + 2), (3, P + 2), (4, P + 1),
                   (6, P + 1)]:
        args = [P] * 7  # x y gate post_weight pre_weight h n
        args[i] = bad
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_residual_norm(shape, *args, None))
    need = K.lib.dllm_hip_residual_norm_backward_workspace(shape)
    backward = [P] * 13  # h y gate post_weight pre_weight dh dn dx dy dgate dpost_weight dpre_weight workspace
    for i, bad in [(0, None), (1, None), (2, None), (6, None), (7, P + 1), (9, P + 2), (10, P + 2), (11, P + 3)]:
        args = list(backward)
        args[i] = bad
        with pytest.raises(ValueError, match="null" if bad is None else "aligned"):
            K.check(K.lib.dllm_hip_residual_norm_backward(shape, *args, need, None))
    for args, size in ((backward, need - 1), ([*backward[:12], None], need), ([*backward[:12], P + 8], need)):
        with pytest.raises(ValueError, match="workspace"):
            K.check(K.lib.dllm_hip_residual_norm_backward(shape, *args, size, None))
    with pytest.raises(ValueError, match="without a gate"):
        K.check(K.lib.dllm_hip_residual_norm_backward(K.ResidualNorm(**{**NORM, "gate": 0}), *backward, need, None))
    with pytest.raises(ValueError, match="not there"):
        K.check(K.lib.dllm_hip_residual_norm_backward(K.ResidualNorm(**{**NORM, "norm_placement": 0}), *backward, need, None))
    with pytest.raises(ValueError, match="null"):  # post alone: the gradient has to come from dh
        K.check(K.lib.dllm_hip_residual_norm_backward(K.ResidualNorm(**{**NORM, "norm_placement": 1}),
                                                      *backward[:5], None, *backward[6:11], None, P, need, None))
    K.check(K.lib.dllm_hip_residual_norm(K.ResidualNorm(**{**NORM, "rows": 0}), *[None] * 7, None))


@needs_library
def test_array_functions_refuse_what_does_not_fit(K):
    x = np.zeros((4, 2, 8), np.float32)
    with pytest.raises(ValueError, match="share one type"):
        K.document_attention(x, x.astype(np.float16), x, [0, 4], 1.0)
    with pytest.raises(ValueError, match="share one type"):
        K.document_attention(*[x.astype(np.float64)] * 3, [0, 4], 1.0)
    for offsets in ([0, 5], [-1, 4], [0, 3, 2], []):
        with pytest.raises(ValueError, match="offsets"):
            K.document_attention(x, x, x, offsets, 1.0)
    with pytest.raises(ValueError, match="prefix"):
        K.document_attention(x, x, x, [0, 4], 1.0, prefix=[1, 1])
    with pytest.raises(ValueError, match="slopes"):
        K.document_attention(x, x, x, [0, 4], 1.0, slopes=[1.0])
    with pytest.raises(ValueError, match="one shape"):
        K.document_attention(x, x, x[:, :1], [0, 4], 1.0)
    with pytest.raises(ValueError, match="positions"):
        K.rope_axes(x, x, np.zeros((3, 5)), np.ones(4), np.zeros(4))
    with pytest.raises(ValueError, match="pair_axis"):
        K.rope_axes(x, x, np.zeros((3, 4)), np.ones(4), [0, 1, 2, 3])
    with pytest.raises(ValueError, match="head_dim"):
        K.rope_axes(x, None, np.zeros((3, 4)), np.ones(5), np.zeros(5))
    with pytest.raises(ValueError, match="one shape"):
        K.residual_norm(x, x[:3])
    with pytest.raises(ValueError, match="gate"):
        K.residual_norm(x, x, gate=np.ones(8))
    with pytest.raises(ValueError, match="weight length"):
        K.residual_norm(x, x, pre_weight=np.ones(7, np.float32))
    with pytest.raises(ValueError, match="dn belongs"):
        K.residual_norm_backward(x, x, x)


# ---- the definitions' gradients against central differences ----
#
# f(x + t d) - f(x - t d) over 2 t is the derivative to (t^2 / 6) |f'''| and the values' rounding, 2^-52 |f| / t: with
# t = 1e-4 and these sizes both are below 1e-7 of the terms.


def directional(f, x, d, t=1e-4):
    return (f(x + t * d) - f(x - t * d)) / (2 * t)


@pytest.mark.parametrize("options", [dict(), dict(window=3), dict(causal=False, window=4), dict(prefix=[3, 0, 2]),
                                     dict(softcap=2.0, slopes=[0.5, 0.1, 0.3, 0.2]), dict(causal=False, softcap=3.0)])
def test_attention_definition_against_differences(options):
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(14, h, 6, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    dout, offsets = torch.randn(14, 4, 6, generator=g, dtype=torch.float64), [1, 8, 9, 13]

    def forward(q, k, v):
        return R.attention(q, k, v, offsets, 0.7, **options)

    # float64 inputs: the bounds mean nothing here, the values are the definition's
    res = forward(q, k, v)
    out, lse = res["out"][0], res["lse"][0]
    grads = R.attention(q, k, v, offsets, 0.7, out=out, lse=lse, dout=dout, **options)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn((q, k, v)[i].shape, generator=g, dtype=torch.float64)

        def value(x):
            args = [q, k, v]
            args[i] = x
            return float((forward(*args)["out"][0] * dout).sum())

        assert abs(directional(value, (q, k, v)[i], d) - float((grads[name][0] * d).sum())) < 1e-6


@pytest.mark.parametrize("placement", [0, 1, 2])
@pytest.mark.parametrize("gate", [0, 1, 2])
def test_residual_norm_definition_against_differences(placement, gate):
    g = torch.Generator().manual_seed(4)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, y, dh, dn = (rand(5, 7) for _ in range(4))
    w = dict(gate=None if gate == 0 else rand(7) if gate == 1 else rand(5, 7),
             post_weight=rand(7) if placement != 0 else None, pre_weight=rand(7) if placement != 1 else None)

    def forward(x, y, w):
        return R.residual_norm(x, y, w["gate"], w["post_weight"], w["pre_weight"], placement, 1e-3, True, 0.6)

    h = forward(x, y, w)["h"][0]
    grads = R.residual_norm(h, y, w["gate"], w["post_weight"], w["pre_weight"], placement, 1e-3, True, 0.6, dh=dh,
                            dn=dn if placement != 1 else None)

    def loss(x, y, w):
        res = forward(x, y, w)
        return float((res["h"][0] * dh).sum() + ((res["n"][0] * dn).sum() if placement != 1 else 0.0))

    for name, at in (("dx", x), ("dy", y), ("dgate", w["gate"]), ("dpost_weight", w["post_weight"]),
                     ("dpre_weight", w["pre_weight"])):
        if at is None:
            assert name not in grads
            continue
        d = rand(*at.shape)

        def value(v):
            if name == "dx":
                return loss(v, y, w)
            return loss(x, v, w) if name == "dy" else loss(x, y, {**w, name[1:]: v})

        assert abs(directional(value, at, d) - float((grads[name][0] * d).sum())) < 1e-6


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_definition_turns_back(interleaved):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 2, 10, generator=g, dtype=torch.float64)
    pos = torch.randint(0, 10 ** 6, (3, 6), generator=g)
    freq, axis = 10.0 ** -torch.arange(4, dtype=torch.float64), torch.tensor([0, 1, 2, 1])
    there = R.rope(x, pos, freq, axis, interleaved, False)[0]
    assert (R.rope(there, pos, freq, axis, interleaved, True)[0] - x).abs().max() < 1e-9
    # a rotation keeps lengths; dimensions past the pairs stay
    assert (there.square().sum(-1) - x.square().sum(-1)).abs().max() < 1e-9 and torch.equal(there[..., 8:], x[..., 8:])


@needs_library
def test_attention_refuses_scales_and_caps_that_float32_does_not_hold(K):
    """A cap that is zero in float32 would be none, and one whose quotient with the scale is no ordinary float32 would bend the
    scores otherwise than it says."""
    for change, message in [(dict(softcap=1e-50), "softcap"), (dict(softcap=1e-30), "softcap"), (dict(softcap=1e30), "softcap"),
                            (dict(softcap=3.4e38), "softcap"), (dict(scale=3e38), "scale"), (dict(scale=1e-40), "scale")]:
        shape = K.DocumentAttention(**{**ATTENTION, **change})
        with pytest.raises(ValueError, match=message):
            K.check(K.lib.dllm_hip_document_attention(shape, *[P] * 9, 1 << 60, None))
        with pytest.raises(ValueError, match=message):
            K.check(K.lib.dllm_hip_document_attention_backward(shape, *[P] * 13, 1 << 60, None))
        assert K.lib.dllm_hip_document_attention_workspace(shape) == 0
    for scale in (2.0 ** -60, 2.0 ** 60):
        for softcap in (0.0, 2.0 ** -64, 2.0 ** 64):
            shape = K.DocumentAttention(**{**ATTENTION, "scale": scale, "softcap": softcap})
            assert K.lib.dllm_hip_document_attention_workspace(shape) > 0


@needs_library
def test_rope_axes_refuses_tokens_that_a_thread_cannot_count(K):
    """A thread's count of a token's elements steps 256 past the last, in 32 bits: tokens of up to 2^31 - 257 elements."""
    for q_heads, k_heads, head_dim in [(32770, 0, 65532), (32769, 0, 65534), (1, 33373, 64346), (65535, 53624, 18022)]:
        assert 2 ** 31 - 256 <= (q_heads + k_heads) * head_dim < 2 ** 31
        shape = K.RopeAxes(**{**ROPE, "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim})
        with pytest.raises(ValueError, match="elements"):
            K.check(K.lib.dllm_hip_rope_axes(shape, *[P] * 7, None))
    shape = K.RopeAxes(**{**ROPE, "q_heads": 32768, "k_heads": 0, "head_dim": 65535})
    with pytest.raises(ValueError, match="null"):  # far enough below: its pointers are looked at
        K.check(K.lib.dllm_hip_rope_axes(shape, None, *[P] * 6, None))


@needs_library
@pytest.mark.parametrize("axis", [256, 512, -256, -1, 3])
def test_rope_axes_refuses_axes_that_eight_bits_wrap(K, axis):
    x = np.zeros((4, 2, 8), np.float32)
    with pytest.raises(ValueError, match="pair_axis"):
        K.rope_axes(x, x, np.zeros((3, 4)), np.ones(4), np.array([0, 1, 2, axis]))


@needs_library
def test_attention_refuses_more_empty_documents_than_tiles(K):
    """A launch has a tile for each document, empty ones too: their number is limited whatever the number of tokens."""
    for change in (dict(documents=(1 << 31) - 1), dict(documents=1 << 22)):
        shape = K.DocumentAttention(**{**ATTENTION, **change})
        with pytest.raises(ValueError, match="too many"):
            K.check(K.lib.dllm_hip_document_attention(shape, *[P] * 9, 1 << 60, None))
        with pytest.raises(ValueError, match="too many"):
            K.check(K.lib.dllm_hip_document_attention_backward(shape, *[P] * 13, 1 << 60, None))
    assert K.lib.dllm_hip_document_attention_workspace(K.DocumentAttention(**{**ATTENTION, "documents": (1 << 22) - 2})) > 0
