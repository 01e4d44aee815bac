"""GPU: the packed-layer operators through the C ABI on device tensors, against their 64-bit definitions within the
bounds of packed_reference, and what they promise beside that: a document's bits are its own, hidden values do not
matter, rows of no document stay as they were, strides, streams, graphs, aliasing."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import packed_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from etalii_dllm_amd import kernels

    return kernels


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


NAMES = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.float16: "float16"}


class Attention:
    """One document_attention problem on device tensors and its calls."""

    def __init__(self, K, q, k, v, offsets, causal=True, window=0, prefix=None, softcap=0.0, slopes=None, scale=None):
        self.K, self.q, self.k, self.v = K, q, k, v
        t, h, hd = q.shape
        self.scale = 1.0 / math.sqrt(hd) if scale is None else scale
        self.offsets = torch.tensor(offsets, dtype=torch.int64, device="cuda")
        self.prefix = None if prefix is None else torch.tensor(prefix, dtype=torch.int64, device="cuda")
        self.slopes = None if slopes is None else torch.as_tensor(slopes, dtype=torch.float32, device="cuda")
        self.options = dict(causal=causal, window=window, prefix=prefix, softcap=softcap, slopes=slopes)
        self.shape = K.DocumentAttention(K.DTYPES[NAMES[q.dtype]], t, len(offsets) - 1, h, k.shape[1], hd, int(causal),
                                         window, self.scale, softcap, q.stride(0), k.stride(0), v.stride(0), h * hd)
        need = max(K.lib.dllm_hip_document_attention_workspace(self.shape),
                   K.lib.dllm_hip_document_attention_backward_workspace(self.shape))
        self.workspace = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        self.out = torch.zeros(t, h, hd, dtype=q.dtype, device="cuda")
        self.lse = torch.zeros(h, t, device="cuda")

    def inputs(self):
        return [self.shape, ptr(self.q), ptr(self.k), ptr(self.v), ptr(self.offsets), ptr(self.prefix), ptr(self.slopes)]

    def forward(self):
        self.K.check(self.K.lib.dllm_hip_document_attention(*self.inputs(), ptr(self.out), ptr(self.lse),
                                                            ptr(self.workspace), self.workspace.numel(), stream()))
        return self.out, self.lse

    def backward(self, dout, grads=None):
        if grads is None:
            grads = [torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda").zero_()
                     for x in (self.q, self.k, self.v)]
        self.K.check(self.K.lib.dllm_hip_document_attention_backward(
            *self.inputs(), ptr(self.out), ptr(self.lse), ptr(dout), *map(ptr, grads), ptr(self.workspace),
            self.workspace.numel(), stream()))
        return grads

    def check(self, dout=None, what=""):
        out, lse = self.forward()
        want = R.attention(self.q, self.k, self.v, self.offsets, self.scale, **self.options)
        R.assert_within(out, want["out"], f"{what} out")
        R.assert_within(lse, want["lse"], f"{what} lse")
        if dout is None:
            return
        grads = self.backward(dout)
        want = R.attention(self.q, self.k, self.v, self.offsets, self.scale, out=out, lse=lse, dout=dout, **self.options)
        for name, got in zip(("dq", "dk", "dv"), grads):
            R.assert_within(got, want[name], f"{what} {name}")


def problem(K, seed, dtype, offsets, tokens, heads, kv_heads, head_dim, **options):
    g = gen(seed)
    q, k, v = (randn(g, tokens, n, head_dim, dtype=dtype) for n in (heads, kv_heads, kv_heads))
    dout = randn(g, tokens, heads, head_dim, dtype=dtype, scale=0.1)
    return Attention(K, q, k, v, offsets, **options), dout


# documents of one token, of none, shorter and longer than any tile, ending inside one; tokens before and after all of them
PACK = [2, 3, 3, 40, 104, 233, 234, 434]
OPTIONS = {
    "causal": dict(),
    "full": dict(causal=False),
    "window": dict(window=33),
    "window_one": dict(window=1),
    "window_full": dict(causal=False, window=70),
    "prefix": dict(prefix=[0, 5, 20, 64, 129, 1, 77]),
    "prefix_window": dict(prefix=[1, 0, 37, 10, 3, 0, 150], window=12),
    "cap": dict(softcap=5.0),
    "bias": dict(slopes=[0.5, 0.25, 0.125, 0.0625]),
    "all": dict(prefix=[1, 0, 3, 64, 100, 1, 0], window=65, softcap=3.0, slopes=[1.0, 0.01, 0.0, 0.3]),
    "all_full": dict(causal=False, window=90, softcap=3.0, slopes=[1.0, 0.01, 0.0, 0.3]),
}


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("options", OPTIONS)
def test_attention_masks(K, dtype, options):
    p, dout = problem(K, 1, R.DTYPES[dtype], PACK, 437, 4, 2, 64, **OPTIONS[options])
    p.check(dout, options)


# every padded width, odd sizes that are no whole 16-byte chunks, one head and shared ones
@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("head_dim", "heads", "kv_heads"),
                         [(1, 2, 2), (8, 3, 1), (17, 4, 4), (32, 2, 1), (63, 3, 3), (80, 4, 2), (96, 5, 1), (128, 6, 2),
                          (129, 2, 1), (160, 2, 2), (192, 2, 1), (255, 1, 1), (256, 4, 2)])
def test_attention_head_layouts(K, dtype, head_dim, heads, kv_heads):
    p, dout = problem(K, 2, R.DTYPES[dtype], [0, 70, 71, 200], 200, heads, kv_heads, head_dim, window=150, softcap=4.0)
    p.check(dout, f"{head_dim}")


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1025])
def test_attention_lengths(K, dtype, tokens):
    p, dout = problem(K, 3, R.DTYPES[dtype], [0, tokens], tokens, 2, 1, 128)
    p.check(dout, f"{tokens}")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_attention_of_many_documents(K, dtype):
    """More documents than a wave has lanes, many of them empty."""
    lengths = [(7 * i) % 11 * ((3 * i) % 4 != 0) for i in range(150)]
    offsets = np.concatenate([[0], np.cumsum(lengths)]).tolist()
    p, dout = problem(K, 4, R.DTYPES[dtype], offsets, offsets[-1] + 1, 2, 1, 64)
    p.check(dout)
    p, dout = problem(K, 4, R.DTYPES[dtype], [0] * 70 + [5] + [5] * 70 + [150], 150, 2, 1, 64, prefix=[2] * 141)
    p.check(dout)


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_attention_of_large_scores(K, dtype):
    """Scores in the hundreds: one key takes all of a row, and the running maximum moves far between tiles."""
    g = gen(5)
    dt = R.DTYPES[dtype]
    q, k, v = randn(g, 300, 2, 64, dtype=dt, scale=6.0), randn(g, 300, 2, 64, dtype=dt, scale=6.0), randn(g, 300, 2, 64, dtype=dt)
    k *= torch.linspace(0.1, 3.0, 300, device="cuda")[:, None, None].to(dt)  # the later keys' scores are larger
    p = Attention(K, q, k, v, [0, 300])
    p.check(randn(g, 300, 2, 64, dtype=dt))
    Attention(K, q, k, v, [0, 300], causal=False, softcap=50.0).check(randn(g, 300, 2, 64, dtype=dt))


@pytest.mark.parametrize("scale", [1e-6, 1e3])
def test_float16_gradients_of_any_size(K, scale):
    """Upstream gradients far below and above one (a loss scale): the float16 products inside keep their bits. With 1e3
    the upstream values go to about 4000; with 1e-6 they are subnormal themselves, and so are the results."""
    g = gen(6)
    q, k, v = (randn(g, 700, h, 64, dtype=torch.float16) for h in (4, 2, 2))
    p = Attention(K, q, k, v, [0, 700])
    p.check((randn(g, 700, 4, 64) * scale).half())


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("options", ["causal", "full", "all"])
def test_a_document_alone_and_in_a_pack(K, dtype, options):
    """The bits of a document's results do not depend on what is packed with it, nor on where it lies."""
    o = OPTIONS[options]
    lengths = [0, 1, 37, 64, 129, 1, 200]
    p, dout = problem(K, 7, R.DTYPES[dtype], PACK, 437, 4, 2, 64, **o)
    out, lse = (t.clone() for t in p.forward())
    grads = p.backward(dout)
    again = p.backward(dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    for d, (b, e) in enumerate(zip(PACK, PACK[1:])):
        if b == e:
            continue
        one = dict(o, prefix=None if o.get("prefix") is None else [o["prefix"][d]])
        s = Attention(K, p.q[b:e].clone(), p.k[b:e].clone(), p.v[b:e].clone(), [0, e - b], **one)
        out1, lse1 = s.forward()
        assert torch.equal(out1, out[b:e]) and torch.equal(lse1, lse[:, b:e]), d
        for got, want in zip(s.backward(dout[b:e].clone()), grads):
            assert torch.equal(got, want[b:e]), d
    assert len(lengths) == 7


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_tokens_of_no_document_are_not_touched(K, dtype):
    p, dout = problem(K, 8, R.DTYPES[dtype], [5, 70, 90], 100, 4, 2, 64)
    want = [t.clone() for t in p.forward()] + [t.clone() for t in p.backward(dout)]
    outside = torch.ones(100, dtype=torch.bool, device="cuda")
    outside[5:90] = False
    for t in (p.q, p.k, p.v, dout):
        t[outside] = float("nan")
    p.out.fill_(7.0), p.lse.fill_(7.0)
    grads = [torch.full_like(t, 7.0) for t in (p.q, p.k, p.v)]
    p.forward()
    p.backward(dout, grads)
    for got, ref in zip([p.out, p.lse.T, *grads], [want[0], want[1].T, *want[2:]]):
        assert torch.equal(got[~outside], ref[~outside]) and bool((got[outside] == 7.0).all())


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("head_dim", [64, 72])
def test_hidden_values_do_not_matter(K, dtype, value, head_dim):
    """A token that holds infinities or NaN spoils the rows that see it and no others, forward and backward: the others
    are within the bounds of the clean inputs' results."""
    n, bad, options = 150, 77, dict(window=40)
    p, dout = problem(K, 9, R.DTYPES[dtype], [0, n, 2 * n], 2 * n, 4, 2, head_dim, **options)
    out, lse = (t.clone() for t in p.forward())
    clean = R.attention(p.q, p.k, p.v, p.offsets, p.scale, **options)
    grads = R.attention(p.q, p.k, p.v, p.offsets, p.scale, out=out, lse=lse, dout=dout, **options)
    q, dout_clean = p.q.clone(), dout.clone()

    def within(got, want, rows, what):
        R.assert_within(got[rows], (want[0][rows], want[1][rows]), what)

    p.k[bad], p.v[bad] = value, value
    got, got_lse = p.forward()
    sees = torch.zeros(2 * n, dtype=torch.bool, device="cuda")
    sees[bad:bad + 40] = True
    within(got, clean["out"], ~sees, "out"), within(got_lse.T, [t.T for t in clean["lse"]], ~sees, "lse")
    assert not bool(torch.isfinite(got[sees]).all(dim=2).any())
    # backward, from the clean forward's results: the rows of dq that do not see the token, and the other keys' dk and dv
    # (dS of the token's own column alone is spoilt)
    p.out.copy_(out), p.lse.copy_(lse)
    dq, dk, dv = p.backward(dout)
    other = torch.ones(2 * n, dtype=torch.bool, device="cuda")
    other[bad] = False
    within(dq, grads["dq"], ~sees, "dq"), within(dk, grads["dk"], other, "dk"), within(dv, grads["dv"], other, "dv")
    # a query and an upstream gradient that hold it: the keys that the query does not see, and the other queries
    p, dout = problem(K, 9, R.DTYPES[dtype], [0, n, 2 * n], 2 * n, 4, 2, head_dim, **options)
    assert torch.equal(p.q, q) and torch.equal(dout, dout_clean)
    p.out.copy_(out), p.lse.copy_(lse)
    p.q[bad], dout[bad] = value, value
    dq, dk, dv = p.backward(dout)
    seen = torch.zeros(2 * n, dtype=torch.bool, device="cuda")
    seen[bad - 39:bad + 1] = True
    within(dq, grads["dq"], other, "dq"), within(dk, grads["dk"], ~seen, "dk"), within(dv, grads["dv"], ~seen, "dv")


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("head_dim", [128, 256])
def test_hidden_values_do_not_matter_to_wide_heads(K, dtype, head_dim):
    """float32 heads of 256 are shared by pairs of waves, which have to agree on the rows that are spoilt."""
    test_hidden_values_do_not_matter(K, dtype, float("nan"), head_dim)
    test_hidden_values_do_not_matter(K, dtype, float("inf"), head_dim)


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("head_dim", [64, 256])
def test_a_document_of_nan(K, dtype, head_dim):
    """Of two documents one is NaN throughout: its results are NaN, the other's are what they were."""
    n = 300
    p, dout = problem(K, 13, R.DTYPES[dtype], [0, n, 2 * n], 2 * n, 4, 2, head_dim)
    want = [t.clone() for t in p.forward()] + [t.clone() for t in p.backward(dout)]
    for t in (p.q, p.k, p.v, dout):
        t[:n] = float("nan")
    out, lse = p.forward()
    for got, ref in zip([out, lse.T, *p.backward(dout)], [want[0], want[1].T, *want[2:]]):
        assert bool(torch.isnan(got[:n]).all()) and torch.equal(got[n:], ref[n:])


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_a_key_of_infinite_score(K, dtype):
    """The rows that see it are NaN where its score is plus infinity, and do without it where that is minus infinity."""
    n, hd = 200, 64
    p, _ = problem(K, 14, R.DTYPES[dtype], [0, n], n, 2, 1, hd)
    p.q[:, :, 0] = torch.where(torch.arange(n, device="cuda")[:, None] % 2 == 0, 1.0, -1.0).to(p.q.dtype)
    p.k[0, 0] = 0.0
    want, want_lse = (t.clone() for t in Attention(K, p.q[1:], p.k[1:], p.v[1:], [0, n - 1]).forward())
    p.k[0, 0, 0] = float("inf")
    p.k[0, 0, 1:] = 1e-3
    out, lse = p.forward()
    even = torch.arange(n, device="cuda") % 2 == 0
    assert bool(torch.isnan(out[even]).all()) and bool(torch.isnan(lse[:, even]).all())
    odd = ~even
    odd[0] = False
    eps = torch.finfo(p.q.dtype).eps
    # the same keys in tiles that start one key earlier: two results within their roundings, and float32's of 200 terms
    tol = (2 * eps + 200 * 2.0**-22) * p.v.float().abs().max().item()
    assert float((out[odd].float() - want[odd[1:]].float()).abs().max()) <= tol
    assert float((lse[:, odd] - want_lse[:, odd[1:]]).abs().max()) <= 200 * 2.0**-22 * 8


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("head_dim", [64, 120, 128, 256])
@pytest.mark.parametrize("options", [dict(), dict(causal=False, window=50)])
def test_a_document_in_a_large_pack(K, dtype, head_dim, options):
    """A document's bits are the same alone and among as many that the gradients are launched otherwise, or the tiles
    come in another order."""
    lengths = [(53 * i) % 211 + 7 for i in range(80)]
    lengths[40] = 600
    offsets = np.concatenate([[0], np.cumsum(lengths)]).tolist()
    p, dout = problem(K, 12, R.DTYPES[dtype], offsets, offsets[-1], 8, 2, head_dim, **options)
    out, lse = p.forward()
    grads = p.backward(dout)
    for d in (0, 17, 40, 79):
        b, e = offsets[d], offsets[d + 1]
        s = Attention(K, p.q[b:e].clone(), p.k[b:e].clone(), p.v[b:e].clone(), [0, e - b], **options)
        out1, lse1 = s.forward()
        assert torch.equal(out1, out[b:e]) and torch.equal(lse1, lse[:, b:e]), d
        for got, want in zip(s.backward(dout[b:e].clone()), grads):
            assert torch.equal(got, want[b:e]), d


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("extra", "shift"), [(0, 0), (8, 0), (3, 0), (0, 1)])
def test_attention_of_a_fused_projection(K, dtype, extra, shift):
    """q, k and v as parts of one projection's rows; strides and starts that are whole 16-byte chunks or not. The gradients
    go into one fused array of the same layout, and what lies between is left as it was."""
    dt, heads, kv, hd, n = R.DTYPES[dtype], 4, 2, 64, 190
    g = gen(10)
    width = (heads + 2 * kv) * hd + extra
    flat = randn(g, n * width + shift, dtype=dt)
    rows = flat[shift:].view(n, width)
    parts = [(0, heads), (heads, kv), (heads + kv, kv)]
    q, k, v = (rows[:, a * hd:(a + c) * hd].unflatten(1, (c, hd)) for a, c in parts)
    p = Attention(K, q, k, v, [0, 100, 190], prefix=[30, 2])
    dout = randn(g, n, heads, hd, dtype=dt)
    p.check(dout)
    fused = torch.full((n * width + shift,), 5.0, dtype=dt, device="cuda")
    frows = fused[shift:].view(n, width)
    into = [frows[:, a * hd:(a + c) * hd].unflatten(1, (c, hd)) for a, c in parts]
    want = p.backward(dout)
    for got, ref in zip(p.backward(dout, into), want):
        assert torch.equal(got, ref)
    assert bool((frows[:, (heads + 2 * kv) * hd:] == 5.0).all()) and bool((fused[:shift] == 5.0).all())


def test_attention_past_32_bit_offsets(K):
    """Token strides that put the last tokens' elements past 2^32 bytes and 2^31 elements."""
    n, stride = 300, 9_000_000
    g = gen(11)
    parts = []
    for heads in (2, 1, 1):
        t = torch.empty_strided((n, heads, 64), (stride, 64, 1), dtype=torch.bfloat16, device="cuda")
        t.copy_(randn(g, n, heads, 64))
        parts.append(t)
    assert (n - 1) * stride > 2 ** 31
    p = Attention(K, *parts, [0, 299])
    near = Attention(K, *(t.contiguous() for t in parts), [0, 299])
    out, lse = near.forward()
    dout = randn(g, n, 2, 64, dtype=torch.bfloat16)
    grads = near.backward(dout)
    assert torch.equal(p.forward()[0], out) and torch.equal(p.lse, lse)
    for got, ref in zip(p.backward(dout), grads):
        assert torch.equal(got, ref)


def test_attention_without_lse_and_with_offsets_out_of_range(K):
    """lse may be left out. Offsets and prefixes beyond the tokens are cut to them: the results are those of the cut ones."""
    p, _ = problem(K, 12, torch.bfloat16, [0, 50, 80], 80, 2, 1, 64, prefix=[50, 0])
    want = p.forward()[0].clone()
    p.offsets.copy_(torch.tensor([-3, 50, 1 << 40]))
    p.prefix.copy_(torch.tensor([1 << 40, -5]))
    p.out.zero_()
    p.K.check(p.K.lib.dllm_hip_document_attention(*p.inputs(), ptr(p.out), None, ptr(p.workspace),
                                                  p.workspace.numel(), stream()))
    assert torch.equal(p.out, want)


def test_attention_of_a_long_document(K):
    p, dout = problem(K, 13, torch.bfloat16, [0, 5001, 5100], 5100, 2, 1, 128, window=1500, prefix=[700, 0])
    p.check(dout)
    p, dout = problem(K, 13, torch.float16, [0, 4099], 4099, 1, 1, 64, causal=False)
    p.check(dout)


# ---- rotary positions ----


def rope(K, q, k, pos, freq, axis, interleaved, inverse, q_out=None, k_out=None):
    t, h, hd = q.shape
    q_out = torch.full_like(q, 9.0) if q_out is None else q_out
    if k is not None and k_out is None:
        k_out = torch.full_like(k, 9.0)
    shape = K.RopeAxes(K.DTYPES[NAMES[q.dtype]], t, h, 0 if k is None else k.shape[1], hd, len(freq), pos.shape[0],
                       int(interleaved), int(inverse), q.stride(0), 0 if k is None else k.stride(0), q_out.stride(0),
                       0 if k is None else k_out.stride(0))
    K.check(K.lib.dllm_hip_rope_axes(shape, ptr(q), ptr(k), ptr(pos), ptr(freq), ptr(axis), ptr(q_out), ptr(k_out), stream()))
    return q_out, k_out


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("tokens", "heads", "kv_heads", "head_dim", "pairs"),
                         [(1, 16, 8, 128, 64), (37, 4, 2, 64, 32), (130, 3, 1, 96, 40), (65, 2, 2, 80, 20), (9, 1, 1, 2, 1),
                          (33, 2, 1, 67, 31), (5, 3, 3, 512, 256), (600, 2, 1, 8, 4), (3, 2, 0, 48, 0)])
def test_rope_axes(K, dtype, inverse, interleaved, tokens, heads, kv_heads, head_dim, pairs):
    g, dt = gen(20), R.DTYPES[dtype]
    q = randn(g, tokens, heads, head_dim, dtype=dt)
    k = randn(g, tokens, kv_heads, head_dim, dtype=dt) if kv_heads else None
    pos = torch.randint(0, 200000, (3, tokens), generator=g, device="cuda")
    freq = 1e6 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / max(pairs, 1))
    axis = (torch.arange(pairs, device="cuda") % 3).to(torch.uint8)
    got = rope(K, q, k, pos, freq, axis, interleaved, inverse)
    for x, y in zip((q, k), got):
        if x is not None:
            R.assert_within(y, R.rope(x, pos, freq, axis, interleaved, inverse), "rope")


def test_rope_axes_in_place_strided_and_unaligned(K):
    """One projection's rows turned in place: q's and k's heads turn, v's and the row's rest stay."""
    g, n, heads, kv, hd = gen(21), 77, 4, 2, 64
    for extra, shift in ((0, 0), (8, 0), (1, 0), (0, 3)):
        width = (heads + 2 * kv) * hd + extra
        rows = randn(g, n * width + shift, dtype=torch.bfloat16)[shift:].view(n, width)
        pos = torch.randint(0, 5000, (2, n), generator=g, device="cuda")
        freq = 1e4 ** (-torch.arange(32, device="cuda", dtype=torch.float64) / 32)
        axis = (torch.arange(32, device="cuda") >= 16).to(torch.uint8)
        before = rows.clone()
        q, k = (rows[:, a * hd:(a + c) * hd].unflatten(1, (c, hd)) for a, c in ((0, heads), (heads, kv)))
        want = [R.rope(x.clone(), pos, freq, axis, False, False) for x in (q, k)]
        rope(K, q, k, pos, freq, axis, False, False, q, k)
        R.assert_within(q, want[0], "q"), R.assert_within(k, want[1], "k")
        assert torch.equal(rows[:, (heads + kv) * hd:], before[:, (heads + kv) * hd:])


def test_rope_axes_far_positions_and_missing_axes(K):
    """Positions past 2^31 keep their angles; a pair whose axis is not there is copied."""
    g = gen(22)
    q = randn(g, 64, 2, 16)
    pos = torch.randint(2 ** 31, 2 ** 33, (1, 64), generator=g, device="cuda")
    freq = torch.tensor([1.0, 0.5, 0.1, 1e-3, 1e-5, 1e-9, 3.0, 2.0], dtype=torch.float64, device="cuda")
    axis = torch.zeros(8, dtype=torch.uint8, device="cuda")
    # the product position * frequency and the turns round to 2^-53 of 2^35: 2^-17 of a radian at most
    value, bound = R.rope(q, pos, freq, axis, False, False)
    R.assert_within(rope(K, q, None, pos, freq, axis, False, False)[0], (value, bound + 2.0 ** -16 * q.abs().amax()), "far")
    axis[2] = 1
    got = rope(K, q, None, pos, freq, axis, False, False)[0]
    assert torch.equal(got[..., 2], q[..., 2]) and torch.equal(got[..., 10], q[..., 10])


# ---- norms around the residual ----


def norm_inputs(seed, dt, rows, dim, placement, gate, unit_offset):
    g = gen(seed)
    centre = 0.0 if unit_offset else 1.0
    w = [centre + randn(g, dim, scale=0.2) if there else None for there in (placement != 0, placement != 1)]
    gates = None if gate == 0 else randn(g, dim) if gate == 1 else randn(g, rows, dim, dtype=dt)
    return randn(g, rows, dim, dtype=dt, scale=2.0), randn(g, rows, dim, dtype=dt), gates, *w, \
        randn(g, rows, dim, dtype=dt, scale=0.1), randn(g, rows, dim, dtype=dt, scale=0.1) if placement != 1 else None


def norm_shape(K, x, placement, gate, unit_offset, scale):
    return K.ResidualNorm(K.DTYPES[NAMES[x.dtype]], x.shape[0], x.shape[1], placement, gate, int(unit_offset), 1e-5, scale)


def norm_forward(K, shape, x, y, gate, post, pre, h=None):
    h = torch.empty_like(x) if h is None else h
    n = torch.empty_like(x) if shape.norm_placement != 1 else None
    K.check(K.lib.dllm_hip_residual_norm(shape, ptr(x), ptr(y), ptr(gate), ptr(post), ptr(pre), ptr(h), ptr(n), stream()))
    return h, n


def norm_backward(K, shape, h, y, gate, post, pre, dh, dn, dx=None, skip=()):
    got = dict(dx=torch.empty_like(h) if dx is None else dx, dy=torch.empty_like(y), dgate=gate, dpost_weight=post,
               dpre_weight=pre)
    for name in ("dgate", "dpost_weight", "dpre_weight"):
        got[name] = None if got[name] is None else torch.empty_like(got[name])
    got.update({name: None for name in skip})
    ws = torch.empty(K.lib.dllm_hip_residual_norm_backward_workspace(shape), dtype=torch.uint8, device="cuda")
    K.check(K.lib.dllm_hip_residual_norm_backward(shape, ptr(h), ptr(y), ptr(gate), ptr(post), ptr(pre), ptr(dh), ptr(dn),
                                                  *map(ptr, got.values()), ptr(ws), ws.numel(), stream()))
    return {n: t for n, t in got.items() if t is not None}


def check_norm(K, seed, dt, rows, dim, placement, gate, unit_offset, scale):
    x, y, gates, post, pre, dh, dn = norm_inputs(seed, dt, rows, dim, placement, gate, unit_offset)
    shape = norm_shape(K, x, placement, gate, unit_offset, scale)
    h, n = norm_forward(K, shape, x, y, gates, post, pre)
    want = R.residual_norm(x, y, gates, post, pre, placement, 1e-5, unit_offset, scale)
    R.assert_within(h, want["h"], "h")
    if n is not None:
        R.assert_within(n, want["n"], "n")
    got = norm_backward(K, shape, h, y, gates, post, pre, dh, dn)
    want = R.residual_norm(h, y, gates, post, pre, placement, 1e-5, unit_offset, scale, dh=dh, dn=dn)
    assert got.keys() == want.keys()
    for name in want:
        R.assert_within(got[name], want[name], name)


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("placement", [0, 1, 2])
@pytest.mark.parametrize("gate", [0, 1, 2])
def test_residual_norm_kinds(K, dtype, placement, gate):
    check_norm(K, 30, R.DTYPES[dtype], 67, 192, placement, gate, gate == 1, 0.22)


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("rows", "dim"), [(1, 1), (1, 8), (3, 17), (300, 64), (5, 576), (70, 896), (2, 1001), (1030, 2304),
                                           (9, 2048), (4, 4096), (2, 5000), (3, 8192), (2, 16384), (2, 16391), (1, 70000),
                                           (5000, 33), (2100, 128)])
def test_residual_norm_sizes(K, dtype, rows, dim):
    check_norm(K, 31, R.DTYPES[dtype], rows, dim, 2, 1, False, 1.0)


def test_residual_norm_rows_are_their_own(K):
    """The bits of a row do not depend on the rows beside it."""
    for dt in R.DTYPES.values():
        for dim in (576, 1001):
            x, y, gate, post, pre, dh, dn = norm_inputs(32, dt, 500, dim, 2, 2, False)
            h, n = norm_forward(K, norm_shape(K, x, 2, 2, False, 0.5), x, y, gate, post, pre)
            all_rows = norm_backward(K, norm_shape(K, x, 2, 2, False, 0.5), h, y, gate, post, pre, dh, dn)
            for a, b in ((0, 1), (17, 80)):
                part = [t[a:b].clone() for t in (x, y, gate, dh, dn)]
                shape = norm_shape(K, part[0], 2, 2, False, 0.5)
                h1, n1 = norm_forward(K, shape, part[0], part[1], part[2], post, pre)
                assert torch.equal(h1, h[a:b]) and torch.equal(n1, n[a:b])
                got = norm_backward(K, shape, h1, part[1], part[2], post, pre, part[3], part[4])
                for name in ("dx", "dy", "dgate"):
                    assert torch.equal(got[name], all_rows[name][a:b]), name


@pytest.mark.parametrize("dim", [576, 1001, 20000])
def test_residual_norm_in_place_and_without_outputs(K, dim):
    """h over x, dx over dh, and every output left out once: the others' bits stay."""
    x, y, gate, post, pre, dh, dn = norm_inputs(33, torch.bfloat16, 90, dim, 2, 1, True)
    shape = norm_shape(K, x, 2, 1, True, 0.5)
    h, n = norm_forward(K, shape, x, y, gate, post, pre)
    x2 = x.clone()
    h2, n2 = norm_forward(K, shape, x2, y, gate, post, pre, h=x2)
    assert torch.equal(h, h2) and torch.equal(n, n2)
    want = norm_backward(K, shape, h, y, gate, post, pre, dh, dn)
    over = dh.clone()
    got = norm_backward(K, shape, h, y, gate, post, pre, over, dn, dx=over)
    assert all(torch.equal(got[name], want[name]) for name in want)
    for name in want:
        got = norm_backward(K, shape, h, y, gate, post, pre, dh, dn, skip=(name,))
        assert name not in got and all(torch.equal(got[o], want[o]) for o in got)
    # no upstream gradient of h, and weights of ones
    got = norm_backward(K, shape, h, y, gate, None, None, None, dn)
    want = R.residual_norm(h, y, gate, None, None, 2, 1e-5, False, 0.5, dn=dn)
    for name in got:
        R.assert_within(got[name], want[name], name)


def test_residual_norm_unaligned_rows(K):
    """Starts that are not whole 16-byte chunks."""
    x, y, gate, post, pre, dh, dn = norm_inputs(34, torch.bfloat16, 60, 256, 2, 1, False)

    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    shape = norm_shape(K, x, 2, 1, False, 1.0)
    h, n = norm_forward(K, shape, moved(x), moved(y), moved(gate), moved(post), moved(pre), h=moved(x))
    want = R.residual_norm(x, y, gate, post, pre, 2, 1e-5, False, 1.0)
    R.assert_within(h, want["h"], "h"), R.assert_within(n, want["n"], "n")
    got = norm_backward(K, shape, moved(h), moved(y), moved(gate), moved(post), moved(pre), moved(dh), moved(dn))
    want = R.residual_norm(h, y, gate, post, pre, 2, 1e-5, False, 1.0, dh=dh, dn=dn)
    for name in want:
        R.assert_within(got[name], want[name], name)


def test_residual_norm_of_no_rows(K):
    """Sums over no rows are zero."""
    x, y, gate, post, pre, dh, dn = norm_inputs(35, torch.float32, 0, 70, 2, 1, False)
    got = norm_backward(K, norm_shape(K, x, 2, 1, False, 1.0), x, y, gate, post, pre, dh, dn)
    assert all(bool((got[name] == 0).all()) for name in ("dgate", "dpost_weight", "dpre_weight"))


# ---- together ----


class Layer:
    """The calls of one attention block of a packed multimodal batch: norm, rotation, attention, and the norms and residual
    after it, forward and backward, on one stream. The projections are torch products."""

    def __init__(self, K, seed, dt):
        g, self.K, self.dt = gen(seed), K, dt
        self.n, self.heads, self.kv, self.hd, self.dim = 330, 4, 2, 64, 192
        self.offsets, self.prefix = [0, 129, 130, 330], [40, 0, 64]
        self.x, self.y0 = randn(g, self.n, self.dim, dtype=dt), randn(g, self.n, self.dim, dtype=dt)
        self.gate, self.w = randn(g, self.dim, scale=0.5), [1 + randn(g, self.dim, scale=0.1) for _ in range(3)]
        self.proj = [randn(g, self.dim, h * self.hd, dtype=dt, scale=self.dim ** -0.5) for h in (self.heads, self.kv, self.kv)]
        self.proj.append(randn(g, self.heads * self.hd, self.dim, dtype=dt, scale=0.1))
        self.pos = torch.randint(0, 4000, (3, self.n), generator=g, device="cuda")
        self.freq = 1e4 ** (-torch.arange(32, device="cuda", dtype=torch.float64) / 32)
        self.axis = (torch.arange(32, device="cuda") % 3).to(torch.uint8)
        self.dh, self.dn = randn(g, self.n, self.dim, dtype=dt), randn(g, self.n, self.dim, dtype=dt)
        shape = lambda h: torch.zeros(self.n, h, self.hd, dtype=dt, device="cuda")  # noqa: E731
        self.attention = Attention(K, shape(self.heads), shape(self.kv), shape(self.kv), self.offsets,
                                   prefix=self.prefix, softcap=20.0)
        self.first = K.ResidualNorm(K.DTYPES[NAMES[dt]], self.n, self.dim, 0, 0, 0, 1e-5, 1.0)
        self.second = K.ResidualNorm(K.DTYPES[NAMES[dt]], self.n, self.dim, 2, 1, 0, 1e-5, 0.5)

    def step(self):
        K, a = self.K, self.attention
        h0, n0 = norm_forward(K, self.first, self.x, self.y0, None, None, self.w[0])
        q, k = ((n0 @ p).view(self.n, -1, self.hd) for p in self.proj[:2])
        rope(K, q, k, self.pos, self.freq, self.axis, False, False, a.q, a.k)
        torch.mm(n0, self.proj[2], out=a.v.view(self.n, -1))
        out, _ = a.forward()
        y1 = out.view(self.n, -1) @ self.proj[3]
        h1, n1 = norm_forward(K, self.second, h0, y1, self.gate, self.w[1], self.w[2])
        g1 = norm_backward(K, self.second, h1, y1, self.gate, self.w[1], self.w[2], self.dh, self.dn)
        dq, dk, dv = a.backward((g1["dy"] @ self.proj[3].T).view(self.n, self.heads, self.hd))
        dq, dk = rope(K, dq, dk, self.pos, self.freq, self.axis, False, True)
        dn0 = sum(d.reshape(self.n, -1) @ p.T for d, p in zip((dq, dk, dv), self.proj))
        g0 = norm_backward(K, self.first, h0, self.y0, None, None, self.w[0], g1["dx"], dn0)
        return dict(h1=h1, n1=n1, dx=g0["dx"], dw0=g0["dpre_weight"], dgate=g1["dgate"], dw1=g1["dpost_weight"],
                    dw2=g1["dpre_weight"])

    def reference(self):
        """The same block by torch's differentiation of its definition in 64 bits."""
        d = lambda t: t.detach().double().requires_grad_()  # noqa: E731
        x, gate, w = d(self.x), d(self.gate), [d(t) for t in self.w]
        rms = lambda v, s: v / torch.sqrt(v.square().mean(dim=1, keepdim=True) + 1e-5) * s  # noqa: E731
        h0 = x + self.y0.double()
        n0 = rms(h0, w[0])
        q, k, v = ((n0 @ p.double()).view(self.n, -1, self.hd) for p in self.proj[:3])
        angle = self.pos[self.axis.long()].double().T * self.freq

        def turn(t):
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            u, v = t[..., :32], t[..., 32:]
            return torch.cat([u * c - v * s, v * c + u * s], dim=-1)

        q, k = turn(q), turn(k)
        outs = []
        for i, (b, e) in enumerate(zip(self.offsets, self.offsets[1:])):
            mask = R.hidden(e - b, True, 0, self.prefix[i]).cuda()
            heads = []
            for h in range(self.heads):
                s = 20.0 * torch.tanh(q[b:e, h] @ k[b:e, h // 2].T / math.sqrt(self.hd) / 20.0)
                heads.append(torch.softmax(s.masked_fill(mask, -math.inf), dim=1) @ v[b:e, h // 2])
            outs.append(torch.cat(heads, dim=1))
        y1 = torch.cat(outs) @ self.proj[3].double()
        h1 = h0 + 0.5 * gate * rms(y1, w[1])
        n1 = rms(h1, w[2])
        grads = torch.autograd.grad([h1, n1], [x, w[0], gate, w[1], w[2]], [self.dh.double(), self.dn.double()])
        return dict(h1=h1, n1=n1, **dict(zip(("dx", "dw0", "dgate", "dw1", "dw2"), grads)))


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_a_layer(K, dtype):
    """The whole block against 64 bits. About ten results are rounded to the type on the way from x to a gradient, each
    off by at most u of itself; every step's condition here is a small factor (norms and softmax of unit-sized rows), so the
    2-norms are held to 100 u, and float32, whose longest sums have 330 terms, to 1000 F."""
    layer = Layer(K, 40, R.DTYPES[dtype])
    got, want = layer.step(), layer.reference()
    limit = max(100 * R.unit(layer.dt), 1000 * R.F) if dtype != "float32" else 1000 * R.F
    for name in want:
        off = float((got[name].double() - want[name].detach()).norm() / want[name].detach().norm())
        assert off < limit, (name, off)


def test_a_layer_on_another_stream_and_in_a_graph(K):
    """The same bits on a stream of its own and from a captured graph, replayed with other work between."""
    layer = Layer(K, 41, torch.bfloat16)
    want = {n: t.clone() for n, t in layer.step().items()}
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer.step()
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer.step()
    for _ in range(4):
        for t in held.values():
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(held[n], want[n]) for n in want)
        assert all(torch.equal(t, want[n]) for n, t in layer.step().items())
        torch.cuda.synchronize()


def test_two_calls_at_once(K):
    """Two streams, a workspace each."""
    a, da = problem(K, 50, torch.bfloat16, [0, 600, 1000], 1000, 4, 2, 64)
    b, db = problem(K, 51, torch.bfloat16, [0, 333, 900], 1000, 4, 2, 64, softcap=9.0)
    want = [[t.clone() for t in (*p.forward(), *p.backward(d))] for p, d in ((a, da), (b, db))]
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for p, d, s in ((a, da, one), (b, db, two)):
        with torch.cuda.stream(s):
            got.append([*p.forward(), *p.backward(d)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))


# ---- the array functions ----


def bits(t: torch.Tensor) -> np.ndarray:
    t = t.cpu()
    return t.view(torch.uint16).numpy() if t.dtype == torch.bfloat16 else t.numpy()


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_array_functions(K, dtype):
    """The NumPy functions give the device calls' bits; bfloat16 as its 16 bits."""
    dt = R.DTYPES[dtype]
    o = dict(window=9, prefix=[3, 0], softcap=4.0, slopes=[0.1, 0.2])
    p, dout = problem(K, 60, dt, [0, 30, 41], 41, 2, 1, 24, **o)
    out, lse = p.forward()
    got = K.document_attention(bits(p.q), bits(p.k), bits(p.v), [0, 30, 41], p.scale, **o)
    assert np.array_equal(got[0], bits(out)) and np.array_equal(got[1], bits(lse))
    grads = K.document_attention_backward(bits(p.q), bits(p.k), bits(p.v), [0, 30, 41], got[0], got[1], bits(dout), p.scale, **o)
    assert all(np.array_equal(a, bits(b)) for a, b in zip(grads, p.backward(dout)))
    g = gen(61)
    pos = torch.randint(0, 99, (2, 41), generator=g, device="cuda")
    freq, axis = torch.tensor([1.0, 0.3, 0.2], dtype=torch.float64, device="cuda"), torch.tensor([0, 1, 0], dtype=torch.uint8, device="cuda")
    a = K.rope_axes(bits(p.q), bits(p.k), pos.cpu().numpy(), freq.cpu().numpy(), axis.cpu().numpy(), True)
    b = rope(K, p.q, p.k, pos, freq, axis, True, False)
    assert np.array_equal(a[0], bits(b[0])) and np.array_equal(a[1], bits(b[1]))
    x, y, gate, post, pre, dh, dn = norm_inputs(62, dt, 20, 40, 2, 2, False)
    h, n = norm_forward(K, norm_shape(K, x, 2, 2, False, 0.5), x, y, gate, post, pre)
    f = lambda t: t.cpu().numpy()  # noqa: E731
    keys = dict(gate=bits(gate), post_weight=f(post), pre_weight=f(pre), norm_placement=2, eps=1e-5, residual_scale=0.5)
    a = K.residual_norm(bits(x), bits(y), **keys)
    assert np.array_equal(a[0], bits(h)) and np.array_equal(a[1], bits(n))
    got = K.residual_norm_backward(a[0], bits(y), bits(dh), bits(dn), **keys)
    want = norm_backward(K, norm_shape(K, x, 2, 2, False, 0.5), h, y, gate, post, pre, dh, dn)
    assert all(np.array_equal(u, bits(v)) for u, v in zip(got, want.values()))
