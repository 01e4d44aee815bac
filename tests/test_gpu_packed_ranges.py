"""GPU: the packed-layer operators at the ends of their ranges: rows of norms far from one, caps of any size and scores that
reach them, upstream gradients of very different sizes, rows that see few keys, many documents, outputs in wider rows. The
bounds are those of packed_reference or, where its are as wide as what is looked for, tighter ones of the same kind (u = eps / 2
of the activations' type, F = 2^-24)."""

from __future__ import annotations

import math

import pytest
import torch

import packed_reference as R
from packed_reference import F
from test_gpu_packed_layers import (PACK, Attention, K, Layer, gen, norm_backward, norm_forward, problem,  # noqa: F401  (K: the fixture)
                                    randn)

pytestmark = pytest.mark.gpu


# ---- attention ----


def tight(p, out=None, lse=None, dout=None, few=0):
    """Results and bounds of a problem of one document, forward, or with dout backward. As packed_reference.attention, but
    - tanh is off by a few F of its value however large the cap is (16-bit types up to a cap of 64: a few F of the cap);
    - rows that see at most `few` keys (keys that as few queries see) have their 16-bit weights and dS multiplied with what
      rounding left of them, as far as all 32 rows of their wave do;
    - float16's p and dS are rounded as multiples of the smallest float16 relative to what the row's (the key's) own largest
      visible value is: p to 2^-25 forward and 2^-40 backward, dS to 2^-34 of the largest (2^-33 for its own roundings)."""
    q, k, v, o = p.q.double(), p.k.double(), p.v.double(), p.options
    dt, n, heads, hd = p.q.dtype, *p.q.shape
    u, group, cap, half = R.unit(dt), heads // p.k.shape[1], o["softcap"], dt == torch.float16
    seen = ~R.hidden(n, o["causal"], o["window"], 0 if o["prefix"] is None else o["prefix"][0]).cuda()

    def rounding(counts):  # of 16-bit weights, by how many the rows of a wave have
        if dt == torch.float32:
            return torch.zeros(n, dtype=torch.float64, device="cuda")
        waves = torch.nn.functional.pad(counts, (0, -n % 32)).view(-1, 32).amax(dim=1).repeat_interleave(32)[:n]
        return torch.where(waves <= few, 2 * u * u, u).double()

    by_row, by_key = rounding(seen.sum(dim=1))[:, None], rounding(seen.sum(dim=0))[None, :]
    i = torch.arange(n, device="cuda")
    distance = (i[:, None] - i[None, :]).abs().double()
    got = {name: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for name, t in
           (("out", q), ("lse", p.lse), ("dq", q), ("dk", k), ("dv", v))}
    off = {name: torch.zeros_like(t) for name, t in got.items()}
    for h in range(heads):
        Q, Kh, V = q[:, h], k[:, h // group], v[:, h // group]
        x = Q @ Kh.T * p.scale
        err = (hd + 4) * F * (Q.abs() @ Kh.abs().T) * p.scale
        slope = torch.ones_like(x)
        if cap:
            t = torch.tanh(x / cap)
            x, slope = cap * t, 1 - t * t
            err = err + 8 * F * (cap if dt != torch.float32 and cap <= 64 else x.abs())
        if o["slopes"] is not None:
            x = x - float(o["slopes"][h]) * distance
            err = err + 4 * F * float(o["slopes"][h]) * distance
        err = (err + 4 * F * x.abs()).masked_fill(~seen, 0.0).amax(dim=1, keepdim=True)
        x = x.masked_fill(~seen, -math.inf)
        if dout is None:
            s = torch.logsumexp(x, dim=1, keepdim=True)
            w = torch.exp(x - s)
            got["lse"][h], off["lse"][h] = s[:, 0], (err + 4 * F * s.abs() + (n + 8) * F)[:, 0]
            got["out"][:, h] = r = w @ V
            off["out"][:, h] = u * r.abs() + (w @ V.abs()) * (2 * err.expm1() + 2 * by_row + (2 * n + 16) * F) * (1 + u) + \
                seen.double() @ V.abs() * (2.0 ** -25 if half else 2.0 ** -126)
            continue
        s = lse[h].double()[:, None]
        w = torch.exp(x - s)
        rel = err.expm1() + 4 * F * s.abs() + 8 * F
        dO, O = dout[:, h].double(), out[:, h].double()
        dP, delta = dO @ V.T, (dO * O).sum(dim=1, keepdim=True)
        size = dO.abs() @ V.abs().T + (dO.abs() * O.abs()).sum(dim=1, keepdim=True)
        dS = w * (dP - delta) * slope * p.scale
        dslope = 2 * (8 * F + err / cap) if cap else 0.0
        eS = w * size * p.scale * (rel + (hd + 16) * F + dslope) + seen * 2.0 ** -126 * (1 + size * p.scale)
        eP = w * (rel + by_key) + seen * (2.0 ** -40 if half else 2.0 ** -126)
        both = [eS + dS.abs() * by for by in (by_row, by_key)]  # dq's and dk's
        if half:
            both = [e + seen * 2.0 ** -33 * (dS.abs() + eS).amax(dim=d, keepdim=True) for e, d in zip(both, (1, 0))]
        got["dq"][:, h] = dS @ Kh
        off["dq"][:, h] = u * got["dq"][:, h].abs() + (both[0] @ Kh.abs() + (2 * n + 8) * F * (dS.abs() @ Kh.abs())) * (1 + u)
        for name, value, e, rows in (("dk", dS, both[1], Q), ("dv", w, eP, dO)):
            got[name][:, h // group] += value.T @ rows
            off[name][:, h // group] += (e.T @ rows.abs() + (2 * n + 8 + heads) * F * (value.abs().T @ rows.abs())) * (1 + u)
    for name in ("dk", "dv"):
        off[name] += u * got[name].abs()
    return {name: (got[name], off[name] + (0.0 if name == "lse" else R.tiny(dt))) for name in got}


def check(p, dout, what="", few=0):
    out, lse = p.forward()
    want = tight(p, few=few)
    R.assert_within(out, want["out"], f"{what} out"), R.assert_within(lse, want["lse"], f"{what} lse")
    want = tight(p, out, lse, dout, few)
    for name, got in zip(("dq", "dk", "dv"), p.backward(dout)):
        R.assert_within(got, want[name], f"{what} {name}")


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("cap", [64.0, 100.0, 1e3, 1e5, 1e8, 1e19])
def test_caps_of_any_size(K, dtype, head_dim, cap):  # noqa: F811
    """A cap far above the scores hardly bends them, and costs them no bits; scores above it are bent flat."""
    g, dt = gen(71), R.DTYPES[dtype]
    q, k, v, dout = (randn(g, 150, h, head_dim, dtype=dt) for h in (2, 1, 1, 2))
    check(Attention(K, q, k, v, [0, 150], softcap=cap), dout, "ordinary scores")
    if cap <= 1e5:
        check(Attention(K, q, k, v, [0, 150], softcap=cap, scale=cap / 8), dout, "scores about the cap's size")
    check(Attention(K, q, k, v, [0, 150], softcap=cap, causal=False, slopes=[0.1, 0.0]), dout, "bias")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("cap", [1.0, 30.0, 100.0])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_gradients_of_scores_near_the_cap(K, dtype, head_dim, cap, sign):  # noqa: F811
    """Scores of 3 to 9 times the cap are bent almost flat: their small derivatives, 1e-2 to 1e-7, are right to the type."""
    g, dt, n = gen(79), R.DTYPES[dtype], 100
    q, k = ((0.75 + 0.5 * torch.rand(n, h, head_dim, generator=g, device="cuda")).to(dt) for h in (2, 1))
    q, v, dout = q * sign, randn(g, n, 1, head_dim, dtype=dt), randn(g, n, 2, head_dim, dtype=dt)
    # of the scores' sizes: q.k is head_dim times 0.6 to 1.5
    p = Attention(K, q, k, v, [0, n], softcap=cap, scale=6 * cap / head_dim)
    if dtype == "float16":
        dout = dout * 1000  # (results of 1e-6 would be subnormal)
    out, lse = p.forward()
    dq, dk, _ = p.backward(dout)
    seen = ~R.hidden(n, True, 0, 0).cuda()
    u, bounds = R.unit(dt), dict(dk=[0.0, 0.0])
    for h in range(2):
        Q, Kh, V, dO, O = (t.double() for t in (q[:, h], k[:, 0], v[:, 0], dout[:, h], out[:, h]))
        z = Q @ Kh.T * (p.scale / cap)
        ez = (head_dim + 8) * F * z.abs()  # (every term has one sign)
        assert float(z[seen].abs().min()) > 2.5 and float(z[seen].abs().max()) < 9.5
        t = torch.tanh(z)
        slope = torch.cosh(z) ** -2
        # e^2z's relative error is 2 ez and its own roundings': so are those of 1 - tanh and of the derivative
        eslope = slope * (2 * ez + 8 * F * (1 + z.abs()))
        w = torch.exp(cap * t - lse[h].double()[:, None]).masked_fill(~seen, 0.0)
        ew = w * (cap * (slope * ez + 8 * F) + 4 * F * (1 + cap) + 8 * F)
        dP, delta = dO @ V.T, (dO * O).sum(dim=1, keepdim=True)
        size = dO.abs() @ V.abs().T + (dO.abs() * O.abs()).sum(dim=1, keepdim=True)
        dS = w * (dP - delta) * slope * p.scale
        eS = p.scale * (size * (w * eslope + ew * slope + w * slope * (head_dim + 16) * F)) + dS.abs() * u
        grown = [2.0 ** -33 * (dS.abs() + eS).amax(dim=d, keepdim=True) * seen * (dtype == "float16") for d in (1, 0)]
        value = dS @ Kh
        bound = u * value.abs() + ((eS + grown[0]) @ Kh + 2 * n * F * (dS.abs() @ Kh)) * (1 + u) + R.tiny(dt)
        R.assert_within(dq[:, h], (value, bound), f"dq {h}")
        bounds["dk"][0] += dS.T @ Q
        bounds["dk"][1] += ((eS + grown[1]).T @ Q.abs() + (2 * n + 10) * F * (dS.abs().T @ Q)) * (1 + u)
    value, bound = bounds["dk"]
    R.assert_within(dk[:, 0], (value, bound + u * value.abs() + R.tiny(dt)), "dk")


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("head_dim", [64, 100, 128, 256])
def test_documents_with_a_large_cap(K, dtype, head_dim):  # noqa: F811
    """Masks, hidden NaN and a document's own bits where large caps have kernels of their own."""
    options = dict(window=65, softcap=1e3, slopes=[1.0, 0.01, 0.0, 0.3])
    prefix = [1, 0, 3, 64, 100, 1, 0]
    p, dout = problem(K, 74, R.DTYPES[dtype], PACK, 437, 4, 2, head_dim, prefix=prefix, **options)
    p.check(dout)
    want = [t.clone() for t in (*p.forward(), *p.backward(dout))]
    for d in (3, 6):
        b, e = PACK[d], PACK[d + 1]
        s = Attention(K, p.q[b:e].clone(), p.k[b:e].clone(), p.v[b:e].clone(), [0, e - b], prefix=[prefix[d]], **options)
        got = [*s.forward(), *s.backward(dout[b:e].clone())]
        assert all(torch.equal(x, (y[:, b:e] if y is want[1] else y[b:e])) for x, y in zip(got, want))
    # the last document's first key is seen by its first 65 queries alone
    b, n = PACK[6], PACK[7] - PACK[6]
    p.k[b], p.v[b] = float("nan"), float("nan")
    out, _ = p.forward()
    sees = torch.zeros(437, dtype=torch.bool, device="cuda")
    sees[b:b + 65] = True
    assert bool(torch.isnan(out[sees]).all()) and n > 65
    assert torch.equal(out[:b], want[0][:b]) and torch.equal(out[b + 128:], want[0][b + 128:])
    clean = R.attention(p.q, torch.nan_to_num(p.k), torch.nan_to_num(p.v), p.offsets, p.scale, prefix=prefix, **options)["out"]
    R.assert_within(out[~sees], (clean[0][~sees], clean[1][~sees]), "beside NaN")


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("options", [dict(), dict(window=20), dict(causal=False, window=90), dict(prefix=[100])])
def test_float16_gradients_beside_a_large_one(K, head_dim, options):  # noqa: F811
    """One query whose upstream gradient is 10^6 to 10^7 times the others': the keys that it does not see keep their bits."""
    g = gen(72)
    q, k, v, dout = (randn(g, 256, h, head_dim) for h in (2, 1, 1, 2))
    for row in (0, 140):
        d = dout * 1e-3
        d[row] = dout[row] * 1e4
        check(Attention(K, q.half(), k.half(), v.half(), [0, 256], **options), d.half(), f"{row}")


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize(("size", "spread"), [(1e-3, 1.0), (1e-3, 4.0), (1.0, 4.0), (1e3, 1.0)])
def test_float16_gradients_of_small_and_large_values(K, head_dim, size, spread):  # noqa: F811
    """Values far below and above one, and weights from one down to e^-60: dS has the size of both, and keeps its bits."""
    g = gen(73)
    q, k, v, dout = (randn(g, 1500, h, head_dim, scale=s).half() for h, s in ((2, spread), (1, spread), (1, size), (2, 1.0)))
    check(Attention(K, q, k, v, [0, 1500]), dout)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("options", [dict(), dict(window=50), dict(causal=False, window=32), dict(prefix=[40]),
                                     dict(window=20, prefix=[44]), dict(window=64, softcap=10.0)])
def test_rows_that_see_few_keys(K, dtype, head_dim, options):  # noqa: F811
    """Where a wave's rows see at most 64 keys (its keys at most as many queries) the weights' rounding to 16 bits does not reach
    the results, in a long document as in a short one."""
    g, dt = gen(75), R.DTYPES[dtype]
    for n in (320, 333):
        q, k, v, dout = (randn(g, n, h, head_dim, dtype=dt) for h in (2, 1, 1, 2))
        p = Attention(K, q, k, v, [0, n], **options)
        seen = ~R.hidden(n, p.options["causal"], p.options["window"], (p.options["prefix"] or [0])[0])
        assert bool((seen.sum(dim=1)[:32] <= 64).all()) or bool((seen.sum(dim=0)[288:320] <= 64).all())
        check(p, dout, f"{n}", few=64)


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize(("extra", "shift"), [(8, 0), (16, 8), (3, 0), (0, 1)])
def test_attention_into_wider_rows(K, dtype, head_dim, extra, shift):  # noqa: F811
    """out and dout as parts of wider rows, whole 16-byte chunks or not: the bits of packed ones (in 16 bits a copy of the
    inputs takes the place of the inputs; the products are the same), and what lies between is left as it was. Infinities too,
    whose rows are computed and written another way."""
    n, heads = 150, 4
    p, dout = problem(K, 76, R.DTYPES[dtype], [3, 90, 150], n, heads, 2, head_dim, window=40, prefix=[0, 9])
    p.k[20], p.v[20], dout[130] = float("inf"), float("inf"), float("inf")
    width = heads * head_dim + extra

    def wide(t):
        flat = torch.full((n * width + shift,), 5.0, dtype=t.dtype, device="cuda")
        part = flat[shift:].view(n, width)[:, :heads * head_dim].unflatten(1, (heads, head_dim))
        part.copy_(t)
        return flat, part

    want = [t.clone() for t in (*p.forward(), *p.backward(dout))]
    flat, out = wide(torch.full_like(p.out, 5.0))
    _, upstream = wide(dout)
    p.out = out
    p.lse.zero_()
    p.shape.out_stride = width
    got = [*p.forward(), *p.backward(upstream)]
    rows = slice(3, 150)
    assert torch.equal(got[0][rows].nan_to_num(), want[0][rows].nan_to_num()) and bool((got[0][:3] == 5.0).all())
    assert torch.equal(got[1].nan_to_num(), want[1].nan_to_num())
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(got[2:], want[2:]))
    assert bool(torch.isnan(got[0][20:60]).any()) and bool(torch.isfinite(got[0][3:20]).all())
    assert bool((flat[shift:].view(n, width)[:, heads * head_dim:] == 5.0).all()) and bool((flat[:shift] == 5.0).all())


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("options", [dict(), dict(causal=False, window=70)])
@pytest.mark.parametrize("repeats", [2, 3, 500])
def test_many_documents_repeat_a_few(K, dtype, options, repeats):  # noqa: F811
    """A pack of 40 documents, empty ones and ends of tiles among them, over and over: each time the bits of the one pack, whose
    documents a wave finds another way; prefixes of their own, and tokens of none before and after."""
    lengths = [0, 1, 2, 127, 128, 129, 0, 0, 64, 65, 200, 1, 63, 3, 17, 256] + [(7 * i) % 23 for i in range(24)]
    prefix = [(5 * i) % 40 for i in range(40)]
    n = sum(lengths)
    offsets = [0]
    for length in lengths:
        offsets.append(offsets[-1] + length)
    one, dout = problem(K, 78, R.DTYPES[dtype], offsets, n, 2, 1, 64, prefix=prefix, **options)
    want = [t.clone() for t in (*one.forward(), *one.backward(dout))]

    def tiled(t):  # 5 tokens of no document, the pack again and again, 9 more
        return torch.cat([t[:5], *[t] * repeats, t[:9]])

    ends = [5 + r * n + o for r in range(repeats) for o in offsets[:-1]] + [5 + repeats * n]
    p = Attention(K, tiled(one.q), tiled(one.k), tiled(one.v), ends, prefix=prefix * repeats, **options)
    got = [*p.forward(), *p.backward(tiled(dout))]
    got[1], want[1] = got[1].T, want[1].T
    for x, y in zip(got, want):
        inside = x[5:5 + repeats * n].reshape(repeats, *y.shape)
        assert torch.equal(inside, y.expand(repeats, *y.shape))
        assert bool((x[:5] == 0).all()) and bool((x[5 + repeats * n:] == 0).all())


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


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_norm_gradients_of_wide_rows_in_a_graph(K, dtype):  # noqa: F811
    """Rows whose parameters take more LDS than a kernel has without asking, captured at the kernel's first call."""
    g, dt, rows, dim = gen(77), R.DTYPES[dtype], 300, 8192
    x, y, dh, dn = (randn(g, rows, dim, dtype=dt) for _ in range(4))
    post, pre = (1 + randn(g, dim, scale=0.2) for _ in range(2))
    shape = K.ResidualNorm(K.DTYPES[dtype], rows, dim, 2, 0, 0, 1e-5, 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = norm_backward(K, shape, x, y, None, post, pre, dh, dn)
    want = R.residual_norm(x, y, None, post, pre, 2, 1e-5, False, 0.5, dh=dh, dn=dn)
    eager = norm_backward(K, shape, x, y, None, post, pre, dh, dn)
    for _ in range(3):
        for t in held.values():
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for name in want:
            R.assert_within(held[name], want[name], name)
            assert torch.equal(held[name], eager[name])


# ---- together ----


class Rounded(torch.autograd.Function):
    """A value, and the gradient that comes back to it, rounded to a type as a kernel's result is."""

    @staticmethod
    def forward(ctx, x, dt):
        ctx.dt = dt
        return x.to(dt).double()

    @staticmethod
    def backward(ctx, g):
        return g.to(ctx.dt).double(), None


def layer(l, dt):
    """Layer.step in 64 bits, with each result that the step leaves in its type rounded to it (dt None: with none rounded)."""
    n, hd = l.n, l.hd
    r = (lambda t: Rounded.apply(t, dt)) if dt is not None else (lambda t: t)
    d = lambda t: t.detach().double().requires_grad_()  # noqa: E731
    x, gate, w = d(l.x), d(l.gate), [d(t) for t in l.w]
    rms = lambda v, s: v / torch.sqrt(v.square().mean(dim=1, keepdim=True) + 1e-5) * s  # noqa: E731
    exact_h0 = x + l.y0.double()
    h0, n0 = r(exact_h0), r(rms(exact_h0, w[0]))
    q, k, v = (r((n0 @ p.double()).view(n, -1, hd)) for p in l.proj[:3])
    angle = l.pos[l.axis.long()].double().T * l.freq
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    q, k = (r(torch.cat([t[..., :32] * c - t[..., 32:] * s, t[..., 32:] * c + t[..., :32] * s], dim=-1)) for t in (q, k))
    outs = []
    for i, (b, e) in enumerate(zip(l.offsets, l.offsets[1:])):
        mask = R.hidden(e - b, True, 0, l.prefix[i]).cuda()
        heads = []
        for h in range(l.heads):
            z = 20.0 * torch.tanh(q[b:e, h] @ k[b:e, h // 2].T / math.sqrt(hd) / 20.0)
            heads.append(r(torch.softmax(z.masked_fill(mask, -math.inf), dim=1)) @ v[b:e, h // 2])
        outs.append(torch.cat(heads, dim=1))
    y1 = r(r(torch.cat(outs)) @ l.proj[3].double())
    exact_h1 = h0 + 0.5 * gate * rms(y1, w[1])
    h1, n1 = r(exact_h1), r(rms(exact_h1, w[2]))
    grads = torch.autograd.grad([h1, n1], [x, w[0], gate, w[1], w[2]], [l.dh.double(), l.dn.double()])
    return dict(h1=h1.detach(), n1=n1.detach(), **dict(zip(("dx", "dw0", "dgate", "dw1", "dw2"), grads)))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_a_layer_is_off_by_its_roundings(K, dtype):  # noqa: F811
    """A block of all three operators is off by as much as the same block in 64 bits with its results rounded at the same places:
    two draws of the same roundings, whose 2-norms over some hundred to some ten thousand values differ by less than a half of
    themselves. (dS, which the kernels round too, and the rounded h that the norms' gradients read, are one rounding each beside
    the dozen on the way: the factor of 2 has room for them.)"""
    l = Layer(K, 42, R.DTYPES[dtype])
    got, exact, rounded = l.step(), layer(l, None), layer(l, l.dt)
    for name in exact:
        off, draw = (float((t[name].double() - exact[name]).norm() / exact[name].norm()) for t in (got, rounded))
        assert 0 < off <= 2 * draw, (name, off, draw)
