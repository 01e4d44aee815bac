"""GPU: what the operators at a packed step's ends keep of their values' bits beside rows and matrices of other sizes, through the
C ABI on device tensors, against their 64-bit definitions."""

from __future__ import annotations

import math

import pytest
import torch

import ends_reference as R
from test_gpu_step_ends import (  # noqa: F401
    K, Loss, Step, embed_backward, gen, loss_problem, momentum, moved, ptr, randn, some_tokens, stream, update)

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


def test_float32_gradients_of_unlikely_tokens(K):  # noqa: F811
    """Probabilities from one half to 1e-13 in dweight's rows: off by 2^-39 as float16 pairs, and by what the logits' sums of 64 terms, 80 F of
    at most 30, make of them."""
    g = gen(76)
    likely = torch.linspace(0.0, -30.0, 400, device="cuda")
    weight = torch.zeros(400, 64, device="cuda")
    weight[:, 0] = likely
    hidden = randn(g, 100, 64)
    hidden[:, 0] = 1.0
    targets = torch.zeros(100, dtype=torch.int64, device="cuda")
    p = Loss(K, hidden, weight, targets)
    dloss = torch.full((100,), 0.01, device="cuda")
    p.check(dloss)
    value = R.loss_backward(hidden, weight, targets, p.lse, dloss)["dweight"][0][1:, 0]  # of hidden states of one
    off = (p.backward(dloss)[1][1:, 0].double() / value - 1).abs()
    assert float(value.max()) > 0.05 and float(value.min()) < 1e-13
    assert bool((off <= 1.01 * 2.0 ** -39 / value + 80 * R.F * 30 + 1e-5).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("softcap", [0.0, 4.0])
@pytest.mark.parametrize(("rows", "vocabulary", "dim"), [(1, 5000, 96), (2, 300, 33), (37, 5000, 200), (64, 20001, 72)])
def test_gradients_of_few_rows_for_tokens_that_are_no_target(K, dtype, softcap, rows, vocabulary, dim):  # noqa: F811
    """dweight's rows that the softmax alone reaches are off by their own rounding, as from products in float32: what a pair leaves of
    an operand is 2^-16 (bfloat16) or 2^-22 of it, and the factor below is for that and float32's sums."""
    g, dt = gen(75), R.DTYPES[dtype]
    weight, hidden = randn(g, vocabulary, dim, dtype=dt, scale=dim ** -0.5), randn(g, rows, dim, dtype=dt)
    targets = torch.randint(0, vocabulary, (rows,), generator=g, device="cuda")
    dloss = torch.exp2(4.0 * torch.rand(rows, generator=g, device="cuda")) * 100.0
    if rows > 2:
        targets[1] = -1
    p = Loss(K, hidden, weight, targets, softcap=softcap)
    _, lse = p.forward()
    counts = targets >= 0
    got = p.backward(dloss, want=(False, True))[1]
    value = R.loss_backward(hidden, weight, targets, lse, dloss, softcap=softcap)["dweight"][0]
    z = hidden.float() @ weight.float().T
    slope = torch.ones_like(z)
    if softcap:
        z = softcap * torch.tanh(z / softcap)
        slope = 1.0 - (z / softcap).square()
    plain = ((torch.exp(z - lse[:, None]) * slope * (dloss * counts)[:, None]).T @ hidden.float()).to(dt)
    others = torch.ones(vocabulary, dtype=torch.bool, device="cuda")
    others[targets[counts]] = False
    off, of_plain = (float(torch.linalg.norm((t.double() - value)[others])) for t in (got, plain))
    assert off <= 1.02 * of_plain, off / of_plain
    assert torch.equal(p.backward(dloss)[1], got)


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("rows", "dim"), [(64, 8), (33, 5)])
def test_gradients_of_few_rows_in_pieces(K, dtype, rows, dim):  # noqa: F811
    """So large a vocabulary that few rows go over it in pieces, added to what dweight holds; rows that do not count, and one alone; dweight
    that is not aligned."""
    p, dloss = loss_problem(K, 78, R.DTYPES[dtype], rows, 2200000, dim, masked=0.2)
    old = randn(gen(79), 2200000, dim, dtype=R.DTYPES[dtype], scale=1e-3)
    p.check(dloss, old)
    dhidden, dweight = (t.clone() for t in p.backward(dloss, old))
    q = Loss(K, p.hidden[9:10].clone(), p.weight, p.targets[9:10].clone())
    q.lse.copy_(p.lse[9:10])
    assert torch.equal(q.backward(dloss[9:10].clone())[0], dhidden[9:10])
    p.shape.accumulate = 1
    into = moved(old)
    K.check(K.lib.dllm_hip_vocabulary_loss_backward(p.shape, *map(ptr, (p.hidden, p.weight, p.targets, p.lse, dloss)), None, ptr(into), ptr(p.workspace),
                                                    p.workspace.numel(), stream()))
    assert torch.equal(into, dweight)


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("dtype", R.DTYPES)
def test_loss_of_infinities(K, dtype, rows, value):  # noqa: F811
    """An infinite weight: rows that it gives a logit of minus infinity have their loss without it, others none, and in float32's
    pairs no row has one. An infinite hidden state is its row's own."""
    g, dt = gen(77), R.DTYPES[dtype]
    weight, hidden = randn(g, 500, 40, dtype=dt), randn(g, rows, 40, dtype=dt)
    targets = torch.randint(0, 77, (rows,), generator=g, device="cuda")
    dloss = torch.full((rows,), 0.1, device="cuda")
    weight[400, 7] = value
    p = Loss(K, hidden, weight, targets)
    loss, lse = p.forward()
    pairs = dtype == "float32" and rows > 256
    gone = (hidden[:, 7].float() * value < 0) & (not pairs)
    assert not bool(torch.isfinite(loss[~gone]).any()) and not bool(torch.isfinite(lse[~gone]).any())
    want = R.loss(hidden[gone], torch.cat([weight[:400], weight[401:]]), targets[gone])
    R.assert_within(loss[gone], want["loss"], "loss")
    R.assert_within(lse[gone], want["lse"], "lse")
    weight[400], hidden[3, 5] = 0.25, value
    p = Loss(K, hidden, weight, targets)
    got = [t.clone() for t in p.forward()]
    dhidden = p.backward(dloss)[0]
    others = torch.arange(rows, device="cuda") != 3
    assert not bool(torch.isfinite(got[0][3])) and bool(dhidden[3].isnan().all())
    assert bool(torch.isfinite(got[0][others]).all()) and bool(torch.isfinite(dhidden[others]).all())


# ---- the table's gradient ----


def in_groups(ids, dout, vocabulary, scale):
    """The sums in the order that is promised, in float32: each token's positions 8 at a time, then those sums."""
    total = torch.zeros(vocabulary, dout.shape[1])
    order = torch.argsort(ids, stable=True)
    tokens, counts = torch.unique_consecutive(ids[order], return_counts=True)
    for token, rows in zip(tokens.tolist(), order.split(counts.tolist())):
        if not 0 <= token < vocabulary:
            continue
        parts = []
        for some in rows.split(8):
            acc = dout[some[0]].float()
            for i in some[1:]:
                acc = acc + dout[i].float()
            parts.append(acc)
        acc = parts[0]
        for part in parts[1:]:
            acc = acc + part
        total[token] = acc * scale
    return total


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("tokens", "vocabulary", "dim"), [(7, 3, 8), (9, 1, 4), (100, 9, 16), (1000, 70, 24), (3000, 40, 3), (16384, 3000, 8), (16385, 5, 8),
                                                           (30000, 20000, 4)])
def test_embedding_gradient_adds_in_its_order(K, dtype, tokens, vocabulary, dim):  # noqa: F811
    g, dt = gen(80), R.DTYPES[dtype]
    ids = some_tokens(g, tokens, vocabulary)
    dout = randn(g, tokens, dim, dtype=dt)
    want = in_groups(ids.cpu(), dout.cpu(), vocabulary, 0.5).to(dt)  # (a power of two: no rounding of its own)
    assert torch.equal(embed_backward(K, ids, dout, vocabulary, 0.5).cpu(), want)


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_embedding_gradient_of_a_token_in_other_company(K, dtype):  # noqa: F811
    """A token's row has the same bits whatever other tokens a batch has."""
    g, dt = gen(81), R.DTYPES[dtype]
    counts = [1, 2, 7, 8, 9, 15, 16, 17, 24, 63, 65, 200, 1000, 6000]
    ids = torch.cat([torch.full((c,), 3 * i + 40, device="cuda") for i, c in enumerate(counts)])
    ids = ids[torch.randperm(len(ids), generator=g, device="cuda")]
    dout = randn(g, len(ids), 40, dtype=dt)
    alone = embed_backward(K, ids, dout, 100)
    seen = torch.unique(ids)
    for others in (1, 3, 500, 9000, 40000):
        more = torch.randint(0, 40, (others,), generator=g, device="cuda")
        if others > 500:  # between them too
            more = torch.where(torch.rand(others, generator=g, device="cuda") < 0.5, more, 41 + 3 * (more % 14))
        keep = torch.rand(len(ids) + others, generator=g, device="cuda").argsort()[:len(ids)].sort().values
        mixed, rows = torch.empty(len(ids) + others, dtype=torch.int64, device="cuda"), randn(g, len(ids) + others, 40, dtype=dt)
        rest = torch.ones(len(mixed), dtype=torch.bool, device="cuda")
        rest[keep] = False
        mixed[keep], mixed[rest], rows[keep] = ids, more, dout
        assert torch.equal(embed_backward(K, mixed, rows, 100)[seen], alone[seen]), others


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_loss_gradients_whose_parts_would_be_many(K, dtype):  # noqa: F811
    """Few tiles of dhidden, and so much of it that they take the vocabulary's units in turn; the same bits as in parts."""
    g, dt = gen(74), R.DTYPES[dtype]
    weight = randn(g, 12287, 2900, dtype=dt, scale=2.0 / math.sqrt(2900))
    hidden = randn(g, 1600, 2900, dtype=dt)
    targets = torch.randint(0, 12287, (1600,), generator=g, device="cuda")
    dloss = torch.rand(1600, generator=g, device="cuda") / 1600
    p = Loss(K, hidden, weight, targets)
    p.check(dloss)
    dhidden = p.backward(dloss)[0]
    p.targets = targets.clone()
    p.targets[:500] = -1  # in parts
    some = p.backward(dloss)[0]
    assert torch.equal(some[500:], dhidden[500:]) and bool((some[:500] == 0).all())
    for first, n in ((0, 1000), (300, 50)):
        q = Loss(K, hidden[first:first + n].clone(), weight, targets[first:first + n].clone())
        q.lse.copy_(p.lse[first:first + n])
        assert torch.equal(q.backward(dloss[first:first + n].clone())[0], dhidden[first:first + n])


# ---- orthogonalisation ----


@pytest.mark.parametrize("steps", [6, 7, 8, 10])
@pytest.mark.parametrize(("batch", "rows", "cols"), [(1, 256, 1024), (3, 576, 576), (2, 1000, 130), (1, 2050, 300)])
def test_bfloat16_updates_of_many_steps(K, steps, batch, rows, cols):  # noqa: F811
    """Singular values near one keep a product's error, so from the fifth step on the operands are pairs: what the kernel adds to the
    result's own rounding (1.66e-3 in the 2-norm, as of any values) is at most 4.5e-4 of it, as the definition with float32's sums and
    those operands has it, a factor of sqrt(1 + 0.27^2) = 1.04; the plain form in float32 is the measure."""
    x = momentum(gen(90), batch, rows, cols, torch.bfloat16)
    got = update(K, x, steps=steps, scale=0.7)
    for i in range(batch):
        value = R.orthogonalize(x[i], steps=steps, scale=0.7)
        plain = R.steps_in_float32(x[i], steps=steps, scale=0.7).bfloat16()
        off, of_plain = (float(torch.linalg.norm(t.double() - value)) for t in (got[i], plain))
        assert off <= 1.05 * of_plain, (i, off / of_plain)
        assert torch.equal(update(K, x[i:i + 1].clone(), steps=steps, scale=0.7)[0], got[i])


def test_bfloat16_updates_of_many_steps_in_place_and_strided(K):  # noqa: F811
    for m, n in ((100, 170), (170, 100)):
        x = momentum(gen(91), 2, m, n, torch.bfloat16)
        want = update(K, x, steps=7)
        wide = torch.full((2, m + 3, n + 11), 5.0, dtype=x.dtype, device="cuda")
        into = wide[:, 1:m + 1, 3:n + 3]
        into.copy_(x)
        assert torch.equal(update(K, into, steps=7, out=into), want)
        into[:] = 5.0
        assert bool((wide == 5.0).all())


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_updates_of_zeroes(K, dtype):  # noqa: F811
    """Zeroes beside any eps; NaN, alone in its batch, without one."""
    x = momentum(gen(93), 2, 20, 70, R.DTYPES[dtype])
    want = update(K, x, eps=0.0)
    x[0] = 0
    for eps in (1e-7, 1e-300, 1e-320):
        assert bool((update(K, x, eps=eps)[0] == 0).all()), eps
    got = update(K, x, eps=0.0)
    assert bool(got[0].isnan().all()) and torch.equal(got[1], want[1])
    assert torch.equal(update(K, x, eps=1e-320)[1], want[1])


def element_limits(x, **options):
    """(value, how far one element may be, how far a row, how far a column, in the 2-norm) as orthogonalize_limits has it for the whole:
    the definition with the operands rounded as they are stated to be is off by so much at most in any element (row, column), and the
    kernel, whose errors are of that kind and as many, may be twice as far; float32's sums too; the result's rounding is added."""
    value = R.orthogonalize(x, **options)
    coarse = x.dtype == torch.bfloat16 and min(x.shape) > 64 and options.get("steps", 5) <= 5
    errors = [R.orthogonalize(x, rounding=R.halves(1 if coarse else 2), **options) - value, R.steps_in_float32(x, **options).double() - value]
    u = R.unit(x.dtype)
    one, row, column = (sum(2 * f(e) for e in errors) for f in (
        lambda e: e.abs().max(), lambda e: e.norm(dim=1).max(), lambda e: e.norm(dim=0).max()))
    return (value, one + 2 * u * value.abs() + R.tiny(x.dtype), row + 2 * u * value.norm(dim=1), column + 2 * u * value.norm(dim=0))


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("batch", "rows", "cols"), [(1, 1, 9), (2, 7, 3), (2, 33, 31), (3, 65, 130), (1, 129, 257), (3, 100, 24), (1, 70, 4200), (65, 2100, 257),
                                                     (1, 1500, 8900), (2, 300, 1001)])
def test_every_element_of_an_update(K, dtype, batch, rows, cols):  # noqa: F811
    """The largest error of an element, and of a row and a column by itself: at the tiles' edges and remainders too."""
    x = momentum(gen(92), batch, rows, cols, R.DTYPES[dtype])
    got = update(K, x, steps=4)
    for i in sorted({0, batch - 1}):
        value, one, row, column = element_limits(x[i], steps=4)
        off = got[i].double() - value
        assert bool((off.abs() <= one).all()), (i, torch.nonzero(off.abs() > one)[0].tolist())
        assert bool((off.norm(dim=1) <= row).all()), (i, torch.nonzero(off.norm(dim=1) > row)[0].tolist())
        assert bool((off.norm(dim=0) <= column).all()), (i, torch.nonzero(off.norm(dim=0) > column)[0].tolist())


# ---- together ----


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_a_step_with_its_roundings(K, dtype):  # noqa: F811
    """The whole step in 16 bits, within twice of what the same step in 64 bits is off by with its results rounded to the type on the
    way (each rounding is one of as many, of random sign), and the last rounding."""
    dt = R.DTYPES[dtype]
    s = Step(K, 42, dt)
    got, want = s.step(), s.reference()

    def rounded(t):
        return t + (t.detach().to(dt).double() - t.detach())

    def rounding(t):
        t.register_hook(lambda g: g.to(dt).double())
        return t

    proj, norm = (t.double().requires_grad_() for t in (s.proj, s.norm))
    ends = [s.table.double().requires_grad_() for _ in range(2)]  # the table's two parts
    x = rounding(rounded(s.scale * ends[0][s.tokens.clamp(min=0)] * (s.tokens >= 0)[:, None]))
    h = rounding(rounded(x + rounded(x @ proj)))
    n = rounding(rounded(h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-5) * norm))
    logits = n @ ends[1].T
    counts, at = s.targets >= 0, s.targets.clamp(min=0)[:, None]
    hot = torch.zeros_like(logits, dtype=torch.bool).scatter_(1, at, True)
    # the softmax's part is an operand in the type, relative to its row; the target's is not
    logits.register_hook(lambda g: torch.where(hot, g, (g * 2.0 ** 20).to(dt).double() / 2.0 ** 20))
    z = 20.0 * torch.tanh(logits / 20.0)
    loss = (torch.logsumexp(z, dim=1) - z.gather(1, at)[:, 0]) * counts
    first, last, dnorm, dproj = torch.autograd.grad((loss * s.dloss.double()).sum(), [*ends, norm, proj])
    close = dict(loss=loss, dtable=(last.to(dt).double() + first).to(dt).double(), dnorm=dnorm, dproj=dproj.to(dt).double())
    for name, value in want.items():
        value = value.detach()
        off, limit = (float((t.detach().double() - value).norm() / value.norm()) for t in (got[name], close[name]))
        assert off <= 2 * limit + R.unit(dt), (name, off, limit)
