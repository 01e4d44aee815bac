"""GPU: the operators at a packed step's ends and its update through the C ABI on device tensors, against their 64-bit
definitions within the bounds of ends_reference, and what they promise beside that."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import ends_reference as R

pytestmark = pytest.mark.gpu

NAMES = {t: n for n, t in R.DTYPES.items()}


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


def space(nbytes):
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device="cuda")


def moved(t):
    """The same values one element further: no array is aligned to 16 bytes."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
    return flat.copy_(t.reshape(-1)).view(t.shape)


# ---- embedding ----


def embed(K, table, tokens, scale=1.0, out=None):
    n, (v, d) = len(tokens), table.shape
    out = torch.full((n, d), math.nan, dtype=table.dtype, device="cuda") if out is None else out
    shape = K.TokenEmbedding(K.DTYPES[NAMES[table.dtype]], n, v, d, 0, scale, out.stride(0) if n else 0)
    K.check(K.lib.dllm_hip_token_embedding(shape, ptr(table), ptr(tokens), ptr(out), stream()))
    return out


def embed_backward(K, tokens, dout, vocabulary, scale=1.0, old=None, workspace=None):
    n, d = dout.shape
    shape = K.TokenEmbedding(K.DTYPES[NAMES[dout.dtype]], n, vocabulary, d, int(old is not None), scale, dout.stride(0) if n else 0)
    got = torch.full((vocabulary, d), math.nan, dtype=dout.dtype, device="cuda") if old is None else old.clone()
    ws = space(K.lib.dllm_hip_token_embedding_backward_workspace(shape)) if workspace is None else workspace
    K.check(K.lib.dllm_hip_token_embedding_backward(shape, ptr(tokens), ptr(dout), ptr(got), ptr(ws), ws.numel(), stream()))
    return got


def some_tokens(g, n, vocabulary):
    """Few tokens often, many seldom, some outside on either side."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    tokens = (torch.exp(u * math.log(vocabulary + 1)).long() - 1).clamp(max=vocabulary - 1)
    strange = torch.rand(n, generator=g, device="cuda") < 0.05
    return torch.where(strange, torch.where(tokens % 2 == 0, -1 - tokens, vocabulary + tokens), tokens)


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("tokens", "vocabulary", "dim"),
                         [(1, 1, 1), (1, 300, 64), (2, 7, 8), (15, 5, 17), (16, 3, 576), (17, 1000, 100), (63, 2, 1025), (1000, 511, 96),
                          (1024, 512, 40), (1025, 513, 24), (5000, 70000, 72), (16384, 300, 16), (16385, 300, 16),
                          (40000, 300000, 9), (33000, 1, 8)])
def test_embedding(K, dtype, tokens, vocabulary, dim):
    g, dt = gen(1), R.DTYPES[dtype]
    ids = some_tokens(g, tokens, vocabulary)
    table, dout, old = (randn(g, n, dim, dtype=dt) for n in (vocabulary, tokens, vocabulary))
    R.assert_within(embed(K, table, ids, 12.5), R.embedding(table, ids, 12.5), "out")
    first = embed_backward(K, ids, dout, vocabulary, 0.3)
    R.assert_within(first, R.embedding_backward(ids, dout, vocabulary, 0.3), "dtable")
    assert torch.equal(first, embed_backward(K, ids, dout, vocabulary, 0.3))
    R.assert_within(embed_backward(K, ids, dout, vocabulary, -2.0, old), R.embedding_backward(ids, dout, vocabulary, -2.0, old), "added")


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_embedding_of_strided_and_unaligned_rows(K, dtype):
    g, dt = gen(2), R.DTYPES[dtype]
    ids = some_tokens(g, 333, 50)
    table, wide = randn(g, 50, 64, dtype=dt), randn(g, 333, 200, dtype=dt)
    for start in (0, 8, 3):  # aligned parts of wider rows, and one that is not
        dout, out = wide[:, start:start + 64], torch.full_like(wide, 7.0)
        R.assert_within(embed(K, table, ids, 2.0, out[:, start:start + 64]), R.embedding(table, ids, 2.0), "out")
        out[:, start:start + 64] = 7.0
        assert bool((out == 7.0).all())  # nothing else was written
        R.assert_within(embed_backward(K, ids, dout, 50), R.embedding_backward(ids, dout, 50), "dtable")
    R.assert_within(embed(K, moved(table), ids), R.embedding(table, ids), "out")
    old = randn(g, 50, 64, dtype=dt)
    shape = K.TokenEmbedding(K.DTYPES[dtype], 333, 50, 64, 1, 1.0, 0)
    got, ws = moved(old), space(K.lib.dllm_hip_token_embedding_backward_workspace(shape))
    dout = moved(wide[:, :64])
    K.check(K.lib.dllm_hip_token_embedding_backward(shape, ptr(ids), ptr(dout), ptr(got), ptr(ws), ws.numel(), stream()))
    R.assert_within(got, R.embedding_backward(ids, wide[:, :64], 50, old=old), "added")


def test_embedding_of_no_tokens_and_of_padding_alone(K):
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    empty, old = torch.zeros(0, 8, device="cuda"), randn(gen(3), 5, 8)
    assert bool((embed_backward(K, none, empty, 5) == 0).all())
    assert torch.equal(embed_backward(K, none, empty, 5, old=old), old)
    for n in (3, 20000):
        pad = torch.full((n,), -100, dtype=torch.int64, device="cuda")
        dout = torch.full((n, 8), math.nan, device="cuda")  # whatever padding holds reaches nothing
        assert bool((embed_backward(K, pad, dout, 5) == 0).all())
        assert torch.equal(embed_backward(K, pad, dout, 5, old=old), old)
        assert bool((embed(K, old, pad) == 0).all())


def test_embedding_backward_reads_no_padding(K):
    """Infinities and NaN in the rows of padding, between others."""
    g = gen(4)
    ids = some_tokens(g, 700, 40)
    dout = randn(g, 700, 24, dtype=torch.bfloat16)
    spoilt = dout.clone()
    spoilt[(ids < 0) | (ids >= 40)] = math.nan
    assert torch.equal(embed_backward(K, ids, spoilt, 40), embed_backward(K, ids, dout, 40))


# ---- loss ----


class Loss:
    """One vocabulary_loss problem on device tensors and its calls."""

    def __init__(self, K, hidden, weight, targets, scale=1.0, softcap=0.0):
        self.K, self.hidden, self.weight, self.targets = K, hidden, weight, targets
        self.options = dict(scale=scale, softcap=softcap)
        t, (v, d) = len(targets), weight.shape
        self.rows, self.dim = t, d
        self.shape = K.VocabularyLoss(K.DTYPES[NAMES[hidden.dtype]], t, v, d, 0, scale, softcap, hidden.stride(0) if t else 0, 0)
        self.workspace = space(max(K.lib.dllm_hip_vocabulary_loss_workspace(self.shape),
                                   K.lib.dllm_hip_vocabulary_loss_backward_workspace(self.shape)))
        self.loss, self.lse = (torch.full((t,), math.nan, device="cuda") for _ in range(2))

    def forward(self):
        self.K.check(self.K.lib.dllm_hip_vocabulary_loss(
            self.shape, ptr(self.hidden), ptr(self.weight), ptr(self.targets), ptr(self.loss), ptr(self.lse), ptr(self.workspace),
            self.workspace.numel(), stream()))
        return self.loss, self.lse

    def backward(self, dloss, old=None, dhidden=None, want=(True, True)):
        if dhidden is None:
            dhidden = torch.full((self.rows, self.dim), math.nan, dtype=self.hidden.dtype, device="cuda")
        dweight = torch.full_like(self.weight, math.nan) if old is None else old.clone()
        self.shape.accumulate, self.shape.dhidden_stride = int(old is not None), dhidden.stride(0) if self.rows else 0
        dhidden, dweight = dhidden if want[0] else None, dweight if want[1] else None
        self.K.check(self.K.lib.dllm_hip_vocabulary_loss_backward(
            self.shape, ptr(self.hidden), ptr(self.weight), ptr(self.targets), ptr(self.lse), ptr(dloss), ptr(dhidden), ptr(dweight),
            ptr(self.workspace), self.workspace.numel(), stream()))
        return dhidden, dweight

    def check(self, dloss=None, old=None):
        loss, lse = self.forward()
        want = R.loss(self.hidden, self.weight, self.targets, **self.options)
        R.assert_within(lse, want["lse"], "lse")
        R.assert_within(loss, want["loss"], "loss")
        if dloss is None:
            return
        dhidden, dweight = self.backward(dloss, old)
        want = R.loss_backward(self.hidden, self.weight, self.targets, lse, dloss, old=old, **self.options)
        R.assert_within(dhidden, want["dhidden"], "dhidden")
        R.assert_within(dweight, want["dweight"], "dweight")


def loss_problem(K, seed, dtype, rows, vocabulary, dim, masked=0.2, **options):
    g = gen(seed)
    weight = randn(g, vocabulary, dim, dtype=dtype, scale=2.0 / math.sqrt(dim))
    targets = torch.randint(0, vocabulary, (rows,), generator=g, device="cuda")
    # from rows that know nothing to rows that are sure of their target
    sure = torch.rand(rows, 1, generator=g, device="cuda") * 4.0
    hidden = (randn(g, rows, dim) + sure * weight[targets].float()).to(dtype)
    strange = torch.rand(rows, generator=g, device="cuda") < masked
    targets = torch.where(strange, torch.where(targets % 2 == 0, -1 - targets, targets + vocabulary), targets)
    dloss = torch.rand(rows, generator=g, device="cuda") / max(rows, 1)
    return Loss(K, hidden, weight, targets, **options), dloss


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("rows", "vocabulary", "dim"),
                         [(1, 1, 1), (1, 300, 64), (2, 127, 8), (3, 128, 17), (31, 129, 100), (32, 257, 128), (33, 1000, 72), (64, 8191, 64),
                          (65, 8192, 24), (129, 8193, 192), (255, 16385, 40), (257, 20000, 136), (600, 700, 576), (1030, 3000, 65)])
def test_loss(K, dtype, rows, vocabulary, dim):
    p, dloss = loss_problem(K, 10, R.DTYPES[dtype], rows, vocabulary, dim)
    p.check(dloss)


# the largest tiles, tiles that add their units in turn, both at once
@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("rows", "vocabulary", "dim"), [(1000, 32700, 508), (2100, 5000, 1200), (4096, 16384, 2560)])
def test_loss_of_large_batches(K, dtype, rows, vocabulary, dim):
    p, dloss = loss_problem(K, 26, R.DTYPES[dtype], rows, vocabulary, dim, masked=0.05)
    p.check(dloss, randn(gen(27), vocabulary, dim, dtype=R.DTYPES[dtype], scale=1e-3))


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("options", [dict(scale=0.25), dict(softcap=3.0), dict(scale=8.0, softcap=5.0), dict(softcap=1e6),
                                     dict(scale=2.0 ** -60, softcap=2.0 ** -64), dict(scale=100.0, softcap=30.0)])
def test_loss_bends(K, dtype, options):
    """Scales and caps; caps that the logits nearly reach, and caps that they never come near."""
    p, dloss = loss_problem(K, 11, R.DTYPES[dtype], 140, 1500, 80, **options)
    old = randn(gen(12), 1500, 80, dtype=R.DTYPES[dtype], scale=1e-3)
    p.check(dloss, old)


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("counted", [1, 255, 257, 700, 2099])
@pytest.mark.parametrize(("vocabulary", "dim"), [(20000, 96), (3000, 1100)])
def test_loss_of_a_batch_of_which_few_rows_count(K, dtype, counted, vocabulary, dim):
    """The tiles are those of the rows that count: at a tile's edge, in few of the launch's, behind many that do not."""
    p, dloss = loss_problem(K, 29, R.DTYPES[dtype], 2100, vocabulary, dim, masked=0.0)
    p.targets[:2100 - counted] = -1
    p.check(dloss, randn(gen(30), vocabulary, dim, dtype=R.DTYPES[dtype], scale=1e-3))


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("counted", [1000, 3900])
def test_loss_of_a_wide_batch_of_which_some_rows_count(K, dtype, counted):
    """Enough tiles for each to take the vocabulary's units in turn, and, of the rows that count, too few; the same bits either way."""
    p, dloss = loss_problem(K, 31, R.DTYPES[dtype], 4096, 16384, 2560, masked=0.0)
    p.targets[:4096 - counted] = -1
    p.check(dloss, randn(gen(32), 16384, 2560, dtype=R.DTYPES[dtype], scale=1e-3))
    lse, dhidden = p.lse.clone(), p.backward(dloss)[0]
    q = Loss(K, p.hidden[-300:].clone(), p.weight, p.targets[-300:].clone())
    q.lse.copy_(lse[-300:])
    assert torch.equal(q.backward(dloss[-300:].clone())[0], dhidden[-300:])


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_loss_of_rows_that_do_not_count(K, dtype):
    """What they hold reaches nothing, and their rows of the results are zero; none at all, and all but none."""
    dt = R.DTYPES[dtype]
    p, dloss = loss_problem(K, 13, dt, 300, 900, 64, masked=0.5)
    out = (p.targets < 0) | (p.targets >= 900)
    want = [t.clone() for t in (*p.forward(), *p.backward(dloss))]
    p.hidden = torch.where(out[:, None], torch.full_like(p.hidden, math.nan), p.hidden)
    got = [*p.forward(), *p.backward(torch.where(out, torch.full_like(dloss, math.inf), dloss))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert bool((got[0][out] == 0).all()) and bool((got[1][out] == 0).all()) and bool((got[2][out] == 0).all())
    p.targets[:] = -100
    old = randn(gen(14), 900, 64, dtype=dt)
    assert all(bool((t == 0).all()) for t in (*p.forward(), *p.backward(dloss)))
    dhidden, dweight = p.backward(dloss, old)
    assert bool((dhidden == 0).all()) and torch.equal(dweight, old)
    p.targets[299] = 17
    p.hidden[299] = 0.5
    p.check(dloss)


def test_loss_of_no_rows(K):
    p, dloss = loss_problem(K, 15, torch.bfloat16, 0, 50, 16)
    p.forward()
    _, dweight = p.backward(dloss)
    assert bool((dweight == 0).all())
    old = randn(gen(16), 50, 16, dtype=torch.bfloat16)
    assert torch.equal(p.backward(dloss, old)[1], old)


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_loss_spoilt_rows_are_their_own(K, dtype):
    """A NaN in one row's hidden state is that row's: the others' loss and dhidden are what they were."""
    p, dloss = loss_problem(K, 17, R.DTYPES[dtype], 70, 400, 64, masked=0.0)
    want = [t.clone() for t in p.forward()] + [p.backward(dloss)[0].clone()]
    p.hidden[33, 5] = math.nan
    got = [t.clone() for t in p.forward()] + [p.backward(dloss)[0]]
    others = torch.arange(70, device="cuda") != 33
    assert all(torch.equal(a[others], b[others]) for a, b in zip(got, want))
    assert bool(got[0][33].isnan()) and bool(got[1][33].isnan()) and bool(got[2][33].isnan().all())


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_loss_of_strided_and_unaligned_arrays(K, dtype):
    dt = R.DTYPES[dtype]
    p, dloss = loss_problem(K, 18, dt, 77, 333, 72)
    want = [t.clone() for t in (*p.forward(), *p.backward(dloss))]
    wide = randn(gen(19), 77, 200, dtype=dt)
    for start in (8, 5):
        part = wide[:, start:start + 72]
        part.copy_(p.hidden)
        q = Loss(K, part, moved(p.weight) if start == 5 else p.weight, p.targets)
        into = torch.full_like(wide, 3.0)
        got = [*q.forward(), *q.backward(dloss, dhidden=into[:, start:start + 72])]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        into[:, start:start + 72] = 3.0
        assert bool((into == 3.0).all())


def test_loss_results_alone(K):
    """Each result without the other."""
    p, dloss = loss_problem(K, 20, torch.bfloat16, 90, 1000, 64)
    loss, lse = (t.clone() for t in p.forward())
    dhidden, dweight = p.backward(dloss)
    assert torch.equal(p.backward(dloss, want=(True, False))[0], dhidden)
    assert torch.equal(p.backward(dloss, want=(False, True))[1], dweight)
    assert p.backward(dloss, want=(False, False)) == (None, None)
    for keep in ("loss", "lse"):
        q, _ = loss_problem(K, 20, torch.bfloat16, 90, 1000, 64)
        setattr(q, "lse" if keep == "loss" else "loss", None)
        q.forward()
        assert torch.equal(getattr(q, keep), loss if keep == "loss" else lse)


# odd and short rows, whose weights are packed also where rows are few
@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("rows", "vocabulary", "dim"), [(1, 3, 2), (5, 700, 33), (40, 2100, 33), (100, 700, 67), (256, 5000, 7)])
def test_loss_of_few_rows_packed(K, dtype, rows, vocabulary, dim):
    p, dloss = loss_problem(K, 28, R.DTYPES[dtype], rows, vocabulary, dim)
    p.check(dloss)


def in_few_rows(K, p):
    """The results of a batch's rows, 256 at once."""
    few = [Loss(K, p.hidden[i:i + 256].clone(), p.weight, p.targets[i:i + 256].clone()).forward() for i in range(0, p.rows, 256)]
    return torch.cat([f[0] for f in few]), torch.cat([f[1] for f in few])


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("vocabulary", "dim"), [(20000, 96), (9000, 130)])
def test_a_row_alone_and_in_a_batch(K, dtype, vocabulary, dim):
    """A row's loss, lse and dhidden are the same bits in batches of any size, and every call gives the same bits. (float32's loss
    and lse: in all of at most 256 rows, and in all of more.)"""
    p, dloss = loss_problem(K, 21, R.DTYPES[dtype], 700, vocabulary, dim, masked=0.1)
    loss, lse = (t.clone() for t in p.forward())
    dhidden, dweight = p.backward(dloss)
    again = p.backward(dloss)
    assert torch.equal(again[0], dhidden) and torch.equal(again[1], dweight)
    few = in_few_rows(K, p)
    assert dtype == "float32" or (torch.equal(few[0], loss) and torch.equal(few[1], lse))
    for first, n in [(0, 1), (5, 30), (64, 64), (100, 65), (300, 129), (13, 257), (1, 600)]:
        rows = slice(first, first + n)
        q = Loss(K, p.hidden[rows].clone(), p.weight, p.targets[rows].clone())
        got, want = q.forward(), few if n <= 256 else (loss, lse)
        assert torch.equal(got[0], want[0][rows]) and torch.equal(got[1], want[1][rows]), n
        q.lse.copy_(lse[rows])
        assert torch.equal(q.backward(dloss[rows].clone())[0], dhidden[rows]), n


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_a_row_alone_and_in_a_batch_of_pieces(K, dtype):
    """The same of a batch that goes over the vocabulary in several pieces, and lists its rows by a launch of its own."""
    p, dloss = loss_problem(K, 25, R.DTYPES[dtype], 20000, 20000, 24)
    loss, lse = (t.clone() for t in p.forward())
    dhidden, _ = p.backward(dloss)
    few = in_few_rows(K, p)
    for first, n in [(0, 3), (7000, 90), (19700, 300)]:
        rows = slice(first, first + n)
        q = Loss(K, p.hidden[rows].clone(), p.weight, p.targets[rows].clone())
        got, want = q.forward(), few if n <= 256 else (loss, lse)
        assert torch.equal(got[0], want[0][rows]) and torch.equal(got[1], want[1][rows]), n
        q.lse.copy_(lse[rows])
        assert torch.equal(q.backward(dloss[rows].clone())[0], dhidden[rows]), n
    assert bool(torch.isfinite(dhidden).all())


@pytest.mark.parametrize("size", [1e-6, 1e3])
def test_float16_loss_gradients_of_any_size(K, size):
    """Upstream gradients far below and above one, and unequal ones."""
    p, dloss = loss_problem(K, 22, torch.float16, 200, 600, 64)
    spread = torch.exp2(-torch.arange(200, device="cuda") % 8).float()
    p.check(dloss * size * spread)


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_loss_of_a_target_that_is_sure(K, dtype):
    """Probabilities of the target within 1e-5 of one: p - 1 is formed from the exponents' difference."""
    dt = R.DTYPES[dtype]
    g = gen(23)
    weight = randn(g, 500, 64, dtype=dt)
    targets = torch.randint(0, 500, (100,), generator=g, device="cuda")
    hidden = (weight[targets].float() * torch.linspace(0.1, 1.0, 100, device="cuda")[:, None]).to(dt)
    Loss(K, hidden, weight, targets).check(torch.full((100,), 0.01, device="cuda"))


def test_loss_of_one_target_for_all(K):
    p, dloss = loss_problem(K, 24, torch.float16, 3000, 40, 32, masked=0.0)
    p.targets[:] = 7
    p.check(dloss)


# ---- orthogonalisation ----


def update(K, x, steps=5, coefficients=None, eps=1e-7, scale=1.0, out=None):
    b, m, n = x.shape
    out = torch.full((b, m, n), math.nan, dtype=x.dtype, device="cuda") if out is None else out
    shape = K.Orthogonalize(K.DTYPES[NAMES[x.dtype]], b, m, n, steps, eps, scale, x.stride(1), x.stride(0), out.stride(1), out.stride(0))
    ws = space(K.lib.dllm_hip_orthogonalize_workspace(shape))
    host = None if coefficients is None else (K.C.c_double * (3 * steps))(*[v for c in coefficients for v in c])
    K.check(K.lib.dllm_hip_orthogonalize(shape, host, ptr(x), ptr(out), ptr(ws), ws.numel(), stream()))
    return out


def check_update(K, x, **options):
    got = update(K, x, **options)
    for i in range(x.shape[0]):
        value, limit = R.orthogonalize_limits(x[i], **options)
        off = float(torch.linalg.norm(got[i].double() - value) / torch.linalg.norm(value))
        assert off <= limit, (i, off, limit)
    return got


def momentum(g, b, m, n, dtype, size=1e-3):
    x = randn(g, b, m, n)
    r = min(4, m, n)
    return ((x + randn(g, b, m, r, scale=6.0) @ randn(g, b, r, n)) * size).to(dtype)


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("batch", "rows", "cols"),
                         [(1, 1, 1), (3, 1, 9), (2, 7, 3), (1, 8, 64), (2, 33, 31), (1, 64, 64), (3, 65, 130), (2, 128, 128), (1, 129, 257),
                          (5, 100, 24), (1, 300, 1000), (1, 1100, 260), (2, 513, 576), (9, 256, 300)])
def test_orthogonalize(K, dtype, batch, rows, cols):
    x = momentum(gen(30), batch, rows, cols, R.DTYPES[dtype])
    got = check_update(K, x, scale=0.7)
    assert torch.equal(got, update(K, x, scale=0.7))
    one = update(K, x[batch - 1:].clone(), scale=0.7)  # a matrix alone has the bits that it has among others
    assert torch.equal(one[0], got[-1])


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize(("batch", "rows", "cols"), [(1, 130, 4200), (1, 1500, 8900), (65, 2100, 257), (3, 700, 3000)])
def test_orthogonalize_long_sides(K, dtype, batch, rows, cols):
    """Sums over a long side in segments, at once (few matrices) and in turn (many): the same bits; the largest tiles."""
    x = momentum(gen(36), batch, rows, cols, R.DTYPES[dtype])
    some = [0, batch // 2, batch - 1]
    got = update(K, x, steps=3)
    for i in sorted(set(some)):
        value, limit = R.orthogonalize_limits(x[i], steps=3)
        off = float(torch.linalg.norm(got[i].double() - value) / torch.linalg.norm(value))
        assert off <= limit, (i, off, limit)
        assert torch.equal(update(K, x[i:i + 1].clone(), steps=3)[0], got[i])


@pytest.mark.parametrize("dtype", R.DTYPES)
@pytest.mark.parametrize("options", [dict(steps=0), dict(steps=1), dict(steps=2, scale=-3.0), dict(steps=8), dict(eps=0.5),
                                     dict(steps=3, coefficients=[(1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (3.0, -3.2, 1.2)])])
def test_orthogonalize_options(K, dtype, options):
    check_update(K, momentum(gen(31), 2, 90, 200, R.DTYPES[dtype]), **options)


@pytest.mark.parametrize(("dtype", "size"), [("float32", 1e-30), ("float32", 1e25), ("bfloat16", 1e-30), ("bfloat16", 1e30), ("float16", 10.0)])
def test_orthogonalize_updates_of_any_size(K, dtype, size):
    """The squares of these are more or less than float32 holds."""
    check_update(K, momentum(gen(32), 1, 40, 90, R.DTYPES[dtype], size), eps=0.0)


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_orthogonalize_strided_in_place_and_unaligned(K, dtype):
    dt = R.DTYPES[dtype]
    for m, n in ((50, 70), (70, 50)):
        x = momentum(gen(33), 2, m, n, dt)
        want = update(K, x)
        wide = torch.full((2, m + 3, n + 11), 5.0, dtype=dt, device="cuda")
        into = wide[:, 1:m + 1, 3:n + 3]
        into.copy_(x)
        assert torch.equal(update(K, into), want)
        assert torch.equal(update(K, into, out=into), want)
        into[:] = 5.0
        assert bool((wide == 5.0).all())
        assert torch.equal(update(K, moved(x)), want)


def test_orthogonalize_nothing(K):
    """A matrix of zeroes stays one, beside another."""
    x = momentum(gen(34), 3, 30, 40, torch.bfloat16)
    x[1] = 0
    got = check_update(K, x[[0, 2]])
    all_three = update(K, x)
    assert bool((all_three[1] == 0).all()) and torch.equal(all_three[[0, 2]], got)


def test_orthogonalize_makes_singular_values_alike(K):
    """What it is for: singular values from 1 to 1 / 30 of the largest all end between 0.6 and 1.3 in eight steps (the published
    coefficients keep them in about [0.68, 1.13]; 16-bit rounding adds a few hundredths)."""
    g = gen(35)
    u, v = (torch.linalg.qr(torch.randn(n, 64, generator=g, device="cuda"))[0] for n in (64, 200))
    x = (u * torch.linspace(1.0, 30.0, 64, device="cuda")) @ v.T
    for dt in R.DTYPES.values():
        s = torch.linalg.svdvals(update(K, x[None].to(dt), steps=8)[0].float())
        assert 0.6 < float(s.min()) and float(s.max()) < 1.3, (dt, s.min(), s.max())


# ---- together ----


class Step:
    """A training step of a small tied model on packed tokens: lookup, norm, a projection, the loss and all gradients; the table's
    from both ends; and the projection's update."""

    def __init__(self, K, seed, dt):
        g, self.K, self.dt = gen(seed), K, dt
        self.n, self.vocabulary, self.dim = 400, 1200, 96
        self.tokens = some_tokens(g, self.n, self.vocabulary).clamp(-1, self.vocabulary - 1)
        self.targets = torch.where(torch.rand(self.n, generator=g, device="cuda") < 0.3, -100,
                                   torch.randint(0, self.vocabulary, (self.n,), generator=g, device="cuda"))
        self.table = randn(g, self.vocabulary, self.dim, dtype=dt, scale=0.3)
        self.proj = randn(g, self.dim, self.dim, dtype=dt, scale=self.dim ** -0.5)
        self.norm = 1 + randn(g, self.dim, scale=0.1)
        self.dloss = torch.full((self.n,), 1.0 / 280, device="cuda")
        self.scale = math.sqrt(self.dim)
        code = K.DTYPES[NAMES[dt]]
        self.residual = K.ResidualNorm(code, self.n, self.dim, 0, 0, 0, 1e-5, 1.0)
        self.embedding = K.TokenEmbedding(code, self.n, self.vocabulary, self.dim, 1, self.scale)
        self.loss_shape = K.VocabularyLoss(code, self.n, self.vocabulary, self.dim, 0, 1.0, 20.0)
        self.update_shape = K.Orthogonalize(code, 1, self.dim, self.dim, 5, 1e-7, 0.2)
        need = [K.lib.dllm_hip_residual_norm_backward_workspace(self.residual), K.lib.dllm_hip_token_embedding_backward_workspace(self.embedding),
                K.lib.dllm_hip_vocabulary_loss_workspace(self.loss_shape), K.lib.dllm_hip_vocabulary_loss_backward_workspace(self.loss_shape),
                K.lib.dllm_hip_orthogonalize_workspace(self.update_shape)]
        self.ws = space(max(need))

    def step(self):
        K, ws = self.K, self.ws
        new = lambda *shape, dtype=self.dt: torch.full(shape, math.nan, dtype=dtype, device="cuda")  # noqa: E731
        x, h, n = (new(self.n, self.dim) for _ in range(3))
        K.check(K.lib.dllm_hip_token_embedding(self.embedding, ptr(self.table), ptr(self.tokens), ptr(x), stream()))
        y = x @ self.proj
        K.check(K.lib.dllm_hip_residual_norm(self.residual, ptr(x), ptr(y), None, None, ptr(self.norm), ptr(h), ptr(n), stream()))
        loss, lse = (new(self.n, dtype=torch.float32) for _ in range(2))
        K.check(K.lib.dllm_hip_vocabulary_loss(self.loss_shape, ptr(n), ptr(self.table), ptr(self.targets), ptr(loss), ptr(lse), ptr(ws),
                                               ws.numel(), stream()))
        dn, dtable, dx, dy = new(self.n, self.dim), new(self.vocabulary, self.dim), new(self.n, self.dim), new(self.n, self.dim)
        K.check(K.lib.dllm_hip_vocabulary_loss_backward(self.loss_shape, ptr(n), ptr(self.table), ptr(self.targets), ptr(lse), ptr(self.dloss),
                                                        ptr(dn), ptr(dtable), ptr(ws), ws.numel(), stream()))
        dnorm = new(self.dim, dtype=torch.float32)
        K.check(K.lib.dllm_hip_residual_norm_backward(self.residual, ptr(h), ptr(y), None, None, ptr(self.norm), None, ptr(dn), ptr(dx), ptr(dy),
                                                      None, None, ptr(dnorm), ptr(ws), ws.numel(), stream()))
        dproj = x.T @ dy
        dx = dx + dy @ self.proj.T
        K.check(K.lib.dllm_hip_token_embedding_backward(self.embedding, ptr(self.tokens), ptr(dx), ptr(dtable), ptr(ws), ws.numel(), stream()))
        turn = new(self.dim, self.dim)
        K.check(K.lib.dllm_hip_orthogonalize(self.update_shape, None, ptr(dproj), ptr(turn), ptr(ws), ws.numel(), stream()))
        return dict(loss=loss, dtable=dtable, dnorm=dnorm, dproj=dproj, turn=turn)

    def reference(self):
        d = lambda t: t.detach().double().requires_grad_()  # noqa: E731
        table, proj, norm = d(self.table), d(self.proj), d(self.norm)
        x = self.scale * table[self.tokens.clamp(min=0)] * (self.tokens >= 0)[:, None]
        h = x + x @ proj
        n = h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-5) * norm
        z = 20.0 * torch.tanh(n @ table.T / 20.0)
        counts = self.targets >= 0
        loss = (torch.logsumexp(z, dim=1) - z.gather(1, self.targets.clamp(min=0)[:, None])[:, 0]) * counts
        grads = torch.autograd.grad((loss * self.dloss.double()).sum(), [table, norm, proj])
        return dict(loss=loss, **dict(zip(("dtable", "dnorm", "dproj"), grads)))


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_a_step(K, dtype):
    """The whole step against 64 bits: about eight results are rounded to the type on the way, each off by at most u of itself, and
    every step's condition is a small factor, so the 2-norms are held to 100 u (float32, whose longest sums have 1200 terms,
    to 2000 F); the update of the gradient that came out, within its own limits."""
    s = Step(K, 40, R.DTYPES[dtype])
    got, want = s.step(), s.reference()
    limit = 2000 * R.F if dtype == "float32" else 100 * R.unit(s.dt)
    for name in want:
        off = float((got[name].double() - want[name].detach()).norm() / want[name].detach().norm())
        assert off < limit, (name, off)
    value, limit = R.orthogonalize_limits(got["dproj"], scale=0.2)
    assert float((got["turn"].double() - value).norm() / value.norm()) <= limit


@pytest.mark.parametrize("dtype", R.DTYPES)
def test_a_step_on_another_stream_and_in_a_graph(K, dtype):
    s = Step(K, 41, R.DTYPES[dtype])
    want = {n: t.clone() for n, t in s.step().items()}
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = s.step()
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = s.step()
    for _ in range(4):
        for t in held.values():
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(held[n], want[n]) for n in want)
        assert all(torch.equal(t, want[n]) for n, t in s.step().items())
        torch.cuda.synchronize()


def test_two_losses_at_once(K):
    """Two streams, a workspace each."""
    problems = [loss_problem(K, 50 + i, torch.bfloat16, 300 + 77 * i, 2000, 64) for i in range(2)]
    want = [[t.clone() for t in (*p.forward(), *p.backward(d))] for p, d in problems]
    torch.cuda.synchronize()
    got = []
    for p, d in problems:
        with torch.cuda.stream(torch.cuda.Stream()):
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
    dt, g = R.DTYPES[dtype], gen(60)
    table, dout = randn(g, 30, 20, dtype=dt), randn(g, 44, 20, dtype=dt)
    ids = some_tokens(g, 44, 30).clamp(-5, 29)
    tokens = ids.cpu().numpy()
    assert np.array_equal(K.token_embedding(bits(table), tokens, 3.0), bits(embed(K, table, ids, 3.0)))
    assert np.array_equal(K.token_embedding_backward(tokens, bits(dout), 30), bits(embed_backward(K, ids, dout, 30)))
    assert np.array_equal(K.token_embedding_backward(tokens, bits(dout), 30, 0.5, bits(table)), bits(embed_backward(K, ids, dout, 30, 0.5, table)))
    p, dloss = loss_problem(K, 61, dt, 44, 90, 20, softcap=4.0)
    p.targets = p.targets.clamp(max=89)
    loss, lse = p.forward()
    args = bits(p.hidden), bits(p.weight), p.targets.cpu().numpy()
    got = K.vocabulary_loss(*args, softcap=4.0)
    assert np.array_equal(got[0], bits(loss)) and np.array_equal(got[1], bits(lse))
    for old in (None, randn(g, 90, 20, dtype=dt)):
        got = K.vocabulary_loss_backward(*args, bits(lse), bits(dloss), softcap=4.0, dweight=None if old is None else bits(old))
        assert all(np.array_equal(a, bits(b)) for a, b in zip(got, p.backward(dloss, old)))
    x = momentum(g, 2, 12, 30, dt)
    assert np.array_equal(K.orthogonalize(bits(x)), bits(update(K, x)))
    assert np.array_equal(K.orthogonalize(bits(x[0]), 2, [(1.5, -0.5, 0.0)] * 2), bits(update(K, x[:1], 2, [(1.5, -0.5, 0.0)] * 2)[0]))
