"""The definitions in 64 bits of the operators at a packed step's ends and of its update, and how far a correct kernel's
results may be from them: absolute bounds per element from the number of roundings, as in packed_reference."""

from __future__ import annotations

import math

import torch

from packed_reference import DTYPES, F, assert_within, tiny, unit  # noqa: F401

QUINTIC = (3.4445, -4.7750, 2.0315)


def embedding(table, tokens, scale=1.0):
    inside = (tokens >= 0) & (tokens < len(table))
    value = scale * table[tokens.clamp(0, len(table) - 1)].double() * inside[:, None]
    # scale's own rounding, the product's, and the result's
    return value, (unit(table.dtype) + 2 * F) * value.abs() * (1 + F) + tiny(table.dtype)


def embedding_backward(tokens, dout, vocabulary, scale=1.0, old=None):
    inside = (tokens >= 0) & (tokens < vocabulary)
    ids, d = tokens[inside], dout[inside].double()
    total, size = (torch.zeros(vocabulary, dout.shape[1], dtype=torch.float64, device=dout.device) for _ in range(2))
    total.index_add_(0, ids, d)
    size.index_add_(0, ids, d.abs())
    n = torch.bincount(ids, minlength=vocabulary)[:, None].double()
    value, err = scale * total, abs(scale) * size * (n + 3) * F
    if old is not None:
        value = value + old.double()
        err = err + F * value.abs()
    seen = torch.ones_like(value) if old is None else (n > 0).double()  # other rows stay as they are
    return value, ((unit(dout.dtype) * value.abs() + err) * (1 + unit(dout.dtype)) + tiny(dout.dtype)) * seen


def _floors(hidden, weight):
    """Float32 values are multiplied as pairs of float16, scaled to below 2^15 by their row's (hidden states) or by 2048 rows'
    (weights) largest: a pair's second part is off by half of float16's least step, 2^-25 there, so 2^-39 of the largest."""
    if hidden.dtype != torch.float32:
        return 0.0, 0.0
    floor = lambda t: 2.0 ** -39 * t.abs().amax()  # noqa: E731
    units = [floor(u).expand(len(u)) for u in weight.double().split(2048)]
    return 2.0 ** -39 * hidden.double().abs().amax(dim=1, keepdim=True), torch.cat(units)[:, None]


def _logits(hidden, weight, scale, softcap):
    """(z, bound, derivative, its bound)."""
    h, w = hidden.double(), weight.double()
    x = scale * (h @ w.T)
    # a sum of dim products in any order, and the scale's two roundings; a pair of float16 is off by 2 F at most, and the product
    # of two pairs' second parts, 4 F, is left out: 8 F of a product
    err = (h.shape[1] + 16) * F * scale * (h.abs() @ w.abs().T)
    fh, fw = _floors(hidden, weight)
    if hidden.dtype == torch.float32:
        err = err + scale * (fh * w.abs().sum(dim=1) + h.abs().sum(dim=1, keepdim=True) * fw.T)
    slope, es = torch.ones_like(x), torch.zeros_like(x)
    if softcap:
        y = x / softcap
        slope = 1.0 / torch.cosh(y).square()
        # tanh to 6 F of itself and its argument's rounding (y F slope, at most F / 2 of the cap's size); the derivative to
        # about 12 F of itself, and twice the argument's error times it, as d slope / dy is at most 2 slope
        err = err * slope + softcap * (8 * F * torch.tanh(y).abs() + 2 * F * y.abs() * slope)
        es = slope * (16 * F + 2 * (scale / softcap) * (h.shape[1] + 16) * F * (h.abs() @ w.abs().T) + 4 * F * y.abs())
        x = softcap * torch.tanh(y)
    return x, err + 2 * F * x.abs(), slope, es


def loss(hidden, weight, targets, scale=1.0, softcap=0.0):
    """{"loss", "lse"}: (value, bound)."""
    inside = (targets >= 0) & (targets < len(weight))
    hidden = torch.where(inside[:, None], hidden, torch.zeros_like(hidden))
    z, err, _, _ = _logits(hidden, weight, scale, softcap)
    lse = torch.logsumexp(z, dim=1)
    at = targets.clamp(0, len(weight) - 1)[:, None]
    # every logit's error reaches the sum with its weight, an exponent's rounding with its distance from the largest; the
    # sum itself is one of 128 terms, then of parts (at most vocabulary / 8192 + 7 of them), each joined with a few roundings
    p = torch.exp(z - lse[:, None])
    steps = 128 + 4 * (len(weight) / 8192 + 8) + 16
    e = (p * (err + 4 * F * (z.amax(dim=1, keepdim=True) - z + 1))).sum(dim=1) + steps * F + 3 * F * lse.abs()
    one = z.gather(1, at)[:, 0]
    got = dict(lse=(lse, e), loss=(lse - one, e + err.gather(1, at)[:, 0] + 2 * F * (lse.abs() + one.abs())))
    return {n: (v * inside, b * inside) for n, (v, b) in got.items()}


def loss_backward(hidden, weight, targets, lse, dloss, scale=1.0, softcap=0.0, old=None):
    """{"dhidden", "dweight"}: (value, bound)."""
    dt = hidden.dtype
    u = unit(dt)
    up = 0.0 if dt == torch.float32 else u  # the softmax's part is an operand in the type
    inside = (targets >= 0) & (targets < len(weight))
    hidden = torch.where(inside[:, None], hidden, torch.zeros_like(hidden))
    lse = torch.where(inside, lse, torch.zeros_like(lse)).double()[:, None]
    z, err, slope, es = _logits(hidden, weight, scale, softcap)
    factor = torch.where(inside, dloss.double() * scale, torch.zeros_like(lse[:, 0]))[:, None]
    at = targets.clamp(0, len(weight) - 1)[:, None]
    e = z - lse
    p = torch.exp(e)
    # the exponent's error, its own roundings (the difference, the product by 1 / log 2, the power's last bit)
    ep = p * (torch.expm1(err + 4 * F * (e.abs() + lse.abs() * 0 + 2)))
    hot = torch.zeros_like(z).scatter_(1, at, 1.0)
    soft = torch.where(hot > 0, torch.expm1(e), p)
    esoft = ep + 4 * F * soft.abs()
    g = soft * slope * factor
    eg = factor.abs() * (esoft * slope + soft.abs() * es + 6 * F * soft.abs() * slope)
    rounded = (g.abs() + eg) * (1 - hot)  # the target's element stays in float32
    eg = eg + rounded * up
    if dt != torch.bfloat16:
        # held times 2^14 relative to the row's weight: near zero off by half of 2^-24 of that; a pair
        # (float32) by 2 F of itself too
        eg = eg + (1 - hot) * factor.abs() * 2.0 ** -39 + (2 * F * rounded if dt == torch.float32 else 0.0)
    h, w = hidden.double(), weight.double()
    n = len(weight) + 16
    value, size = g @ w, g.abs() @ w.abs()
    got = dict(dhidden=(value, eg @ w.abs() + (n + 16) * F * size))
    fh, fw = _floors(hidden, weight)
    if dt == torch.float32:
        got = dict(dhidden=(value, got["dhidden"][1] + g.abs() @ fw.expand(-1, w.shape[1])))
    value, bound = g.T @ h, eg.T @ h.abs() + (len(h) + 32) * F * (g.abs().T @ h.abs())
    if dt == torch.float32:
        # the hidden states as operands here: below 2^15 by the largest row's, weighted
        heavy = (factor.abs() * h.abs().amax(dim=1, keepdim=True)).max() * 2.0 ** -38
        bound = bound + (soft.abs() * (1 - hot) * slope * (factor != 0)).sum(dim=0)[:, None] * heavy
    if dt == torch.float16:
        # the hidden states of light rows are held relative to the heaviest: off by half of 2^-24 there, times the weight
        soft16 = soft.abs() * (1 - hot) * slope * (factor.abs() > 0)
        bound = bound + soft16.T @ (torch.full_like(h, 2.0 ** -24) * (h != 0)) * factor.abs().max()
    if old is not None:
        value = value + old.double()
    got["dweight"] = (value, bound + 2 * F * value.abs())
    return {k: (v, (u * v.abs() + b) * (1 + u) + tiny(dt)) for k, (v, b) in got.items()}


def orthogonalize(x, steps=5, coefficients=None, eps=1e-7, scale=1.0, rounding=None):
    """One matrix in float64; `rounding` is applied to the products' operands X, A and B."""
    rounding = rounding or (lambda t: t)
    x = x.double()
    turned = x.shape[0] > x.shape[1]
    if turned:
        x = x.T
    x = x / (torch.linalg.norm(x) + eps)
    for i in range(steps):
        a, b, c = QUINTIC if coefficients is None else coefficients[i]
        r = rounding(x)
        gram = rounding(r @ r.T)
        x = a * x + rounding(b * gram + c * gram @ gram) @ r
    return scale * (x.T if turned else x)


def halves(planes: int):
    """Rounding to a sum of float16 parts, of values around one."""

    def rounding(t):
        left, total = t.clone(), torch.zeros_like(t)
        for _ in range(planes):
            part = (left * 256.0).half().double() / 256.0
            total, left = total + part, left - part
        return total

    return rounding


def orthogonalize_limits(x, **options):
    """(value, how far in the 2-norm, relative). A rounding's way through the steps is no matter of a few factors (small
    singular values grow by 3.4 in each, errors with them), so the definition is computed with the operands rounded as they are
    stated to be (float16 for bfloat16 matrices with more than 64 on the smaller side, else pairs of it), and the kernel may be twice as far away; what float32's sums add
    (dim terms each, of random sign: the root of their number) is taken from the same steps in float32, twice too."""
    value = orthogonalize(x, **options)
    norm = torch.linalg.norm(value)
    rounded = orthogonalize(x, rounding=halves(1 if x.dtype == torch.bfloat16 and min(x.shape) > 64 else 2), **options)
    held = orthogonalize(x, rounding=lambda t: t.float().double(), **options)
    sums = steps_in_float32(x, **options)
    off = sum(torch.linalg.norm(t.double() - value) for t in (rounded, held, sums)) * 2 / norm if norm > 0 else 0.0
    return value, float(off) + unit(x.dtype) + 16 * F


def steps_in_float32(x, steps=5, coefficients=None, eps=1e-7, scale=1.0):
    x = x.double()
    turned = x.shape[0] > x.shape[1]
    if turned:
        x = x.T
    x = (x / (torch.linalg.norm(x) + eps)).float()
    for i in range(steps):
        a, b, c = QUINTIC if coefficients is None else coefficients[i]
        gram = x @ x.T
        x = a * x + (b * gram + c * gram @ gram) @ x
    return scale * (x.T if turned else x)


def finite_difference(f, x, d, step=1e-6):
    return (f(x + step * d) - f(x - step * d)) / (2 * step)


assert math.isfinite(F)


def light_rows(hidden, weight, targets, lse, dloss, scale=1.0, softcap=0.0, old=None):
    """loss_backward of float16 with what dweight's hidden states are held to as operands: times the power of two of their dloss,
    below 2^15 by the largest such product, so off by half of 2^-24 there, 2^-40 of it, and twice that for each of the two powers."""
    assert hidden.dtype == torch.float16
    got = loss_backward(hidden, weight, targets, lse, dloss, scale, softcap, old)
    inside = (targets >= 0) & (targets < len(weight))
    factor = torch.where(inside, dloss.double().abs() * scale, torch.zeros_like(dloss, dtype=torch.float64))[:, None]
    counted = torch.where(inside[:, None], hidden, torch.zeros_like(hidden))
    z, _, slope, _ = _logits(counted, weight, scale, softcap)
    hot = torch.zeros_like(z).scatter_(1, targets.clamp(0, len(weight) - 1)[:, None], 1.0)
    soft = torch.exp(z - torch.where(inside, lse, torch.zeros_like(lse)).double()[:, None]) * (1 - hot) * slope * (factor > 0)
    stated = soft.T @ (2.0 ** -24 * (counted != 0).double()) * factor.max()  # loss_backward's bound of the same
    held = soft.sum(dim=0)[:, None] * (factor * counted.double().abs().amax(dim=1, keepdim=True)).max() * 2.0 ** -38
    value, bound = got["dweight"]
    return dict(got, dweight=(value, bound + (held - stated) * (1 + unit(hidden.dtype))))
