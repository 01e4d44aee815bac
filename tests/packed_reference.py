"""The packed-layer operators' definitions in 64 bits, and how far a correct kernel's results may be from them.

Every bound is an absolute one per element, from the number of roundings: an activation type rounds by at most
u = eps / 2 of the value, float32 by F = 2^-24, and a sum of n terms in float32 (any order) is off by at most n F times
the sum of the terms' magnitudes. The magnitudes (sums of absolute values) are formed here beside the results.
"""

from __future__ import annotations

import math

import torch

F = 2.0 ** -24
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def unit(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half the distance of the smallest subnormals: a rounding's error near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def hidden(n: int, causal: bool, window: int, prefix: int) -> torch.Tensor:
    i = torch.arange(n)
    away = i[:, None] - i[None, :]
    out = (away < 0) if causal else torch.zeros(n, n, dtype=torch.bool)
    if window:
        out |= away.abs() >= window
    out[:, :prefix] = False
    return out


def attention(q, k, v, offsets, scale, causal=True, window=0, prefix=None, softcap=0.0, slopes=None, out=None,
              lse=None, dout=None):
    """Results and bounds of the forward, or with dout of the backward, as dicts of (value, bound). Tokens of no document
    are zero with bound 0. Inputs in their type, on any device; computed in float64 there."""
    dt, dev = q.dtype, q.device
    u = unit(dt)
    up = 0.0 if dt == torch.float32 else u  # probabilities and dS are rounded to the type for the second product
    heads, hd = q.shape[1], q.shape[2]
    group = heads // k.shape[1]
    names = {"out": q} if dout is None else {"dq": q, "dk": k, "dv": v}
    got = {n: torch.zeros(t.shape, dtype=torch.float64, device=dev) for n, t in names.items()}
    mag = {n: torch.zeros(t.shape, dtype=torch.float64, device=dev) for n, t in names.items()}
    if dout is None:
        got["lse"] = torch.zeros(heads, q.shape[0], dtype=torch.float64, device=dev)
        mag["lse"] = torch.zeros_like(got["lse"])
    offsets = [int(o) for o in offsets]
    for d, (b, e) in enumerate(zip(offsets, offsets[1:])):
        n = e - b
        if n == 0:
            continue
        mask = hidden(n, causal, window, 0 if prefix is None else min(max(int(prefix[d]), 0), n)).to(dev)
        i = torch.arange(n, device=dev)
        distance = (i[:, None] - i[None, :]).abs().double()
        for h in range(heads):
            # hidden rows' contents count for nothing: they are left out of the products below by zeroes there
            Q, K, V = q[b:e, h].double(), k[b:e, h // group].double(), v[b:e, h // group].double()
            x = Q @ K.T * scale
            # the dot product's error, the cap's (tanh to a few F of its value, at most 8 F cap) and the bias's rounding
            err = (hd + 4) * F * (Q.abs() @ K.abs().T) * abs(scale)
            slope = torch.ones_like(x)
            if softcap:
                t = torch.tanh(x / softcap)
                x, slope = softcap * t, 1 - t * t
                err = err + 8 * F * softcap
            if slopes is not None:
                x = x - float(slopes[h]) * distance
                err = err + 4 * F * float(slopes[h]) * distance
            err = err + 4 * F * x.abs()
            x = x.masked_fill(mask, -math.inf)
            err = err.masked_fill(mask, 0.0).amax(dim=1, keepdim=True)
            if dout is None:
                s = torch.logsumexp(x, dim=1, keepdim=True)
                p = torch.exp(x - s)
                got["lse"][h, b:e], mag["lse"][h, b:e] = s[:, 0], (err + 4 * F * s.abs() + (n + 8) * F)[:, 0]
                got["out"][b:e, h] = o = p @ V
                # p off by 2 err (its own score and the sum's), rounded once (up; the sum of the rounded or the exact
                # ones: up again), added in float32
                # (and 2^-126 absolutely, where float32 loses its relative precision)
                mag["out"][b:e, h] = u * o.abs() + (~mask).double() @ V.abs() * 2.0 ** -126 + (p @ V.abs()) * (2 * err.expm1() + 2 * up + (2 * n + 16) * F) * (1 + u)
                continue
            s = lse[h, b:e].double()[:, None]
            p = torch.exp(x - s)
            rel = err.expm1() + 4 * F * s.abs() + 8 * F  # of p
            dO, O = dout[b:e, h].double(), out[b:e, h].double()
            dP, delta = dO @ V.T, (dO * O).sum(dim=1, keepdim=True)
            size = dO.abs() @ V.abs().T + (dO.abs() * O.abs()).sum(dim=1, keepdim=True)
            dS = p * (dP - delta) * slope * scale
            # |dS| error: its factors' relative errors, the dot products' absolute ones, the cap derivative's (t off by
            # 8 F and by err / cap)
            dslope = 2 * (8 * F + err / softcap) if softcap else 0.0
            eS = p * size * abs(scale) * (rel + up + (hd + 16) * F + dslope)
            eP = p * (rel + up)
            # float32 keeps its relative precision down to 2^-126 alone: p and dS below that are off by as much, times what
            # they are multiplied by (p below it is exp of less than -87, as in rows that one key takes)
            eP = eP + (~mask) * 2.0 ** -126
            eS = eS + (~mask) * 2.0 ** -126 * (1 + size * abs(scale))
            if dt == torch.float16:
                # rounded as multiples of the smallest float16: p times 2^8, dS relative to dout's largest row too
                eP = eP + (~mask) * 2.0 ** -33
                eS = eS + (~mask) * 2.0 ** -32 * abs(scale) * dO.norm(dim=1).max()
            got["dq"][b:e, h] = dS @ K
            mag["dq"][b:e, h] = u * got["dq"][b:e, h].abs() + (eS @ K.abs() + (2 * n + 8) * F * (dS.abs() @ K.abs())) * (1 + u)
            got["dk"][b:e, h // group] += dS.T @ Q
            mag["dk"][b:e, h // group] += (eS.T @ Q.abs() + (2 * n + 8 + heads) * F * (dS.abs().T @ Q.abs())) * (1 + u)
            got["dv"][b:e, h // group] += p.T @ dO
            mag["dv"][b:e, h // group] += (eP.T @ dO.abs() + (2 * n + 8 + heads) * F * (p.T @ dO.abs())) * (1 + u)
    for n in ("dk", "dv"):
        if n in got:
            mag[n] += u * got[n].abs()
    return {n: (got[n], mag[n] + (0.0 if n == "lse" else tiny(dt))) for n in got}


def rope(x, positions, inv_freq, pair_axis, interleaved, inverse):
    """(value, bound) of one tensor's rotation."""
    pairs = len(inv_freq)
    u = unit(x.dtype)
    angle = positions[pair_axis.long()].double().T * inv_freq.double()  # [tokens, pairs]
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    s = -s if inverse else s
    z = x.double().clone()
    bound = torch.zeros_like(z)
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    first, second = z[..., a].clone(), z[..., b].clone()
    z[..., a], z[..., b] = first * c - second * s, second * c + first * s
    # sine and cosine to 4 F (argument reduced in double, rounded to float32 once: pi F; the function: F), two products
    for part in (a, b):
        bound[..., part] = u * z[..., part].abs() + (first.abs() + second.abs()) * 8 * F * (1 + u) + tiny(x.dtype)
    return z, bound


def residual_norm(x, y, gate, post_weight, pre_weight, placement, eps, unit_offset, scale, dh=None, dn=None):
    """Results and bounds of the forward, or of the backward where x is h and dh or dn are given."""
    u, dim = unit(x.dtype), x.shape[1]
    off = 1.0 if unit_offset else 0.0
    post, pre = placement != 0, placement != 1
    X, Y = x.double(), y.double()
    wp = off + post_weight.double() if post_weight is not None else torch.ones(dim, dtype=torch.float64, device=x.device)
    wn = off + pre_weight.double() if pre_weight is not None else torch.ones(dim, dtype=torch.float64, device=x.device)
    G = gate.double() if gate is not None else torch.ones(dim, dtype=torch.float64, device=x.device)
    R = (dim / 2 + 12) * F  # relative error of 1 / sqrt(mean square + eps): half the sum's, and a few roundings
    ry = 1 / torch.sqrt(Y.square().mean(dim=1, keepdim=True) + eps) if post else torch.ones(len(Y), 1, dtype=torch.float64, device=x.device)
    hat = Y * ry
    z = hat * wp if post else Y
    if dh is None and dn is None:
        h = X + scale * G * z
        eh = (scale * G * z).abs() * (R * post + 8 * F) + 2 * F * h.abs()
        res = {"h": (h, u * h.abs() + eh * (1 + u) + tiny(x.dtype))}
        if pre:
            r = 1 / torch.sqrt(h.square().mean(dim=1, keepdim=True) + eps)
            n = h * r * wn
            # h's error reaches n directly and through the mean square (Cauchy-Schwarz)
            through = (eh.square().sum(dim=1, keepdim=True).sqrt() / math.sqrt(dim)) * r
            en = (r * wn).abs() * eh + n.abs() * (through + R + 8 * F)
            res["n"] = (n, u * n.abs() + en * (1 + u) + tiny(x.dtype))
        return res
    D = dh.double() if dh is not None else torch.zeros_like(X)
    res = {}

    def through(v, r, d):
        """(gradient, bound) of v r for the upstream d: r d - v r^3 mean(d v)."""
        dot, size = (d * v).mean(dim=1, keepdim=True), (d * v).abs().mean(dim=1, keepdim=True)
        value = r * d - v * r ** 3 * dot
        return value, (r * d).abs() * (R + 8 * F) + v.abs() * r ** 3 * (dot.abs() * (3 * R + 8 * F) + size * (dim + 8) * F)

    g, eg = D, torch.zeros_like(D)
    if pre:
        r = 1 / torch.sqrt(X.square().mean(dim=1, keepdim=True) + eps)
        value, err = through(X, r, dn.double() * wn)
        g, eg = D + value, err + 2 * F * (D.abs() + value.abs())
        terms = dn.double() * X * r
        res["dpre_weight"] = (terms.sum(dim=0), terms.abs().sum(dim=0) * (R + (len(X) + 16) * F))
    res["dx"] = (g, u * g.abs() + eg * (1 + u) + tiny(x.dtype))
    dz, ez = scale * g, abs(scale) * (eg + 4 * F * g.abs())
    if gate is not None:
        terms, et = dz * z, ez * z.abs() + (dz * z).abs() * (R * post + 8 * F)
        if gate.dim() == 1:
            res["dgate"] = (terms.sum(dim=0), et.sum(dim=0) + terms.abs().sum(dim=0) * (len(X) + 16) * F)
        else:
            res["dgate"] = (terms, u * terms.abs() + et * (1 + u) + tiny(x.dtype))
    du, eu = dz * G, (ez + 2 * F * dz.abs()) * G.abs()
    if post:
        terms, et = du * hat, eu * hat.abs() + (du * hat).abs() * (R + 8 * F)
        res["dpost_weight"] = (terms.sum(dim=0), et.sum(dim=0) + terms.abs().sum(dim=0) * (len(X) + 16) * F)
        value, err = through(Y, ry, du * wp)
        # du's error reaches dy directly and through the dot product
        err = err + ry * (eu * wp.abs()) + Y.abs() * ry ** 3 * (eu * wp.abs() * Y.abs()).mean(dim=1, keepdim=True)
        du, eu = value, err + 4 * F * value.abs()
    res["dy"] = (du, u * du.abs() + eu * (1 + u) + tiny(x.dtype))
    return res


def assert_within(got: torch.Tensor, want, what: str) -> None:
    value, bound = want
    got = got.double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got - value).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        at = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {got.numel()} outside their bound, first at {at}: "
                             f"{float(got[tuple(at)])} is not {float(value[tuple(at)])} +- {float(bound[tuple(at)])}")
