"""Operators of a decoder layer fine-tuned on packed documents, on data in GPU memory: attention within documents, rotary
positions of several axes, and the norms around a residual addition, each with its gradient.

A case is a dict of plain values; its "op" names the operator, its "dtype" the type of the activations. Parameters
(norm weights, channel gates, ALiBi slopes) and their gradients are float32. The sizes are those of the models that the
benchmark and the tests use: SmolLM2-135M (hidden 576, 9/3 heads of 64), Qwen2.5-0.5B (896), Qwen2.5-1.5B (1536, 12/2
heads of 128), Qwen3-0.6B (16/8 heads of 128), Gemma-2-2B (2304, 8/4 heads of 256, soft-capped scores) and OLMo-2-1B
(2048).

With `own` false, `run` computes the operators from elementary torch operations in 32 bits (rotary angles in 64) and
rounds once at the end; with `own` true it calls the library's entry points.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

# ---- the cases ----


def _attention(name, op, dtype, documents, heads, kv_heads, head_dim, causal=True, window=0, prefix="", softcap=0.0,
               alibi=False):
    return dict(name=name, op=op, dtype=dtype, documents=documents, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                causal=causal, window=window, prefix=prefix, softcap=softcap, alibi=alibi)


def listed() -> list[dict]:
    return [
        # an evaluation of one short answer: the smallest call, where latency counts
        _attention("attention_short", "attention", "bfloat16", "37", 9, 3, 64),
        # a packed training batch of instruction documents of unequal lengths
        _attention("attention_packed", "attention", "bfloat16", "1531,64,803,1,290,511,2048,896,129,1919", 16, 8, 128),
        # a long document in a windowed, soft-capped layer with wide heads
        _attention("attention_capped", "attention", "bfloat16", "8000,192", 8, 4, 256, window=4096, softcap=50.0),
        # float32 documents with distance biases, each with an instruction that every token sees
        _attention("attention_bias_f32", "attention", "float32", "700,1024,33,291", 12, 2, 128, prefix="200,64,33,0",
                   alibi=True),
        # the gradients of a small model's four windows in float32
        _attention("attention_backward_windows", "attention_backward", "float32", "256,256,256,256", 9, 3, 64),
        # the gradients of the packed batch above
        _attention("attention_backward_packed", "attention_backward", "bfloat16",
                   "1531,64,803,1,290,511,2048,896,129,1919", 16, 8, 128),
        # the largest: the gradients of one long document whose first part (an image, a passage) every token sees
        _attention("attention_backward_long", "attention_backward", "float16", "8191", 12, 2, 128, prefix="1200"),
        # one new token's queries and keys
        dict(name="rope_token", op="rope", dtype="bfloat16", tokens=1, heads=16, kv_heads=8, head_dim=128, pairs=64,
             interleaved=False, inverse=False, spread="sections"),
        # a batch of text and images, backward: the gradients of the rotated queries and keys
        dict(name="rope_batch_backward", op="rope", dtype="bfloat16", tokens=16384, heads=12, kv_heads=2, head_dim=128,
             pairs=64, interleaved=False, inverse=True, spread="sections"),
        # one window between two layers, pre-norm with a residual multiplier
        dict(name="norm_window", op="norm", dtype="float32", rows=257, dim=896, placement=0, gate=0, unit_offset=False,
             scale=0.22),
        # a batch between two layers with sandwich norms of unit offset
        dict(name="norm_batch_backward", op="norm_backward", dtype="bfloat16", rows=8192, dim=2304, placement=2, gate=0,
             unit_offset=True, scale=1.0),
        # a ragged batch of a post-norm model with a learned gate for each channel
        dict(name="norm_gated_backward", op="norm_backward", dtype="float32", rows=4099, dim=2048, placement=2, gate=1,
             unit_offset=False, scale=0.5),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))), lo), hi)


def _draw_attention(rng) -> dict:
    op = rng.choice(["attention", "attention_backward"])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4])
    # most models have heads of 64, 128 or 256; every fourth draw takes any size
    head_dim = rng.choice([64, 128, 128, 256]) if rng.random() < 0.75 else rng.randint(8, 256)
    total = _log_int(rng, 1, 8192)
    while heads * head_dim * total ** 2 > 12 * 128 * 8191 ** 2:
        total //= 2
    left, lengths = total, []
    while left:  # up to a dozen documents of unequal lengths
        n = left if len(lengths) == 11 else min(left, _log_int(rng, 1, total))
        lengths.append(n)
        left -= n
    rng.shuffle(lengths)
    prefix = ",".join(str(rng.randint(0, n)) for n in lengths) if rng.random() < 0.3 else ""
    case = _attention("", op, rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), ",".join(map(str, lengths)),
                      heads, kv, head_dim, causal=rng.random() < 0.8,
                      window=_log_int(rng, 1, 4096) if rng.random() < 0.3 else 0, prefix=prefix,
                      softcap=rng.choice([20.0, 50.0]) if rng.random() < 0.3 else 0.0, alibi=rng.random() < 0.25)
    del case["name"]
    return case


def draw(rng) -> dict:
    """A case of the same ranges: one token to a batch, odd and ragged lengths, every type, mask, gate and direction."""
    kind = rng.random()
    if kind < 0.5:
        return _draw_attention(rng)
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind < 0.7:
        head_dim = rng.choice([64, 96, 128, 256]) if rng.random() < 0.75 else rng.randint(8, 256)
        pairs = head_dim // 2 if rng.random() < 0.7 else rng.randint(1, head_dim // 2)
        kv = rng.choice([1, 2, 4, 8])
        return dict(op="rope", dtype=dtype, tokens=_log_int(rng, 1, 16384), heads=kv * rng.choice([1, 2, 3]),
                    kv_heads=kv, head_dim=head_dim, pairs=pairs, interleaved=rng.random() < 0.3,
                    inverse=rng.random() < 0.5, spread=rng.choice(["sections", "strided"]))
    dim = 32 * _log_int(rng, 2, 256) if rng.random() < 0.75 else _log_int(rng, 17, 8192)
    rows = _log_int(rng, 1, 16384)
    while rows * dim > 8192 * 4096:
        rows //= 2
    return dict(op=rng.choice(["norm", "norm_backward"]), dtype=dtype, rows=rows, dim=dim,
                placement=rng.choice([0, 1, 2]), gate=rng.choice([0, 1, 2]), unit_offset=rng.random() < 0.5,
                scale=rng.choice([1.0, 0.22, 0.5]))


def _ints(text: str) -> list[int]:
    return [int(n) for n in text.split(",")] if text else []


# ---- inputs ----

EPS = 1e-6
THETA = 1e6


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale: float = 1.0) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _media_positions(g, tokens: int) -> torch.Tensor:
    """int64 [3, tokens]: spans of text, where time, height and width advance together, and images of a 24-column grid,
    where time stands still; each starts after the largest position before it, deep in a long context."""
    t = torch.arange(tokens, device="cuda")
    offset = int(torch.randint(0, 100000, (1,), generator=g, device="cuda"))
    span, inside = t // 480, t % 480  # 480 tokens of text, then an image of 20 x 24, in turn
    image = span % 2 == 1
    start = offset + (span // 2) * (480 + 24) + torch.where(image, 480, 0)
    axes = [torch.where(image, torch.zeros_like(t), inside), torch.where(image, inside // 24, inside),
            torch.where(image, inside % 24, inside)]
    return torch.stack([start + a for a in axes]).contiguous()


def _inputs(case: dict, seed: int) -> dict:
    g, op, dt = _gen(seed), case["op"], DTYPES[case["dtype"]]
    if op in ("attention", "attention_backward"):
        lengths = _ints(case["documents"])
        t, h, kv, hd = sum(lengths), case["heads"], case["kv_heads"], case["head_dim"]
        s = dict(q=_randn(g, t, h, hd, scale=1.5).to(dt), k=_randn(g, t, kv, hd).to(dt), v=_randn(g, t, kv, hd).to(dt),
                 offsets=torch.tensor([0, *np.cumsum(lengths).tolist()], dtype=torch.int64, device="cuda"),
                 prefix=torch.tensor(_ints(case["prefix"]), dtype=torch.int64, device="cuda") if case["prefix"] else None,
                 slopes=2.0 ** (-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h)
                 if case["alibi"] else None)
        if op == "attention_backward":
            # upstream gradients: the tokens of unequal size
            s["dout"] = (_randn(g, t, h, hd, scale=0.1) * torch.exp(0.5 * _randn(g, t, 1, 1))).to(dt)
        return s
    if op == "rope":
        t, pairs = case["tokens"], case["pairs"]
        i = torch.arange(pairs, device="cuda")
        # which axis turns a pair: three sections of the pairs in order, or one axis after the other
        axis = torch.clamp(i * 3 // max(pairs, 1), max=2) if case["spread"] == "sections" else i % 3
        return dict(q=_randn(g, t, case["heads"], case["head_dim"]).to(dt),
                    k=_randn(g, t, case["kv_heads"], case["head_dim"]).to(dt), positions=_media_positions(g, t),
                    inv_freq=THETA ** (-i.double() / max(pairs, 1)), pair_axis=axis.to(torch.uint8))
    rows, dim = case["rows"], case["dim"]
    # a residual stream whose channels have unequal sizes, and a block's smaller output
    s = dict(x=(_randn(g, rows, dim, scale=2.0) * torch.exp(0.5 * _randn(g, dim))).to(dt),
             y=(_randn(g, rows, dim, scale=0.5) * torch.exp(0.5 * _randn(g, rows, 1))).to(dt))
    centre = 0.0 if case["unit_offset"] else 1.0
    s["post_weight"] = centre + _randn(g, dim, scale=0.1) if case["placement"] != 0 else None
    s["pre_weight"] = centre + _randn(g, dim, scale=0.1) if case["placement"] != 1 else None
    s["gate"] = None if case["gate"] == 0 else 0.5 + _randn(g, dim, scale=0.1) if case["gate"] == 1 else \
        torch.sigmoid(_randn(g, rows, dim)).to(dt)
    if op == "norm_backward":
        s["dh"] = (_randn(g, rows, dim, scale=1e-2) * torch.exp(0.5 * _randn(g, rows, 1))).to(dt)
        s["dn"] = (_randn(g, rows, dim, scale=1e-2) * torch.exp(0.5 * _randn(g, rows, 1))).to(dt) \
            if case["placement"] != 1 else None
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    op = case["op"]
    s.update(op=op, case=case)
    if op == "attention_backward":
        # what the forward pass left: its output and the logarithm of each row's sum
        out, lse = _attention_forward(s)
        s["out"], s["lse"] = out.to(s["q"].dtype), lse
        del out, lse
        s["dq"], s["dk"], s["dv"] = (torch.zeros_like(s[n]) for n in "qkv")
    elif op == "attention":
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(s["q"].shape[1], s["q"].shape[0], device="cuda")
    elif op == "rope":
        s["q_out"], s["k_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
    elif op == "norm":
        s["h"], s["n"] = torch.zeros_like(s["x"]), torch.zeros_like(s["x"]) if case["placement"] != 1 else None
    else:
        s["h"] = s.pop("x")
        s["dx"], s["dy"] = torch.zeros_like(s["h"]), torch.zeros_like(s["y"])
        for name, of in (("dgate", "gate"), ("dpost_weight", "post_weight"), ("dpre_weight", "pre_weight")):
            s[name] = None if s[of] is None else torch.zeros_like(s[of])
    if own:
        _plan(s)
    return s


def _plan(s: dict) -> None:
    """The shape that a program states once, and the workspace that it keeps."""
    from etalii_dllm_amd import kernels as K

    c, op = s["case"], s["op"]
    dtype = K.DTYPES[c["dtype"]]
    nbytes = 0
    if op in ("attention", "attention_backward"):
        s["shape"] = K.DocumentAttention(dtype, s["q"].shape[0], s["offsets"].numel() - 1, c["heads"], c["kv_heads"],
                                         c["head_dim"], int(c["causal"]), c["window"], 1.0 / math.sqrt(c["head_dim"]),
                                         c["softcap"])
        nbytes = getattr(K.lib, f"dllm_hip_document_{op}_workspace")(s["shape"])
    elif op == "rope":
        s["shape"] = K.RopeAxes(dtype, c["tokens"], c["heads"], c["kv_heads"], c["head_dim"], c["pairs"], 3,
                                int(c["interleaved"]), int(c["inverse"]))
    else:
        s["shape"] = K.ResidualNorm(dtype, c["rows"], c["dim"], c["placement"], c["gate"], int(c["unit_offset"]), EPS,
                                    c["scale"])
        if op == "norm_backward":
            nbytes = K.lib.dllm_hip_residual_norm_backward_workspace(s["shape"])
    s["workspace"] = torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device="cuda")


# ---- the plain forms ----


def _visible(s: dict) -> torch.Tensor:
    """[tokens, tokens]: whether a row's query sees a column's key."""
    c, offsets = s["case"], s["offsets"]
    t = torch.arange(s["q"].shape[0], device="cuda")
    doc = torch.searchsorted(offsets, t, right=True) - 1
    away = t[:, None] - t[None, :]
    seen = away >= 0 if c["causal"] else torch.ones_like(away, dtype=torch.bool)
    if c["window"]:
        seen = seen & (away.abs() < c["window"])
    if s["prefix"] is not None:
        seen = seen | (t < offsets[doc] + s["prefix"][doc])[None, :]
    return seen & (doc[:, None] == doc[None, :])


def _scores(s: dict):
    """Scores [heads, tokens, tokens] in 32 bits, hidden keys at minus infinity; the slope of the cap at each."""
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    q = s["q"].float().transpose(0, 1)
    k = s["k"].float().repeat_interleave(group, dim=1).transpose(0, 1)
    x = torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(c["head_dim"]))
    slope = None
    if c["softcap"]:
        tanh = torch.tanh(x / c["softcap"])
        x, slope = c["softcap"] * tanh, 1.0 - tanh * tanh
    if s["slopes"] is not None:
        t = torch.arange(x.shape[1], device="cuda")
        x = x - s["slopes"][:, None, None] * (t[:, None] - t[None, :]).abs()
    return x.masked_fill(~_visible(s), -math.inf), slope


def _attention_forward(s: dict):
    """(out [tokens, heads, head_dim] in 32 bits, lse [heads, tokens])."""
    x, _ = _scores(s)
    top = x.amax(dim=2, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(dim=2, keepdim=True)
    v = s["v"].float().repeat_interleave(s["case"]["heads"] // s["case"]["kv_heads"], dim=1).transpose(0, 1)
    out = torch.matmul(p, v) / total
    return out.transpose(0, 1).contiguous(), (top + torch.log(total)).squeeze(2)


def _attention_backward(s: dict):
    c = s["case"]
    t, h, hd = s["q"].shape
    kv, group, scale = c["kv_heads"], h // c["kv_heads"], 1.0 / math.sqrt(hd)
    x, slope = _scores(s)
    p = torch.exp(x - s["lse"][:, :, None])
    del x
    q, dout, out = (s[n].float().transpose(0, 1) for n in ("q", "dout", "out"))
    k, v = (s[n].float().repeat_interleave(group, dim=1).transpose(0, 1) for n in "kv")
    dp = torch.matmul(dout, v.transpose(1, 2))
    ds = p * (dp - (dout * out).sum(dim=2, keepdim=True))
    del dp
    ds = ds * (slope * scale) if slope is not None else ds * scale
    dq = torch.matmul(ds, k).transpose(0, 1)
    dk = torch.matmul(ds.transpose(1, 2), q).view(kv, group, t, hd).sum(dim=1).transpose(0, 1)
    dv = torch.matmul(p.transpose(1, 2), dout).view(kv, group, t, hd).sum(dim=1).transpose(0, 1)
    dt = s["q"].dtype
    return dict(dq=dq.contiguous().to(dt), dk=dk.contiguous().to(dt), dv=dv.contiguous().to(dt))


def _rope(s: dict):
    c = s["case"]
    pairs, rot = c["pairs"], 2 * c["pairs"]
    angle = s["positions"].double()[s["pair_axis"].long()].T * s["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    sin = -sin if c["inverse"] else sin

    def turn(x):
        a, rest = x[..., :rot].float(), x[..., rot:]
        first, second = (a[..., 0::2], a[..., 1::2]) if c["interleaved"] else (a[..., :pairs], a[..., pairs:])
        one, two = first * cos - second * sin, second * cos + first * sin
        turned = torch.stack([one, two], dim=-1).flatten(-2) if c["interleaved"] else torch.cat([one, two], dim=-1)
        return torch.cat([turned.to(x.dtype), rest], dim=-1)

    return dict(q=turn(s["q"]), k=turn(s["k"]))


def _weight(w, c):
    return 1.0 + w if c["unit_offset"] else w


def _norm(s: dict):
    c, dt = s["case"], s["x"].dtype
    z = s["y"].float()
    if s["post_weight"] is not None:
        z = z * torch.rsqrt(z.square().mean(dim=1, keepdim=True) + EPS) * _weight(s["post_weight"], c)
    if s["gate"] is not None:
        z = z * s["gate"].float()
    h = s["x"].float() + c["scale"] * z
    if s["pre_weight"] is None:
        return dict(h=h.to(dt))
    n = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * _weight(s["pre_weight"], c)
    return dict(h=h.to(dt), n=n.to(dt))


def _norm_backward(s: dict):
    c, dt = s["case"], s["h"].dtype
    g, got = s["dh"].float(), {}

    def through(x, dout, weight):
        """(dx, dweight) of x / rms(x) * weight."""
        r = torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS)
        hat, d = x * r, dout * _weight(weight, c)
        return r * (d - hat * (d * hat).mean(dim=1, keepdim=True)), (dout * hat).sum(dim=0)

    if s["pre_weight"] is not None:
        dx, got["dpre_weight"] = through(s["h"].float(), s["dn"].float(), s["pre_weight"])
        g = g + dx
    got["dx"] = g.to(dt)
    z = y = s["y"].float()
    if s["post_weight"] is not None:
        z = y * torch.rsqrt(y.square().mean(dim=1, keepdim=True) + EPS) * _weight(s["post_weight"], c)
    dz = c["scale"] * g
    if c["gate"] == 1:
        got["dgate"] = (dz * z).sum(dim=0)
    elif c["gate"] == 2:
        got["dgate"] = (dz * z).to(dt)
    if c["gate"]:
        dz = dz * s["gate"].float()
    if s["post_weight"] is not None:
        dz, got["dpost_weight"] = through(y, dz, s["post_weight"])
    got["dy"] = dz.to(dt)
    return got


# ---- one pass ----


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(s: dict):
    from etalii_dllm_amd import kernels as K

    op, shape, ws, stream = s["op"], s["shape"], s["workspace"], torch.cuda.current_stream().cuda_stream
    if op == "attention":
        K.check(K.lib.dllm_hip_document_attention(
            shape, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["offsets"].data_ptr(), _ptr(s["prefix"]),
            _ptr(s["slopes"]), s["out"].data_ptr(), s["lse"].data_ptr(), ws.data_ptr(), ws.numel(), stream))
        return dict(out=s["out"], lse=s["lse"])
    if op == "attention_backward":
        K.check(K.lib.dllm_hip_document_attention_backward(
            shape, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["offsets"].data_ptr(), _ptr(s["prefix"]),
            _ptr(s["slopes"]), s["out"].data_ptr(), s["lse"].data_ptr(), s["dout"].data_ptr(), s["dq"].data_ptr(),
            s["dk"].data_ptr(), s["dv"].data_ptr(), ws.data_ptr(), ws.numel(), stream))
        return dict(dq=s["dq"], dk=s["dk"], dv=s["dv"])
    if op == "rope":
        K.check(K.lib.dllm_hip_rope_axes(
            shape, s["q"].data_ptr(), s["k"].data_ptr(), s["positions"].data_ptr(), s["inv_freq"].data_ptr(),
            s["pair_axis"].data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr(), stream))
        return dict(q=s["q_out"], k=s["k_out"])
    if op == "norm":
        K.check(K.lib.dllm_hip_residual_norm(
            shape, s["x"].data_ptr(), s["y"].data_ptr(), _ptr(s["gate"]), _ptr(s["post_weight"]),
            _ptr(s["pre_weight"]), s["h"].data_ptr(), _ptr(s["n"]), stream))
        return dict(h=s["h"]) if s["n"] is None else dict(h=s["h"], n=s["n"])
    K.check(K.lib.dllm_hip_residual_norm_backward(
        shape, s["h"].data_ptr(), s["y"].data_ptr(), _ptr(s["gate"]), _ptr(s["post_weight"]), _ptr(s["pre_weight"]),
        s["dh"].data_ptr(), _ptr(s["dn"]), s["dx"].data_ptr(), s["dy"].data_ptr(), _ptr(s["dgate"]),
        _ptr(s["dpost_weight"]), _ptr(s["dpre_weight"]), ws.data_ptr(), ws.numel(), stream))
    return {n: s[n] for n in ("dx", "dy", "dgate", "dpost_weight", "dpre_weight") if s[n] is not None}


def run(state: dict):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "attention":
        out, lse = _attention_forward(state)
        return dict(out=out.to(state["q"].dtype), lse=lse)
    return {"attention_backward": _attention_backward, "rope": _rope, "norm": _norm,
            "norm_backward": _norm_backward}[op](state)


# ---- what a pass cannot do without ----


def _pairs(case: dict) -> int:
    """Visible (query, key) pairs of one head."""
    lengths = _ints(case["documents"])
    total = 0
    for n, fixed in zip(lengths, _ints(case["prefix"]) or [0] * len(lengths)):
        i = np.arange(n, dtype=np.int64)
        w = case["window"] or n
        low = np.maximum(i - w + 1, 0)
        high = i + 1 if case["causal"] else np.minimum(i + w, n)
        fixed = min(fixed, n)
        # [low, high) joined with [0, fixed)
        total += int((np.maximum(high - np.maximum(low, fixed), 0) + fixed).sum())
    return total


def work(case: dict) -> dict:
    op, size = case["op"], 4 if case["dtype"] == "float32" else 2
    if op in ("attention", "attention_backward"):
        t, h, kv, hd = sum(_ints(case["documents"])), case["heads"], case["kv_heads"], case["head_dim"]
        q, k = t * h * hd * size, t * kv * hd * size
        pairs = h * _pairs(case)
        if op == "attention":  # q, k, v in; out and lse out; two products
            return dict(bytes=2 * q + 2 * k + 4 * h * t, flops=4 * hd * pairs)
        # q, k, v, out, dout, lse in; dq, dk, dv out; five products
        return dict(bytes=4 * q + 4 * k + 4 * h * t, flops=10 * hd * pairs)
    if op == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return dict(bytes=2 * n * case["head_dim"] * size + 24 * case["tokens"], flops=6 * n * case["pairs"])
    n = case["rows"] * case["dim"]
    element = n * size * (case["gate"] == 2)
    if op == "norm":  # x, y (and gates) in; h (and the normalised h) out
        return dict(bytes=n * size * (3 if case["placement"] == 1 else 4) + element, flops=10 * n)
    # h, y, dh (and dn) in; dx and dy out; gates in and their gradients out
    return dict(bytes=n * size * (5 if case["placement"] == 1 else 6) + 2 * element, flops=25 * n)


# ---- the definitions in 64 bits ----


def _exact_attention(case: dict, s: dict, backward: bool):
    lengths = _ints(case["documents"])
    fixed = _ints(case["prefix"]) or [0] * len(lengths)
    h, hd = case["heads"], case["head_dim"]
    group, scale = h // case["kv_heads"], 1.0 / math.sqrt(hd)
    names = ("dq", "dk", "dv") if backward else ("out",)
    like = dict(dq="q", dk="k", dv="v", out="q")
    got = {n: torch.zeros(s[like[n]].shape, dtype=torch.float64, device="cuda") for n in names}
    if not backward:
        got["lse"] = torch.zeros(h, sum(lengths), dtype=torch.float64, device="cuda")
    begin = 0
    for n, f in zip(lengths, fixed):
        rows = slice(begin, begin + n)
        i = torch.arange(n, device="cuda")
        distance = (i.view(-1, 1) - i.view(1, -1))
        hidden = distance < 0 if case["causal"] else torch.zeros(n, n, dtype=torch.bool, device="cuda")
        if case["window"]:
            hidden |= distance.abs() >= case["window"]
        hidden[:, :f] = False
        for head in range(h):
            q, k, v = s["q"][rows, head].double(), s["k"][rows, head // group].double(), \
                s["v"][rows, head // group].double()
            z = (q @ k.t()) * scale
            slope = None
            if case["softcap"]:
                slope = 1.0 / torch.cosh(z / case["softcap"]).square()
                z = case["softcap"] * torch.tanh(z / case["softcap"])
            if s["slopes"] is not None:
                z -= float(s["slopes"][head]) * distance.abs()
            z[hidden] = -math.inf
            if not backward:
                got["lse"][head, rows] = torch.logsumexp(z, dim=1)
                got["out"][rows, head] = torch.softmax(z, dim=1) @ v
                continue
            # the forward's row sums and outputs are inputs of the gradient
            p = torch.exp(z - s["lse"][head, rows].double()[:, None])
            do = s["dout"][rows, head].double()
            got["dv"][rows, head // group] += p.t() @ do
            dz = p * (do @ v.t() - (do * s["out"][rows, head].double()).sum(dim=1, keepdim=True)) * scale
            if slope is not None:
                dz *= slope
            got["dq"][rows, head] = dz @ k
            got["dk"][rows, head // group] += dz.t() @ q
        begin += n
    return got


def _exact_rope(case: dict, s: dict):
    pairs = case["pairs"]
    axis = s["pair_axis"].long()
    turns = torch.stack([s["positions"][int(a)].double() * s["inv_freq"][i] for i, a in enumerate(axis)], dim=1)
    turn = torch.polar(torch.ones_like(turns), -turns if case["inverse"] else turns)[:, None, :]
    got = {}
    for name in "qk":
        x = s[name].double().clone()
        at = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if case["interleaved"] else \
            (slice(0, pairs), slice(pairs, 2 * pairs))
        z = torch.complex(x[..., at[0]], x[..., at[1]]) * turn
        x[..., at[0]], x[..., at[1]] = z.real, z.imag
        got[name] = x
    return got


def _exact_norm(case: dict, s: dict, backward: bool):
    """Forward as defined; the gradients through torch's differentiation of the definition in 64 bits."""
    w = {n: None if s[n] is None else s[n].double().requires_grad_(backward) for n in ("post_weight", "pre_weight", "gate")}
    offset = 1.0 if case["unit_offset"] else 0.0

    def rms(x, weight):
        return x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPS) * (offset + weight)

    def branch(y):
        z = y if w["post_weight"] is None else rms(y, w["post_weight"])
        return case["scale"] * (z if w["gate"] is None else z * w["gate"])

    y = s["y"].double().requires_grad_(backward)
    if not backward:
        h = s["x"].double() + branch(y)
        return dict(h=h) if w["pre_weight"] is None else dict(h=h, n=rms(h, w["pre_weight"]))
    h = s["x"].double().requires_grad_()
    got, g = {}, s["dh"].double()
    if w["pre_weight"] is not None:
        dx, got["dpre_weight"] = torch.autograd.grad(rms(h, w["pre_weight"]), (h, w["pre_weight"]), s["dn"].double())
        g = g + dx
    got["dx"] = g
    wanted = {"dy": y, "dgate": w["gate"], "dpost_weight": w["post_weight"]}
    wanted = {n: t for n, t in wanted.items() if t is not None}
    got.update(zip(wanted, torch.autograd.grad(branch(y), list(wanted.values()), g)))
    return got


def exact(case: dict, seed: int):
    s, op = _inputs(case, seed), case["op"]
    if op == "attention":
        return _exact_attention(case, s, False)
    if op == "attention_backward":
        # the outputs and row sums that prepare() hands over, made again as it makes them
        out, s["lse"] = _attention_forward({**s, "case": case})
        s["out"] = out.to(s["q"].dtype)
        del out
        return _exact_attention(case, s, True)
    if op == "rope":
        return _exact_rope(case, s)
    return _exact_norm(case, s, op == "norm_backward")
