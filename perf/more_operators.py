"""Operators at both ends of a decoder trained on packed batches, and of its update, on data in GPU memory: the lookup of
tokens in an embedding table and its gradient, the cross-entropy over the vocabulary from the last hidden states and its
gradients, and the orthogonalised update of a weight matrix.

A case is a dict of plain values; its "op" names the operator, its "dtype" the type of activations, tables and updates. The
sizes are those of the models that the benchmark and the tests use: SmolLM2-135M (vocabulary 49152, hidden 576,
intermediate 1536, 3 key heads of 64), Qwen2.5-0.5B (151936, 896, 4864), Qwen2.5-1.5B (151936, 1536, 8960) and Gemma-2-2B
(256000, 2304, logits capped at 30, embeddings times the root of the hidden size).

With `own` false, `run` computes the operators from elementary torch operations in 32 bits and rounds once at the end;
with `own` true it calls the library's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-7
QUINTIC = (3.4445, -4.7750, 2.0315)  # the coefficients that Muon's authors published

# ---- the cases ----


def _embedding(name, op, dtype, tokens, vocabulary, dim, scale=1.0, accumulate=False):
    return dict(name=name, op=op, dtype=dtype, tokens=tokens, vocabulary=vocabulary, dim=dim, scale=scale,
                accumulate=accumulate)


def _loss(name, op, dtype, rows, vocabulary, dim, masked=0.0, scale=1.0, softcap=0.0, accumulate=False):
    return dict(name=name, op=op, dtype=dtype, rows=rows, vocabulary=vocabulary, dim=dim, masked=masked, scale=scale,
                softcap=softcap, accumulate=accumulate)


def _update(name, dtype, batch, rows, cols, steps=5, scale=1.0):
    return dict(name=name, op="orthogonalize", dtype=dtype, batch=batch, rows=rows, cols=cols, steps=steps, scale=scale)


def listed() -> list[dict]:
    return [
        # one new token's embedding: the smallest call, where latency counts
        _embedding("embedding_token", "embedding", "bfloat16", 1, 151936, 896),
        # a packed batch's embeddings, scaled
        _embedding("embedding_batch", "embedding", "bfloat16", 16384, 256000, 2304, scale=48.0),
        # the gradient of a table that nothing else has written
        _embedding("embedding_backward", "embedding_backward", "bfloat16", 8192, 151936, 1536),
        # a small model's windows onto the gradient of a tied table, which holds the loss's part
        _embedding("embedding_backward_tied", "embedding_backward", "float32", 16381, 49152, 576, accumulate=True),
        # an answer of 37 tokens scored
        _loss("loss_answer", "loss", "bfloat16", 37, 151936, 896),
        # a training batch of packed documents
        _loss("loss_batch", "loss", "bfloat16", 8192, 151936, 1536),
        # the gradients of a small model's four windows in float32
        _loss("loss_backward_windows", "loss_backward", "float32", 1020, 49152, 576, scale=0.25),
        # a batch of instructions, whose prompts do not count, with capped logits
        _loss("loss_backward_capped", "loss_backward", "float16", 2047, 256000, 2304, masked=0.4, softcap=30.0),
        # the largest: the gradients of the training batch
        _loss("loss_backward_batch", "loss_backward", "bfloat16", 8192, 151936, 1536),
        # the update of a small model's key projection in float32
        _update("update_small", "float32", 1, 192, 576),
        # one layer's wide projection, taller than wide
        _update("update_layer", "bfloat16", 1, 8960, 1536, scale=0.2 * math.sqrt(8960)),
        # a projection of all layers of a model at once
        _update("update_layers", "bfloat16", 24, 896, 4864, scale=0.2 * math.sqrt(4864)),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))), lo), hi)


def draw(rng) -> dict:
    """A case of the same ranges: one token to a batch, odd and ragged sizes, every type, option and direction."""
    kind = rng.random()
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    # most tables are a model's, every fourth draw takes any size
    if rng.random() < 0.75:
        vocabulary, dim = rng.choice([(49152, 576), (151936, 896), (151936, 1024), (151936, 1536), (100352, 2048),
                                      (256000, 2304)])
    else:
        vocabulary, dim = _log_int(rng, 300, 256000), _log_int(rng, 16, 2304)
    if kind < 0.25:
        return dict(op=rng.choice(["embedding", "embedding_backward"]), dtype=dtype, tokens=_log_int(rng, 1, 32768),
                    vocabulary=vocabulary, dim=dim, scale=rng.choice([1.0, 12.0, math.sqrt(dim)]),
                    accumulate=rng.random() < 0.5)
    if kind < 0.65:
        rows = _log_int(rng, 1, 8192)
        most = 8192 * 151936 * 1536 // (6 if dtype == "float32" else 1)
        while rows * vocabulary * dim > most:
            rows //= 2
        return dict(op=rng.choice(["loss", "loss_backward"]), dtype=dtype, rows=rows, vocabulary=vocabulary, dim=dim,
                    masked=rng.choice([0.0, 0.3, 0.6]), scale=rng.choice([1.0, 1.0, 0.25]),
                    softcap=rng.choice([0.0, 0.0, 30.0]), accumulate=rng.random() < 0.3)
    if rng.random() < 0.75:
        rows, cols = rng.choice([(576, 576), (192, 576), (576, 1536), (896, 896), (896, 4864), (1536, 1536), (256, 1536),
                                 (1536, 8960), (2048, 8192)])
    else:
        rows, cols = _log_int(rng, 1, 2048), _log_int(rng, 1, 8960)
    if rng.random() < 0.5:
        rows, cols = cols, rows
    batch = _log_int(rng, 1, 32)
    while batch > 1 and batch * min(rows, cols) ** 2 * max(rows, cols) > 2 * 24 * 896 ** 2 * 4864:
        batch //= 2
    return dict(op="orthogonalize", dtype=dtype, batch=batch, rows=rows, cols=cols, steps=rng.choice([3, 5, 5, 5, 6]),
                scale=rng.choice([1.0, 0.2 * math.sqrt(max(rows, cols))]))


# ---- inputs ----


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale: float = 1.0) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _tokens(g, n: int, vocabulary: int) -> torch.Tensor:
    """int64 [n]: few tokens often and many seldom, as in text (the k-th most frequent about 1 / k of the time)."""
    rank = torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(vocabulary)).long() - 1
    return rank.clamp(0, vocabulary - 1) * 40503 % vocabulary


def _table(g, vocabulary: int, dim: int, dtype) -> torch.Tensor:
    """An embedding table whose channels have unequal sizes."""
    size = 0.03 * torch.exp(0.3 * _randn(g, dim))
    return torch.randn(vocabulary, dim, generator=g, device="cuda").mul_(size).to(dtype)


def _inputs(case: dict, seed: int) -> dict:
    g, op, dt = _gen(seed), case["op"], DTYPES[case["dtype"]]
    if op in ("embedding", "embedding_backward"):
        t, v, d = case["tokens"], case["vocabulary"], case["dim"]
        s = dict(tokens=_tokens(g, t, v))
        if op == "embedding":
            s["table"] = _table(g, v, d, dt)
        else:
            s["dout"] = (_randn(g, t, d, scale=1e-2) * torch.exp(0.5 * _randn(g, t, 1))).to(dt)
            s["dtable"] = (_randn(g, v, d, scale=1e-2)).to(dt) if case["accumulate"] else \
                torch.zeros(v, d, dtype=dt, device="cuda")
        return s
    if op in ("loss", "loss_backward"):
        t, v, d = case["rows"], case["vocabulary"], case["dim"]
        s = dict(weight=_table(g, v, d, dt), targets=_tokens(g, t, v))
        # a trained model's states: normed, and turned towards the token that comes, sure of it or less so
        toward = s["weight"][s["targets"]].float()
        toward = toward / toward.square().sum(dim=1, keepdim=True)
        sure = 16.0 * torch.rand(t, 1, generator=g, device="cuda") / case["scale"]
        s["hidden"] = (_randn(g, t, d, scale=1.2) + sure * toward).to(dt)
        kept = torch.arange(t, device="cuda") % 256 >= round(256 * case["masked"])  # each sequence's prompt does not count
        s["targets"] = torch.where(kept, s["targets"], torch.full_like(s["targets"], -100))
        if op == "loss_backward":
            # the mean over the tokens that count, documents of unequal weight
            weight = torch.exp(0.3 * _randn(g, t))
            s["dloss"] = weight / max(round(t * (1.0 - case["masked"])), 1)
            s["dweight"] = _randn(g, v, d, scale=1e-4).to(dt) if case["accumulate"] else \
                torch.zeros(v, d, dtype=dt, device="cuda")
        return s
    # a momentum: a few strong directions over much noise
    b, m, n = case["batch"], case["rows"], case["cols"]
    r = min(8, m, n)
    x = _randn(g, b, m, n)
    x += torch.matmul(_randn(g, b, m, r) * torch.linspace(8.0, 1.0, r, device="cuda"), _randn(g, b, r, n))
    return dict(x=(x * 1e-3).to(dt))


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    op = case["op"]
    s.update(op=op, case=case)
    if op == "embedding":
        s["out"] = torch.zeros(case["tokens"], case["dim"], dtype=s["table"].dtype, device="cuda")
    elif op == "loss":
        s["loss"], s["lse"] = (torch.zeros(case["rows"], device="cuda") for _ in range(2))
    elif op == "loss_backward":
        # what the forward pass left: the logarithm of each row's sum
        s["lse"] = _loss_forward(s)["lse"]
        s["dhidden"] = torch.zeros_like(s["hidden"])
    elif op == "orthogonalize":
        s["out"] = torch.zeros_like(s["x"])
    if own:
        _plan(s)
    return s


def _plan(s: dict) -> None:
    """The shape that a program states once, and the workspace that it keeps."""
    from etalii_dllm_amd import kernels as K

    c, op = s["case"], s["op"]
    dtype = K.DTYPES[c["dtype"]]
    nbytes = 0
    if op in ("embedding", "embedding_backward"):
        s["shape"] = K.TokenEmbedding(dtype, c["tokens"], c["vocabulary"], c["dim"], int(c["accumulate"]), c["scale"])
        if op == "embedding_backward":
            nbytes = K.lib.dllm_hip_token_embedding_backward_workspace(s["shape"])
    elif op in ("loss", "loss_backward"):
        s["shape"] = K.VocabularyLoss(dtype, c["rows"], c["vocabulary"], c["dim"], int(c["accumulate"]), c["scale"],
                                      c["softcap"])
        nbytes = getattr(K.lib, f"dllm_hip_vocabulary_{op}_workspace")(s["shape"])
    else:
        s["shape"] = K.Orthogonalize(dtype, c["batch"], c["rows"], c["cols"], c["steps"], EPS, c["scale"])
        nbytes = K.lib.dllm_hip_orthogonalize_workspace(s["shape"])
    s["workspace"] = torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device="cuda")


# ---- the plain forms ----


def _embedding_forward(s: dict):
    table = s["table"]
    return dict(out=(table[s["tokens"]].float() * s["case"]["scale"]).to(table.dtype))


def _embedding_backward(s: dict):
    d, c = s["dtable"], s["case"]
    total = torch.zeros(d.shape, device="cuda")
    total.index_add_(0, s["tokens"], s["dout"].float())
    total *= c["scale"]
    if c["accumulate"]:
        total += d
    d.copy_(total)
    return dict(dtable=d)


def _logits(s: dict) -> torch.Tensor:
    """Capped logits in 32 bits."""
    c = s["case"]
    z = torch.matmul(s["hidden"].float(), s["weight"].float().t())
    z *= c["scale"]
    if c["softcap"]:
        z = torch.tanh(z.div_(c["softcap"])).mul_(c["softcap"])
    return z


def _loss_forward(s: dict):
    z = _logits(s)
    counts = s["targets"] >= 0
    top = z.amax(dim=1, keepdim=True)
    at = z.gather(1, s["targets"].clamp(min=0)[:, None])[:, 0]
    lse = top[:, 0] + torch.log(torch.exp(z.sub_(top)).sum(dim=1))
    zero = torch.zeros_like(lse)
    return dict(loss=torch.where(counts, lse - at, zero), lse=torch.where(counts, lse, zero))


def _loss_backward(s: dict):
    c, dt = s["case"], s["hidden"].dtype
    z = _logits(s)
    counts = s["targets"] >= 0
    g = torch.exp(z - s["lse"][:, None])
    at = s["targets"].clamp(min=0)[:, None]
    # p - 1 at the target, from the difference of the exponents: p is near 1 there
    target = torch.expm1(z.gather(1, at) - s["lse"][:, None])
    g.scatter_(1, at, target)
    if c["softcap"]:
        g *= 1.0 - (z / c["softcap"]).square()
    del z
    g *= torch.where(counts, s["dloss"] * c["scale"], torch.zeros_like(s["dloss"]))[:, None]
    dhidden = torch.matmul(g, s["weight"].float())
    dweight = torch.matmul(g.t(), s["hidden"].float())
    if c["accumulate"]:
        dweight += s["dweight"]
    s["dweight"].copy_(dweight)
    return dict(dhidden=dhidden.to(dt), dweight=s["dweight"])


def _orthogonalize(s: dict):
    c, (a, b, q) = s["case"], QUINTIC
    x = s["x"].float()
    turned = c["rows"] > c["cols"]
    if turned:
        x = x.transpose(1, 2)
    x = x / (x.square().sum(dim=(1, 2), keepdim=True).sqrt() + EPS)
    for _ in range(c["steps"]):
        gram = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * gram + q * torch.matmul(gram, gram), x)
    x = x * c["scale"]
    if turned:
        x = x.transpose(1, 2)
    return dict(out=x.contiguous().to(s["x"].dtype))


# ---- one pass ----


def _run_own(s: dict):
    from etalii_dllm_amd import kernels as K

    op, shape, ws, stream = s["op"], s["shape"], s["workspace"], torch.cuda.current_stream().cuda_stream
    if op == "embedding":
        K.check(K.lib.dllm_hip_token_embedding(shape, s["table"].data_ptr(), s["tokens"].data_ptr(), s["out"].data_ptr(),
                                               stream))
        return dict(out=s["out"])
    if op == "embedding_backward":
        K.check(K.lib.dllm_hip_token_embedding_backward(shape, s["tokens"].data_ptr(), s["dout"].data_ptr(),
                                                        s["dtable"].data_ptr(), ws.data_ptr(), ws.numel(), stream))
        return dict(dtable=s["dtable"])
    if op == "loss":
        K.check(K.lib.dllm_hip_vocabulary_loss(shape, s["hidden"].data_ptr(), s["weight"].data_ptr(),
                                               s["targets"].data_ptr(), s["loss"].data_ptr(), s["lse"].data_ptr(),
                                               ws.data_ptr(), ws.numel(), stream))
        return dict(loss=s["loss"], lse=s["lse"])
    if op == "loss_backward":
        K.check(K.lib.dllm_hip_vocabulary_loss_backward(
            shape, s["hidden"].data_ptr(), s["weight"].data_ptr(), s["targets"].data_ptr(), s["lse"].data_ptr(),
            s["dloss"].data_ptr(), s["dhidden"].data_ptr(), s["dweight"].data_ptr(), ws.data_ptr(), ws.numel(), stream))
        return dict(dhidden=s["dhidden"], dweight=s["dweight"])
    K.check(K.lib.dllm_hip_orthogonalize(shape, None, s["x"].data_ptr(), s["out"].data_ptr(), ws.data_ptr(), ws.numel(),
                                         stream))
    return dict(out=s["out"])


def run(state: dict):
    if own:
        return _run_own(state)
    return {"embedding": _embedding_forward, "embedding_backward": _embedding_backward, "loss": _loss_forward,
            "loss_backward": _loss_backward, "orthogonalize": _orthogonalize}[state["op"]](state)


# ---- what a pass cannot do without ----


def work(case: dict) -> dict:
    op, size = case["op"], 4 if case["dtype"] == "float32" else 2
    if op == "embedding":
        n = case["tokens"] * case["dim"]
        return dict(bytes=2 * n * size + 8 * case["tokens"], flops=n)
    if op == "embedding_backward":
        t, v, d = case["tokens"], case["vocabulary"], case["dim"]
        # the gradients in; the table out, or the rows of the tokens that occur (of the stated frequencies) in and out
        seen = sum(1.0 - math.exp(-t / (k * math.log(v))) for k in range(1, v + 1)) if case["accumulate"] else 0.0
        return dict(bytes=t * d * size + 8 * t + (2 * seen if case["accumulate"] else v) * d * size, flops=t * d)
    if op in ("loss", "loss_backward"):
        v, d = case["vocabulary"], case["dim"]
        masked = round(256 * case["masked"])
        t = case["rows"] // 256 * (256 - masked) + max(case["rows"] % 256 - masked, 0)  # rows that count
        if op == "loss":
            return dict(bytes=(t + v) * d * size + 16 * case["rows"], flops=2 * t * v * d)
        table = 3 if case["accumulate"] else 2
        return dict(bytes=(t + case["rows"] + table * v) * d * size + 16 * case["rows"], flops=6 * t * v * d)
    m, n = sorted((case["rows"], case["cols"]))
    # of the two symmetric products only one half each
    return dict(bytes=2 * case["batch"] * m * n * size, flops=case["batch"] * case["steps"] * (m * m * n + m ** 3 + 2 * m * m * n))


# ---- the definitions in 64 bits ----


def _exact_loss(case: dict, s: dict, backward: bool):
    w, t = s["weight"].double(), case["rows"]
    if backward:
        got = dict(dhidden=torch.zeros(t, case["dim"], dtype=torch.float64, device="cuda"), dweight=torch.zeros_like(w))
    else:
        got = {n: torch.zeros(t, dtype=torch.float64, device="cuda") for n in ("loss", "lse")}
    rows = torch.nonzero(s["targets"] >= 0)[:, 0]
    for part in rows.split(512):  # only the rows that count
        h, y = s["hidden"][part].double(), s["targets"][part]
        z = case["scale"] * (h @ w.t())
        slope = None
        if case["softcap"]:
            z = z / case["softcap"]
            slope = 1.0 / torch.cosh(z).square() if backward else None
            z = case["softcap"] * torch.tanh(z)
        if not backward:
            got["lse"][part] = torch.logsumexp(z, dim=1)
            got["loss"][part] = -torch.log_softmax(z, dim=1)[torch.arange(len(part), device="cuda"), y]
            continue
        # the forward's logarithm of the sum is an input of the gradient
        e = z - s["lse"][part].double()[:, None]
        at = (torch.arange(len(part), device="cuda"), y)
        target = torch.expm1(e[at])
        g = e.exp_()
        g[at] = target
        if slope is not None:
            g *= slope
        g *= (s["dloss"][part].double() * case["scale"])[:, None]
        got["dhidden"][part] = g @ w
        got["dweight"] += g.t() @ h
    if backward and case["accumulate"]:
        got["dweight"] += s["dweight"].double()
    return got


def exact(case: dict, seed: int):
    s, op = _inputs(case, seed), case["op"]
    if op == "embedding":
        return dict(out=torch.cat([case["scale"] * s["table"][i].double() for i in s["tokens"].split(4096)]))
    if op == "embedding_backward":
        order = torch.argsort(s["tokens"], stable=True)
        ids, counts = torch.unique_consecutive(s["tokens"][order], return_counts=True)
        sums = torch.cumsum(s["dout"][order].double(), dim=0)[torch.cumsum(counts, 0) - 1]
        total = s["dtable"].double()
        total[ids] += case["scale"] * torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1]))
        return dict(dtable=total)
    if op == "loss":
        return _exact_loss(case, s, False)
    if op == "loss_backward":
        s["lse"] = _loss_forward({**s, "case": case})["lse"]  # made again as prepare() makes it
        return _exact_loss(case, s, True)
    # with the smaller side's products, whichever side that is: X p(X^T X) = p(X X^T) X
    a, b, q = QUINTIC
    got = []
    for x in s["x"].double():
        x = x / (torch.linalg.norm(x) + EPS)
        for _ in range(case["steps"]):
            if case["rows"] > case["cols"]:
                gram = x.t() @ x
                x = a * x + x @ (b * gram + q * gram @ gram)
            else:
                gram = x @ x.t()
                x = a * x + (b * gram + q * gram @ gram) @ x
        got.append(case["scale"] * x)
    return dict(out=torch.stack(got))
