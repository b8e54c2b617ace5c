"""What is timed of the operators at the vocabulary: distillation from a teacher's top logits through the head, the
embedding with its gradient, and sampling from the head's logits.

A case is a dict of plain values; its ``op`` names the operator, the rest are sizes and options.  ``listed()`` holds the
named cases, ``draw()`` gives further ones of the same ranges, ``prepare()`` makes what the caller holds before the
call, ``run()`` is one pass: with ``own`` through the framework's entry points, otherwise in plain torch operations.
``exact()`` computes the same outputs in 64 bits.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False  # whether run() goes through the framework's entry points

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # A streamed turn's few scored positions against a teacher's twenty returned logits, frozen head.
        {"name": "distill_turn", "op": "distill", "rows": 48, "hidden": 4096, "vocab": 151936, "top": 20,
         "temperature": 1.0, "train": False, "dtype": "bf16"},
        # A batch of completions' scored positions, sixty-four teacher logits each, softened, frozen head.
        {"name": "distill_batch", "op": "distill", "rows": 2048, "hidden": 4096, "vocab": 151936, "top": 64,
         "temperature": 2.0, "train": False, "dtype": "bf16"},
        # A smaller decoder's trainable head in half precision over an odd number of rows.
        {"name": "distill_train", "op": "distill", "rows": 1999, "hidden": 2048, "vocab": 151936, "top": 100,
         "temperature": 1.0, "train": True, "dtype": "fp16"},
        # A small single-precision run with a trainable head and an odd vocabulary.
        {"name": "distill_fp32", "op": "distill", "rows": 600, "hidden": 1024, "vocab": 32003, "top": 32,
         "temperature": 0.7, "train": True, "dtype": "fp32"},
        # The lookup of one decoding step of a batch of rollouts.
        {"name": "embed_step", "op": "embed", "rows": 64, "hidden": 4096, "vocab": 151936, "scale": 1.0, "grad": False,
         "dtype": "bf16"},
        # A streamed turn's lookup with the table's gradient, half precision, width that is no power of two.
        {"name": "embed_turn", "op": "embed", "rows": 500, "hidden": 2560, "vocab": 50257, "scale": 1.0, "grad": True,
         "dtype": "fp16"},
        # A training batch's lookup with the table's gradient.
        {"name": "embed_batch", "op": "embed", "rows": 16384, "hidden": 4096, "vocab": 151936, "scale": 1.0,
         "grad": True, "dtype": "bf16"},
        # A long single-precision batch over a small table, scaled by the root of the width.
        {"name": "embed_scaled", "op": "embed", "rows": 65536, "hidden": 1024, "vocab": 32000, "scale": 32.0,
         "grad": True, "dtype": "fp32"},
        # One sequence's next token with the filters of an interactive rollout.
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 151936, "mode": "all", "dtype": "bf16"},
        # A decoding step of a batch of rollouts, single-precision logits, nucleus alone.
        {"name": "sample_nucleus", "op": "sample", "rows": 64, "vocab": 151936, "mode": "top_p", "dtype": "fp32"},
        # A decoding step of a large batch that draws from the policy itself, as a policy gradient asks.
        {"name": "sample_policy", "op": "sample", "rows": 512, "vocab": 151936, "mode": "none", "dtype": "bf16"},
        # A batch whose requests bring their own settings, greedy ones among them, over an odd vocabulary.
        {"name": "sample_mixed", "op": "sample", "rows": 333, "vocab": 50257, "mode": "rows", "dtype": "fp16"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("distill", "distill", "embed", "sample", "sample"))
    if op == "distill":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        single = dtype == "fp32"
        hidden = rng.choice((128, 1000, 1024) if single else (1024, 2048, 2560, 4096))
        vocab = _log_int(rng, 1000, 32003 if single else 151936)
        # no more work than the largest listed case of the type
        most = 600 * 1024 * 32003 if single else 1999 * 2048 * 151936
        return {"op": op, "rows": _log_int(rng, 1, max(1, min(4096, most // (hidden * vocab)))), "hidden": hidden,
                "vocab": vocab, "top": min(_log_int(rng, 1, 128), vocab), "temperature": rng.choice((0.7, 1.0, 1.0, 2.0)),
                "train": rng.random() < 0.4, "dtype": dtype}
    if op == "embed":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        hidden = rng.choice((128, 1000, 1024, 2048, 2560, 4096))
        vocab = _log_int(rng, 1000, min(151936, (1 << 28) // hidden if dtype == "fp32" else 151936))
        return {"op": op, "rows": _log_int(rng, 1, min(65536, (1 << 26) // hidden)), "hidden": hidden, "vocab": vocab,
                "scale": rng.choice((1.0, math.sqrt(hidden))), "grad": rng.random() < 0.75, "dtype": dtype}
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    vocab = _log_int(rng, 1000, 151936)
    return {"op": op, "rows": _log_int(rng, 1, 256 if dtype == "fp32" else 512), "vocab": vocab,
            "mode": rng.choice(("none", "top_k", "top_p", "min_p", "all", "rows")), "dtype": dtype}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _zipf(vocab):
    """How often the tokens of a text occur, by rank."""
    p = 1.0 / (np.arange(vocab, dtype=np.float64) + 2.7)
    return p / p.sum()


def prepare(case, seed):
    op, dt, v = case["op"], DTYPES[case["dtype"]], case["vocab"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if op == "distill":
        n, d, k = case["rows"], case["hidden"], case["top"]
        s["weight"] = (_normal(g, v, d) * (1.5 / math.sqrt(d))).to(dt).requires_grad_(case["train"])
        s["hidden"] = _normal(g, n, d).to(dt).requires_grad_()
        # the teacher sees much the same as the student: its logits are the student's and a difference
        ids, logits = [], []
        with torch.no_grad():
            for part in s["hidden"].split(512):
                scores = (part @ s["weight"].T).float() + _normal(g, part.shape[0], v)
                top = scores.topk(k, dim=1)
                ids.append(top.indices)
                logits.append(top.values + 3.0)
        s["ids"], s["teacher"] = torch.cat(ids), torch.cat(logits)
        # some rows have fewer teacher logits than the widest, a few (prompt positions) none
        have = torch.randint(1, k + 1, (n, 1), generator=g, device="cuda")
        have = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.5, k, have)
        have = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.03, 0, have)
        absent = torch.arange(k, device="cuda") >= have
        s["teacher"].masked_fill_(absent, -math.inf)
        s["ids"].masked_fill_(absent, -1)
        s["grad"] = torch.rand(n, generator=g, device="cuda") + 0.5  # a loss scale and per-row weights
    elif op == "embed":
        n, d = case["rows"], case["hidden"]
        s["weight"] = _normal(g, v, d).mul_(0.02).to(dt).requires_grad_(case["grad"])
        text = torch.from_numpy(np.cumsum(_zipf(v))).cuda()
        rank = torch.searchsorted(text, torch.rand(n, generator=g, device="cuda", dtype=torch.float64)).clamp_(max=v - 1)
        s["ids"] = torch.randperm(v, generator=g, device="cuda")[rank]
        if case["grad"]:
            s["dout"] = _normal(g, n, d).to(dt)
    else:
        b = case["rows"]
        bias = torch.from_numpy(np.log(_zipf(v)) - np.log(_zipf(v))[0]).float().cuda()
        bias = bias[torch.randperm(v, generator=g, device="cuda")]
        sharp = 0.5 + 1.5 * torch.rand(b, 1, generator=g, device="cuda")
        logits = (1.5 * _normal(g, b, v) + bias) * sharp
        logits[:, v - v // 500:] = -math.inf  # rows of the head that no token uses
        s["logits"] = logits.to(dt)
        s["uniform"] = torch.rand(b, generator=g, device="cuda")
        s["options"] = {
            "none": {}, "top_k": {"top_k": 50}, "top_p": {"temperature": 0.7, "top_p": 0.95},
            "min_p": {"temperature": 1.3, "min_p": 0.02},
            "all": {"temperature": 0.8, "top_k": 200, "top_p": 0.9, "min_p": 0.01},
        }.get(case["mode"])
        if case["mode"] == "rows":
            rand = lambda: torch.rand(b, generator=g, device="cuda")  # noqa: E731
            off = lambda: rand() < 0.4  # noqa: E731
            s["options"] = {
                "temperature": torch.where(rand() < 0.1, 0.0, 0.4 + rand()),
                "top_k": torch.where(off(), 0, torch.randint(1, min(v, 2000), (b,), generator=g, device="cuda")).int(),
                "top_p": torch.where(off(), 1.0, 0.3 + 0.69 * rand()),
                "min_p": torch.where(off(), 0.0, 0.1 * rand()),
            }
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "distill":
        return _distill_own(s, case) if own else _distill_plain(s, case)
    if case["op"] == "embed":
        return _embed_own(s, case) if own else _embed_plain(s, case)
    return _sample_own(s, case) if own else _sample_plain(s, case)


def _distill_own(s, case):
    from thundersync_amd.fused_distill import fused_distill

    leaves = [s["hidden"], s["weight"]] if case["train"] else [s["hidden"]]
    loss = fused_distill(s["hidden"], s["weight"], s["ids"], s["teacher"], temperature=case["temperature"])
    grads = torch.autograd.grad(loss, leaves, s["grad"].to(loss.dtype))
    return {"loss": loss.detach(), "grads": list(grads)}


@torch.no_grad()
def _distill_plain(s, case):
    h, w, t = s["hidden"].float(), s["weight"].float(), case["temperature"]
    present = (s["ids"] >= 0) & (s["teacher"] > -math.inf)
    some = present.any(dim=1)
    x = (s["teacher"] / t).masked_fill(~present, -math.inf)
    x = torch.exp(x - x.amax(dim=1, keepdim=True).masked_fill(~some[:, None], 0.0))
    slots = x / x.sum(dim=1, keepdim=True).masked_fill(~some[:, None], 1.0)
    z = (h @ w.T) / t
    p = torch.zeros_like(z).scatter_add_(1, s["ids"].clamp(min=0), slots)
    z -= z.amax(dim=1, keepdim=True)
    q = torch.exp(z)
    total = q.sum(dim=1, keepdim=True)
    log_q = z - torch.log(total)
    loss = torch.where(p > 0, p * (torch.log(p) - log_q), 0.0).sum(dim=1)
    dz = (q / total - p) * (s["grad"] / t)[:, None]
    dz = torch.where(some[:, None], dz, 0.0)
    grads = [(dz @ w).to(s["hidden"].dtype)]
    if case["train"]:
        grads.append((dz.T @ h).to(s["weight"].dtype))
    return {"loss": torch.where(some, loss, 0.0), "grads": grads}


def _embed_own(s, case):
    from thundersync_amd.embedding import embedding

    out = embedding(s["ids"], s["weight"], scale=case["scale"])
    if not case["grad"]:
        return {"out": out}
    (grad,) = torch.autograd.grad(out, s["weight"], s["dout"])
    return {"out": out.detach(), "grad": grad}


@torch.no_grad()
def _embed_plain(s, case):
    w = s["weight"]
    out = {"out": (w[s["ids"]].float() * case["scale"]).to(w.dtype)}
    if case["grad"]:
        total = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        total.index_add_(0, s["ids"], s["dout"].float())
        out["grad"] = (total * case["scale"]).to(w.dtype)
    return out


def _sample_own(s, case):
    from thundersync_amd.sampling import sample_tokens

    tokens, logprobs = sample_tokens(s["logits"], s["uniform"], **s["options"])
    return {"tokens": tokens, "logprobs": logprobs}


@torch.no_grad()
def _sample_plain(s, case):
    z, o = s["logits"].double(), s["options"]
    b, v = z.shape
    at = torch.arange(v, device=z.device)

    def option(name, default):
        x = o.get(name, default)
        return x.double()[:, None] if isinstance(x, torch.Tensor) else torch.full((b, 1), float(x), device=z.device,
                                                                                dtype=torch.float64)

    t, k, top_p, min_p = option("temperature", 1.0), option("top_k", 0), option("top_p", 1.0), option("min_p", 0.0)
    top = z.amax(dim=1, keepdim=True)
    greedy = t == 0
    w = torch.exp((z - top) / torch.where(greedy, 1.0, t))
    w = torch.where(greedy, (z == top).double(), w)
    k = torch.where(greedy, 1.0, k)
    # the tokens by falling logit, equal ones by their index
    order = z.sort(dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    keep = (at < k) | (k <= 0)
    ws_k = torch.where(keep, ws, 0.0)
    before = ws_k.cumsum(dim=1) - ws_k
    keep &= (before < top_p * ws_k.sum(dim=1, keepdim=True)) | (top_p >= 1)
    keep &= (ws >= min_p) & (ws > 0)
    keep |= at == 0
    wk = torch.where(torch.zeros_like(keep).scatter_(1, order, keep), w, 0.0)
    running = wk.cumsum(dim=1)
    total = running[:, -1:]
    last = torch.where(wk > 0, at, 0).amax(dim=1)
    tokens = torch.minimum((running <= s["uniform"].double()[:, None] * total).sum(dim=1), last)
    return {"tokens": tokens, "logprobs": torch.log(wk.gather(1, tokens[:, None]) / total)[:, 0].float()}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    n, v = case["rows"], case["vocab"]
    if case["op"] == "distill":
        # hidden, weight, ids and teacher logits in; the loss and the gradients out.  The logits, the hidden states'
        # gradient and the weight's are a product each.
        d, train = case["hidden"], case["train"]
        return {"bytes": size * (2 * n * d + v * d * (2 if train else 1)) + 12 * n * case["top"] + 8 * n,
                "flops": (6 if train else 4) * n * v * d}
    if case["op"] == "embed":
        # the ids and the table's rows that occur, once each; the output; the output's gradient and the table's
        d = case["hidden"]
        rows = float(-np.expm1(n * np.log1p(-_zipf(v))).sum())
        grad = size * d * (n + v) if case["grad"] else 0
        return {"bytes": int(8 * n + size * d * (rows + n) + grad), "flops": n * d * (2 if case["grad"] else 1)}
    return {"bytes": size * n * v + 16 * n, "flops": 4 * n * v}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "distill":
        h, w, t = s["hidden"].double(), s["weight"].double(), case["temperature"]
        n, v = h.shape[0], w.shape[0]
        row = torch.arange(n, device=h.device)[:, None].expand_as(s["ids"])
        there = (s["ids"] >= 0) & ~torch.isneginf(s["teacher"])
        p = torch.zeros(n, v, dtype=torch.float64, device=h.device)
        lse_t = torch.logsumexp(s["teacher"].double().where(there, torch.tensor(-math.inf, device=h.device)) / t, dim=1)
        p.index_put_((row[there], s["ids"][there]), torch.exp(s["teacher"].double() / t - lse_t[:, None])[there],
                     accumulate=True)
        log_q = torch.log_softmax(h @ w.T / t, dim=1)
        some = there.any(dim=1)
        loss = (torch.special.xlogy(p, p) - p * log_q).sum(dim=1) * some
        dz = (log_q.exp() - p) * (s["grad"].double() * some / t)[:, None]
        return {"loss": loss, "grads": [dz @ w, dz.T @ h] if case["train"] else [dz @ w]}
    if case["op"] == "embed":
        w = s["weight"].double()
        out = {"out": w[s["ids"]] * case["scale"]}
        if case["grad"]:
            out["grad"] = torch.zeros_like(w).index_put_((s["ids"],), s["dout"].double() * case["scale"],
                                                         accumulate=True)
        return out
    logits, uniform = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy()
    options = {k: x.double().cpu().numpy() if isinstance(x, torch.Tensor) else np.full(len(logits), float(x))
               for k, x in s["options"].items()}
    tokens, logprobs = [], []
    for i, z in enumerate(logits):
        t, k, top_p, min_p = (float(options[o][i]) if o in options else d for o, d in
                              (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
        if t == 0:
            tokens.append(int(np.argmax(z)))
            logprobs.append(0.0)
            continue
        weight = np.exp((z - z.max()) / t)
        chosen = np.flatnonzero(weight > 0)
        if k > 0 or top_p < 1:
            chosen = chosen[np.argsort(-z[chosen], kind="stable")]
            chosen = chosen[: int(k)] if k > 0 else chosen
            if top_p < 1:
                c = np.cumsum(weight[chosen])
                chosen = chosen[: 1 + int(np.count_nonzero(c[:-1] < top_p * c[-1]))]
            chosen.sort()
        chosen = chosen[weight[chosen] >= min_p]
        c = np.cumsum(weight[chosen])
        at = min(int(np.searchsorted(c, uniform[i] * c[-1], side="right")), len(chosen) - 1)
        tokens.append(int(chosen[at]))
        logprobs.append(math.log(weight[chosen[at]] / c[-1]))
    return {"tokens": torch.tensor(tokens), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}
