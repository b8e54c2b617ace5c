"""What is timed of a decoding step's operators: appending rotated keys and values to a paged cache, attention over that
cache, and the adjustment of logits before a token is drawn.

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
BLOCK = 16  # tokens of a page that share a scale
E4M3_MAX = 448.0


def listed():
    return [
        # One decoding step of a batch of rollouts into a 16-bit cache.
        {"name": "append_step", "op": "append", "seqs": 64, "low": 16, "high": 2047, "new": 1, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "bits": 16, "rotary": 128, "interleaved": False,
         "dtype": "bf16"},
        # Parts of several prompts, some of them continuing a block, with a quarter of wide heads rotated in pairs.
        {"name": "append_parts", "op": "append", "seqs": 6, "low": 0, "high": 500, "new": 1600, "ragged": True,
         "heads": 24, "kv_heads": 4, "dim": 256, "page": 16, "bits": 8, "rotary": 64, "interleaved": True,
         "dtype": "fp16"},
        # A batch of whole prompts into an 8-bit cache.
        {"name": "append_prompts", "op": "append", "seqs": 16, "low": 0, "high": 0, "new": 1024, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "bits": 8, "rotary": 128, "interleaved": False,
         "dtype": "bf16"},
        # One interactive sequence far into its context.
        {"name": "attend_one", "op": "attend", "seqs": 1, "low": 120000, "high": 131072, "new": 1, "ragged": False,
         "idle": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "bits": 8, "dtype": "bf16"},
        # A small model's step over a padded batch: the last rows hold no sequence.
        {"name": "attend_small", "op": "attend", "seqs": 48, "low": 1, "high": 3000, "new": 1, "ragged": False,
         "idle": 5, "heads": 16, "kv_heads": 8, "dim": 64, "page": 16, "bits": 8, "dtype": "fp16"},
        # A decoding step of a large batch of rollouts of every length.
        {"name": "attend_batch", "op": "attend", "seqs": 256, "low": 256, "high": 16384, "new": 1, "ragged": False,
         "idle": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "bits": 8, "dtype": "bf16"},
        # The same step's smaller batch over a cache that was kept in 16 bits.
        {"name": "attend_wide", "op": "attend", "seqs": 64, "low": 256, "high": 4096, "new": 1, "ragged": False,
         "idle": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "bits": 16, "dtype": "bf16"},
        # Up to five drafted tokens a sequence to verify, wide heads in groups of six.
        {"name": "attend_verify", "op": "attend", "seqs": 64, "low": 100, "high": 6000, "new": 5, "ragged": True,
         "idle": 0, "heads": 24, "kv_heads": 4, "dim": 256, "page": 32, "bits": 8, "dtype": "bf16"},
        # Prompts taken in chunks of 512 queries, late in long contexts.
        {"name": "attend_chunk", "op": "attend", "seqs": 4, "low": 1024, "high": 15872, "new": 512, "ragged": False,
         "idle": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "bits": 8, "dtype": "bf16"},
        # One sequence's logits under a repetition penalty alone.
        {"name": "logits_one", "op": "logits", "rows": 1, "vocab": 151936, "history": 3000, "penalties": "repetition",
         "biases": 0, "mask": False, "dtype": "bf16"},
        # A batch whose requests bring every penalty and a few biases, single-precision logits.
        {"name": "logits_batch", "op": "logits", "rows": 64, "vocab": 151936, "history": 4096, "penalties": "rows",
         "biases": 32, "mask": False, "dtype": "fp32"},
        # A large batch of structured answers: grammar masks beside the penalties, an odd number of rows.
        {"name": "logits_grammar", "op": "logits", "rows": 509, "vocab": 151936, "history": 8192, "penalties": "all",
         "biases": 8, "mask": True, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "logits"))
    if op == "logits":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        return {"op": op, "rows": _log_int(rng, 1, 254 if dtype == "fp32" else 509), "vocab": _log_int(rng, 1000, 151936),
                "history": _log_int(rng, 1, 8192), "penalties": rng.choice(("none", "repetition", "all", "rows")),
                "biases": rng.choice((0, 1, 8, 60)), "mask": rng.random() < 0.5, "dtype": dtype}
    heads, kv_heads, dim = rng.choice(((32, 8, 128), (32, 8, 128), (16, 8, 64), (40, 8, 128), (24, 4, 256), (8, 8, 64),
                                       (32, 2, 128), (12, 4, 192)))
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice((16, 32, 64, 128, 256)),
            "bits": rng.choice((8, 8, 16)), "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    row = kv_heads * dim
    if op == "append":
        # no more tokens than the largest listed case has elements for
        most = (16 * 1024 * 48 * 128) // ((heads + 2 * kv_heads) * dim)
        new = rng.choice((1, 1, _log_int(rng, 2, 4096)))
        seqs = _log_int(rng, 1, max(1, min(256, most // new)))
        case |= {"seqs": seqs, "low": 0, "high": _log_int(rng, 1, max(1, min(2048, most // seqs))), "new": new,
                 "ragged": new > 1 and rng.random() < 0.7, "rotary": rng.choice((dim, dim, dim // 2, 32)),
                 "interleaved": rng.random() < 0.3}
        return case
    new = rng.choice((1, 1, 1, _log_int(rng, 2, 8), _log_int(rng, 16, 1024)))
    seqs = _log_int(rng, 1, 256 if new < 16 else 8)
    most = 256 * 16384 * 8 * 128 // (seqs * row)  # elements of the listed largest cache
    if new > 1:
        most = min(most, 4 * 32 * 512 * 16384 // (seqs * heads * new))  # scores of the listed chunks
    high = _log_int(rng, 1, max(1, min(131072, most) - new))
    case |= {"seqs": seqs, "low": rng.choice((0, 0, high // 2, high)), "high": high, "new": new,
             "ragged": new > 1 and rng.random() < 0.7, "idle": rng.choice((0, 0, 1, 3)) if seqs > 3 and new == 1 else 0}
    return case


# ---------------------------------------------------------------------------
# the 8-bit form of a block of tokens
# ---------------------------------------------------------------------------
def _two_to(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale_for(most):
    """The smallest power of two by which values up to ``most`` fit e4m3."""
    m, e = torch.frexp(most.float())
    return _two_to(torch.where(most > 0, e - torch.where(m <= 0.875, 9, 8), -118).clamp(min=-118))


def _blocks(x):
    """``[pages, heads, page, dim]`` as ``[pages, heads, blocks, BLOCK, dim]``."""
    return x.unflatten(2, (-1, BLOCK))


def _codes(x, scale):
    return (x / scale).to(torch.float8_e4m3fn)


def _wide(codes, scale, dtype=torch.float32):
    """What pages of codes stand for."""
    return (_blocks(codes).to(dtype) * scale[..., None, None].to(dtype)).flatten(2, 3)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _zipf(vocab):
    """How often the tokens of a text occur, by rank."""
    p = 1.0 / (np.arange(vocab, dtype=np.float64) + 2.7)
    return p / p.sum()


def _prepare_cache(s, case, g, lengths, fill):
    """Pages in no order, the page table and, where ``fill``, keys and values in every page."""
    dt, page, hkv, d = DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["dim"]
    need = (lengths + page - 1) // page
    width = max(1, (case["high"] + case["new"] + page - 1) // page)
    pages = case["seqs"] * width + 4
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(width, device="cuda")
    first = need.cumsum(0) - need
    s["table"] = torch.where(at < need[:, None], order[(first[:, None] + at).clamp(max=pages - 1)], 0).to(torch.int32)
    shape = (pages, hkv, page, d)
    for name, spread in (("key", 2.0), ("value", 1.0)):
        bits8 = case["bits"] == 8
        s[name] = torch.zeros(shape, dtype=torch.float8_e4m3fn if bits8 else dt, device="cuda")
        s[name + "_scale"] = torch.full(shape[:2] + (page // BLOCK,), 2.0 ** -118, device="cuda") if bits8 else None
        if not fill:
            continue
        # some channels of a head are larger than the others, as keys' are
        channel = spread * torch.exp(0.5 * _normal(g, hkv, 1, d)) / math.exp(0.125)
        for part in range(0, pages, 4096):
            x = (_normal(g, min(4096, pages - part), *shape[1:]) * channel).to(dt).float()
            if bits8:
                scale = _scale_for(_blocks(x).abs().amax(dim=(-1, -2)))
                s[name + "_scale"][part:part + 4096] = scale
                s[name][part:part + 4096] = _codes(_blocks(x), scale[..., None, None]).flatten(2, 3)
            else:
                s[name][part:part + 4096] = x.to(dt)


def _new_tokens(case):
    """New tokens of each sequence: the case's own, so that a pass gives as many rows on any inputs."""
    if not case["ragged"]:
        return np.full(case["seqs"], case["new"])
    n = np.random.RandomState(case["seqs"] + case["new"]).randint(1, case["new"] + 1, case["seqs"])
    n[0] = case["new"]
    return n


def _rows_of(case, g):
    """New tokens of each sequence, and its length with them."""
    b = case["seqs"]
    n = torch.from_numpy(_new_tokens(case)).cuda()
    before = torch.randint(case["low"], case["high"] + 1, (b,), generator=g, device="cuda")
    lengths = before + n
    if case.get("idle"):
        lengths[b - case["idle"]:] = 0
    return n, lengths


def prepare(case, seed):
    dt = DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "logits":
        return _prepare_logits(s, case, dt, g)
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    n, lengths = _rows_of(case, g)
    total = int(n.sum())
    s["lengths"] = lengths.to(torch.int32)
    s["offsets"] = None
    if case["new"] > 1:
        s["offsets"] = torch.cat([n.new_zeros(1), n.cumsum(0)]).to(torch.int32)
    _prepare_cache(s, case, g, lengths, case["op"] == "attend")
    if case["op"] == "attend":
        s["query"] = _normal(g, total, h, d).to(dt)
        s["scale"] = d ** -0.5
        return s
    for name, heads in (("query_in", h), ("key_in", hkv), ("value_in", hkv)):
        s[name] = _normal(g, total, heads, d).to(dt)
    rot = case["rotary"]
    angle = torch.arange(case["high"] + case["new"], device="cuda", dtype=torch.float64)[:, None] * \
        (1e6 ** (-2.0 / rot * torch.arange(rot // 2, device="cuda", dtype=torch.float64)))
    s["rotary"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
    # what the sequences hold already, in the form the cache keeps it
    before = {"key_in": _normal(g, int(lengths.sum()) - total, hkv, d).to(dt),
              "value_in": _normal(g, int(lengths.sum()) - total, hkv, d).to(dt)}
    old = lengths - n
    start = torch.cat([old.new_zeros(1), old.cumsum(0)]).to(torch.int32)
    keep = {k: s[k] for k in ("lengths", "offsets", "rotary")}
    s |= {"lengths": old.to(torch.int32), "offsets": start, "rotary": None}
    if int(old.sum()):
        _append(s | {"query_in": before["key_in"]} | before, case, torch.float32)
    s |= keep
    return s


def _prepare_logits(s, case, dt, g):
    b, v, h = case["rows"], case["vocab"], case["history"]
    bias = torch.from_numpy(np.log(_zipf(v)) - np.log(_zipf(v))[0]).float().cuda()
    order = torch.randperm(v, generator=g, device="cuda")
    logits = 1.5 * _normal(g, b, v) + bias[order]
    logits[:, v - v // 500:] = -math.inf  # rows of the head that no token uses
    s["logits"] = logits.to(dt)
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
    s["options"] = {}
    if case["penalties"] != "none":
        text = torch.from_numpy(np.cumsum(_zipf(v))).cuda()
        rank = torch.searchsorted(text, rand(b, h).double()).clamp_(max=v - 1)
        tokens = torch.empty_like(order).scatter_(0, order, torch.arange(v, device="cuda"))[rank]
        lengths = (h * (0.3 + 0.7 * rand(b))).round().clamp(min=1).to(torch.int32)
        tokens.masked_fill_(torch.arange(h, device="cuda") >= lengths[:, None], -1)
        s["options"] |= {"history": tokens, "lengths": lengths, "prompt_lengths": (lengths * rand(b)).to(torch.int32)}
    if case["penalties"] == "repetition":
        s["options"] |= {"repetition": 1.1}
    elif case["penalties"] == "all":
        s["options"] |= {"repetition": 1.2, "frequency": 0.1, "presence": 0.5}
    elif case["penalties"] == "rows":
        off = rand(b) < 0.3
        s["options"] |= {"repetition": torch.where(off, 1.0, 1.0 + 0.5 * rand(b)),
                         "frequency": torch.where(off, 0.0, 0.3 * rand(b)), "presence": rand(b) - 0.2}
    if case["biases"]:
        ids = torch.randint(0, v, (b, case["biases"]), generator=g, device="cuda")
        ids.masked_fill_(rand(b, case["biases"]) < 0.2, -1)
        value = 4.0 * _normal(g, b, case["biases"])
        value[:, 0] = -100.0
        s["options"] |= {"bias_ids": ids, "bias": value}
    if case["mask"]:
        # a grammar allows few tokens at most places and most of them inside a text
        share = torch.where(rand(b, 1) < 0.5, 0.002, 0.95)
        bits = torch.zeros(b, (v + 31) // 32, dtype=torch.int64, device="cuda")
        for i in range(32):
            bits |= (rand(b, bits.shape[1]) < share).to(torch.int64) << i
        s["options"] |= {"allowed": torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)}
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "append":
        return _append_own(s, case) if own else _append_plain(s, case)
    if case["op"] == "attend":
        return _attend_own(s, case) if own else _attend_plain(s, case)
    return _logits_own(s, case) if own else _logits_plain(s, case)


def _cache(s):
    from thundersync_amd.paged import PagedCache

    if "cache" not in s:  # the handle that a program keeps beside the pages
        s["cache"] = PagedCache(s["key"], s["value"], s["key_scale"], s["value_scale"], dtype=DTYPES[s["case"]["dtype"]])
    return s["cache"]


def _append_own(s, case):
    from thundersync_amd.paged import append_tokens

    cache = _cache(s)
    query = append_tokens(cache, s["table"], s["lengths"], s["key_in"], s["value_in"], query=s["query_in"],
                          offsets=s["offsets"], rotary=s["rotary"], interleaved=case["interleaved"])
    key, value = cache.values()
    return {"query": query, "key": key, "value": value}


def _places(s, total):
    """The sequence and the position of each new token."""
    token = torch.arange(total, device="cuda")
    if s["offsets"] is None:
        return token, s["lengths"].long() - 1, torch.zeros_like(token)
    offsets = s["offsets"].long()
    seq = torch.searchsorted(offsets[1:], token, right=True)
    i = token - offsets[seq]
    return seq, s["lengths"].long()[seq] - (offsets[seq + 1] - offsets[seq]) + i, i


def _rotate(x, table, position, interleaved):
    rot = table.shape[1]
    cos, sin = table[position][:, None, :].chunk(2, dim=-1)
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _append(s, case, wide):
    """The new tokens into the pages; the rotated query."""
    dt, page = DTYPES[case["dtype"]], case["page"]
    seq, position, _ = _places(s, s["key_in"].shape[0])
    at_page, slot = s["table"].long()[seq, position // page], position % page
    q, k, v = (s[x].to(wide) for x in ("query_in", "key_in", "value_in"))
    if s["rotary"] is not None:
        q, k = (_rotate(x, s["rotary"].to(wide), position, case["interleaved"]) for x in (q, k))
    for name, x in (("key", k), ("value", v)):
        if case["bits"] == 16:
            s[name][at_page, :, slot] = x.to(dt)
            continue
        scale = s[name + "_scale"]
        pages, heads, blocks = scale.shape
        block = at_page * blocks + slot // BLOCK
        where = block[:, None].expand(-1, heads)
        most = torch.zeros(pages * blocks, heads, device="cuda", dtype=wide)
        most.scatter_reduce_(0, where, x.abs().amax(dim=-1), "amax")
        first = torch.full((pages * blocks,), BLOCK, device="cuda")
        first.scatter_reduce_(0, block, slot % BLOCK, "amin")
        first = first.view(pages, 1, blocks)
        need = _scale_for(most.view(pages, blocks, heads).transpose(1, 2))
        held = (first > 0) & (first < BLOCK)
        new = torch.where(first < BLOCK, torch.where(held, torch.maximum(scale, need), need), scale)
        # a block's older tokens by its new scale
        codes = _blocks(s[name])
        older = held[..., None, None] & (torch.arange(BLOCK, device="cuda")[:, None] < first[..., None, None])
        codes = torch.where(older, codes.float() * (scale / new)[..., None, None], codes.float())
        s[name].copy_(codes.to(torch.float8_e4m3fn).flatten(2, 3))
        s[name][at_page, :, slot] = _codes(x, new[at_page, :, slot // BLOCK][..., None].to(wide))
        scale.copy_(new)
    return q


@torch.no_grad()
def _append_plain(s, case):
    dt = DTYPES[case["dtype"]]
    query = _append(s, case, torch.float32).to(dt)
    if case["bits"] == 16:
        return {"query": query, "key": s["key"], "value": s["value"]}
    return {"query": query, "key": _wide(s["key"], s["key_scale"]).to(dt),
            "value": _wide(s["value"], s["value_scale"]).to(dt)}


def _attend_own(s, case):
    from thundersync_amd.paged import paged_attention

    return {"out": paged_attention(s["query"], _cache(s), s["table"], s["lengths"], s["scale"], offsets=s["offsets"])}


def _gathered(s, name, wide):
    """``[seqs, heads, width * page, dim]`` of the pages of each sequence."""
    table = s["table"].long()
    x = s[name]
    if s[name + "_scale"] is None:
        x = x[table].to(wide)
    else:
        x = x.view(torch.uint8)[table].view(torch.float8_e4m3fn).to(wide).unflatten(3, (-1, BLOCK))
        x = x.mul_(s[name + "_scale"][table][..., None, None].to(wide)).flatten(3, 4)
    return x.transpose(1, 2).flatten(2, 3)


@torch.no_grad()
def _attend_plain(s, case):
    b, h, hkv, d, new = (case[x] for x in ("seqs", "heads", "kv_heads", "dim", "new"))
    q = s["query"].float()
    seq, position, i = _places(s, q.shape[0])
    rows = torch.zeros(b, new, h, d, device="cuda")
    rows[seq, i] = q
    sees = torch.full((b, new), -1, device="cuda")
    sees[seq, i] = position
    # the heads of a group beside the tokens: [b, hkv, new * group, d]
    rows = rows.view(b, new, hkv, h // hkv, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    key = _gathered(s, "key", torch.float32)
    z = (rows @ key.transpose(2, 3)).mul_(s["scale"])
    del key
    at = torch.arange(z.shape[-1], device="cuda")
    hidden = (at > sees[..., None]).repeat_interleave(h // hkv, dim=1)[:, None]
    z = z.masked_fill_(hidden, -math.inf)
    z = z.sub_(z.amax(dim=-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = z.sum(dim=-1, keepdim=True)
    out = (z @ _gathered(s, "value", torch.float32)) / torch.where(total > 0, total, 1.0)
    out = out.view(b, hkv, new, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, new, h, d)
    return {"out": out[seq, i].to(s["query"].dtype)}


def _logits_own(s, case):
    from thundersync_amd.logits import adjust_logits

    return {"logits": adjust_logits(s["logits"], **s["options"])}


def _unpacked(bits, vocab):
    return ((bits[..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).flatten(1)[:, :vocab] != 0


@torch.no_grad()
def _logits_plain(s, case):
    z, o = s["logits"].float(), s["options"]
    b, v = z.shape
    column = lambda x: x[:, None] if isinstance(x, torch.Tensor) else x  # noqa: E731
    if "history" in o:
        at = torch.arange(o["history"].shape[1], device="cuda")
        there = (o["history"] >= 0) & (at < o["lengths"][:, None])
        made = there & (at >= o["prompt_lengths"][:, None])
        ids = o["history"].clamp(min=0)
        count = torch.zeros(b, v, device="cuda").scatter_add_(1, ids, made.float())
        seen = torch.zeros(b, v, device="cuda").scatter_add_(1, ids, there.float()) > 0
        r = column(o.get("repetition", 1.0))
        z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
        z = z - torch.where(count > 0, column(o.get("frequency", 0.0)) * count + column(o.get("presence", 0.0)), 0.0)
    if "bias" in o:
        there = o["bias_ids"] >= 0
        z = z + torch.zeros_like(z).scatter_add_(1, o["bias_ids"].clamp(min=0), o["bias"] * there)
    if "allowed" in o:
        z = z.masked_fill(~_unpacked(o["allowed"], v), -math.inf)
    return {"logits": z.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "logits":
        # the logits in and out, the history once, biases and mask bits
        size, n, v = (4 if case["dtype"] == "fp32" else 2), case["rows"], case["vocab"]
        history = 0 if case["penalties"] == "none" else 0.65 * 8 * case["history"]
        return {"bytes": int(n * (2 * size * v + history + 12 * case["biases"] + (v / 8 if case["mask"] else 0))),
                "flops": n * v}
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    new = float(_new_tokens(case).mean())
    live = case["seqs"] - case.get("idle", 0)
    before = (case["low"] + case["high"]) / 2
    each = 1 + 4 / (BLOCK * d) if case["bits"] == 8 else 2
    if case["op"] == "append":
        # query, key and value in, query and codes out; of an 8-bit cache also what it stands for
        tokens = case["seqs"] * new
        pages = case["seqs"] * -(-(case["high"] + case["new"]) // case["page"]) + 4
        back = pages * case["page"] * 2 * hkv * d * (each + 2) if case["bits"] == 8 else 0
        return {"bytes": int(tokens * d * (2 * 2 * h + 2 * hkv * (2 + each)) + back), "flops": int(tokens * (h + hkv) * 3 * d)}
    return {"bytes": int(live * (before + new) * 2 * hkv * d * each + 4 * case["seqs"] * new * h * d),
            "flops": int(4 * live * new * (before + (new + 1) / 2) * h * d)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _logits_exact(s)
    lengths = s["lengths"].tolist()
    offsets = list(range(len(lengths) + 1)) if s["offsets"] is None else s["offsets"].tolist()
    page, h, hkv, d = case["page"], case["heads"], case["kv_heads"], case["dim"]
    table = s["table"].long()
    if case["op"] == "append":
        return _append_exact(s, case, lengths, offsets, table)
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(lengths):
        n = offsets[i + 1] - offsets[i]
        if length == 0:
            continue
        pages = table[i, :(length + page - 1) // page]
        kv = []
        for name in ("key", "value"):
            x = s[name][pages].double() if s[name + "_scale"] is None else \
                s[name].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * \
                s[name + "_scale"][pages].double().repeat_interleave(BLOCK, dim=-1)[..., None]
            kv.append(x.transpose(0, 1).reshape(hkv, -1, d)[:, :length])
        at = torch.arange(length, device="cuda")
        hidden = at > (length - n + torch.arange(n, device="cuda"))[:, None]
        for j in range(h):
            z = s["query"][offsets[i]:offsets[i + 1], j].double() @ kv[0][j * hkv // h].T * s["scale"]
            out[offsets[i]:offsets[i + 1], j] = torch.softmax(z.masked_fill(hidden, -math.inf), dim=-1) @ kv[1][j * hkv // h]
    return {"out": out}


def _append_exact(s, case, lengths, offsets, table):
    page, bits, d, rot = case["page"], case["bits"], case["dim"], case["rotary"]
    rotary = s["rotary"].double()

    def turned(x, position):
        c, t = rotary[position, :rot // 2][:, None], rotary[position, rot // 2:][:, None]
        z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) if case["interleaved"] else \
            torch.complex(x[..., :rot // 2], x[..., rot // 2:rot])
        z = z * torch.complex(c, t)
        both = torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], dim=-1)
        return torch.cat([both, x[..., rot:]], dim=-1)

    result = {"query": torch.empty(s["query_in"].shape, dtype=torch.float64, device="cuda")}
    for name in ("key", "value"):
        x = s[name].double()
        result[name] = x if bits == 16 else x * s[name + "_scale"].double().repeat_interleave(BLOCK, dim=-1)[..., None]
    for i, length in enumerate(lengths):
        rows = slice(offsets[i], offsets[i + 1])
        position = torch.arange(length - (offsets[i + 1] - offsets[i]), length, device="cuda")
        result["query"][rows] = turned(s["query_in"][rows].double(), position)
        new = {"key": turned(s["key_in"][rows].double(), position), "value": s["value_in"][rows].double()}
        where, slot = table[i, position // page], position % page
        for name, x in new.items():
            result[name][where, :, slot] = x
            if bits == 16:
                continue
            blocks = s[name + "_scale"].shape[2]
            block = (where * blocks + slot // BLOCK)
            grid = result[name].view(-1, case["kv_heads"], blocks, BLOCK, d)
            codes = s[name].view(-1, case["kv_heads"], blocks, BLOCK, d)
            for b in block.unique().tolist():
                held = int(slot[block == b].min()) % BLOCK  # older tokens of the block
                upto = int(slot[block == b].max()) % BLOCK + 1
                vals = grid[b // blocks, :, b % blocks]
                old = s[name + "_scale"][b // blocks, :, b % blocks].double()
                top = vals[:, held:upto].abs().amax(dim=(1, 2))
                m, e = torch.frexp(top)
                scale = torch.ldexp(torch.ones_like(top), e - torch.where(m <= 0.875, 9, 8))
                scale = torch.maximum(scale, old) if held else scale
                vals[:, :upto] = (vals[:, :upto] / scale[:, None, None]).float().to(torch.float8_e4m3fn).double() * \
                    scale[:, None, None]
                # slots behind the new tokens hold no token: their codes stay
                vals[:, upto:] = codes[b // blocks, :, b % blocks, upto:].double() * scale[:, None, None]
    return result


def _logits_exact(s):
    z, o = s["logits"].double(), s["options"]
    v = z.shape[1]
    out = []
    for i, row in enumerate(z):
        at = lambda x, default: float(x[i]) if isinstance(x, torch.Tensor) else (default if x is None else x)  # noqa: E731
        if "history" in o:
            n, p = int(o["lengths"][i]), int(o["prompt_lengths"][i])
            seen = torch.bincount(o["history"][i, :n], minlength=v) > 0
            count = torch.bincount(o["history"][i, p:n], minlength=v).double()
            r = at(o.get("repetition"), 1.0)
            row = torch.where(seen, torch.where(row > 0, row / r, row * r), row)
            row = row - at(o.get("frequency"), 0.0) * count - at(o.get("presence"), 0.0) * (count > 0)
        if "bias" in o:
            there = o["bias_ids"][i] >= 0
            row = row.index_add(0, o["bias_ids"][i][there], o["bias"][i][there].double())
        if "allowed" in o:
            bits = o["allowed"][i].long()[torch.arange(v, device="cuda") // 32] >> (torch.arange(v, device="cuda") % 32)
            row = torch.where(bits & 1 == 1, row, -math.inf)
        out.append(row)
    return {"logits": torch.stack(out)}
