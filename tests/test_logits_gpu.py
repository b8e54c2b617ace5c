"""Adjusted logits against the oracle in 64 bits, within bounds that count its roundings."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import logits as ref
from tests.paged_cases import excess, int32
from thundersync_amd.logits import adjust_logits, pack_allowed
from thundersync_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(cuda, rows, vocab, *, dtype=torch.float32, ids=torch.int64, history=40, biases=6, mask=True, per_row=True, seed=0,
          rows_of_masks=None, repetition=1.3, frequency=0.2, presence=0.4):
    g = torch.Generator().manual_seed(seed)
    z = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    z[torch.rand(rows, vocab, generator=g) < 0.01] = -math.inf
    options, cpu = {}, [dict(z=z[i].double()) for i in range(rows)]
    counts, bias_size = torch.zeros(rows, vocab), torch.zeros(rows, vocab)
    if history:
        tokens = torch.randint(-1, max(2, min(vocab + 2, 60)), (rows, history), generator=g)
        tokens[:, ::3] = vocab - 1
        lengths = torch.randint(0, history + 1, (rows,), generator=g)
        lengths[0] = history
        prompts = (lengths * torch.rand(rows, generator=g)).int()
        options |= dict(history=tokens.to(ids), lengths=lengths.int(), prompt_lengths=prompts)
        value = lambda x: x * (0.5 + torch.rand(rows, generator=g)) if per_row else x  # noqa: E731
        options |= dict(repetition=value(repetition), frequency=value(frequency), presence=value(presence))
        for i in range(rows):
            h = tokens[i, :lengths[i]].tolist()
            cpu[i] |= dict(history=h, prompt=int(prompts[i]))
            cpu[i] |= {k: float(options[k][i]) if per_row else options[k] for k in ("repetition", "frequency", "presence")}
            for t in h:
                if 0 <= t < vocab:
                    counts[i, t] += 1
    if biases:
        at = torch.randint(-2, vocab + 2, (rows, biases), generator=g)
        at[:, -1] = at[:, 0]  # a token's biases add up
        add = 5 * torch.randn(rows, biases, generator=g)
        options |= dict(bias_ids=at.to(ids), bias=add)
        for i in range(rows):
            cpu[i] |= dict(bias_ids=at[i].tolist(), bias=add[i].tolist())
            for t, x in zip(at[i].tolist(), add[i].tolist()):
                if 0 <= t < vocab:
                    bias_size[i, t] += abs(x)
    if mask:
        n = rows if rows_of_masks is None else max(max(rows_of_masks), 0) + 1
        allowed = torch.rand(n, vocab, generator=g) < 0.6
        allowed[0] = False  # a mask that allows nothing
        options["allowed"] = pack_allowed(allowed)
        which = list(range(rows)) if rows_of_masks is None else rows_of_masks
        if rows_of_masks is not None:
            options["allowed_rows"] = torch.tensor(rows_of_masks, dtype=torch.int32)
        for i, m in enumerate(which):
            cpu[i] |= dict(allowed=None if m < 0 else allowed[m].tolist())
    on = {k: x.to(cuda) if isinstance(x, torch.Tensor) else x for k, x in options.items()}
    zc = z.to(cuda)
    out = adjust_logits(zc, **on)
    assert out.dtype == dtype and torch.equal(zc, z.to(cuda))
    want = torch.stack([ref.adjust(**c) for c in cpu])
    f = options.get("frequency", 0.0)
    p = options.get("presence", 0.0)
    column = lambda x: x.double()[:, None] if isinstance(x, torch.Tensor) else x  # noqa: E731
    size = z.double().abs() * 2 + abs(column(f)) * counts + abs(column(p)) + bias_size
    bound = want.abs() * torch.finfo(dtype).eps / 2 + (size + want.abs()) * 8 * 2.0 ** -24 + torch.finfo(dtype).tiny
    assert excess(out, want, bound) <= 0
    return zc, on, out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 31), (2, 33), (4, 1000), (3, 8191), (2, 8193), (1, 20011)])
def test_everything(cuda, dtype, ids, rows, vocab):
    check(cuda, rows, vocab, dtype=dtype, ids=ids)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("history, biases, mask", [(0, 0, False), (9, 0, False), (0, 5, False), (0, 0, True), (7, 3, False),
                                                   (1, 0, True), (0, 1, True)])
@pytest.mark.parametrize("per_row", [False, True])
def test_parts(cuda, dtype, history, biases, mask, per_row):
    check(cuda, 5, 9001, dtype=dtype, history=history, biases=biases, mask=mask, per_row=per_row)


def test_many_rows_and_tokens(cuda):
    check(cuda, 70, 300, history=900, biases=40)
    check(cuda, 2, 151936, history=5000, biases=300, dtype=torch.bfloat16)


def test_masks_by_row(cuda):
    check(cuda, 6, 500, rows_of_masks=[0, 2, -1, 1, 2, -7])


@pytest.mark.parametrize("rows", [1, 2, 300, 70000])
def test_numbers_of_rows(cuda, rows):
    """Every row is adjusted, also past 2^16 of them."""
    z = torch.zeros(rows, 40, device=cuda)
    h = (torch.arange(rows, device=cuda) % 40)[:, None]
    out = adjust_logits(z, history=h, presence=1.0)
    want = torch.zeros(rows, 40, device=cuda).scatter_(1, h, -1.0)
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place_and_strided(cuda, dtype):
    z, on, out = check(cuda, 4, 9001, dtype=dtype)
    wide = torch.zeros(4, 9100, dtype=dtype, device=cuda)
    for lead in (0, 1, 3, 8):
        view = wide[:, lead:lead + 9001]
        view.copy_(z)
        strided = dict(on, history=torch.cat([on["history"]] * 2, dim=1)[:, :on["history"].shape[1]],
                       allowed=torch.cat([on["allowed"]] * 2, dim=1)[:, :on["allowed"].shape[1]])
        assert torch.equal(adjust_logits(view, **strided), out)
        assert torch.equal(view, z)
        got = adjust_logits(view, out=view, **strided)
        assert got.data_ptr() == view.data_ptr() and torch.equal(view, out)
        assert wide[:, lead + 9001:].abs().max() == 0 and (lead == 0 or wide[:, :lead].abs().max() == 0)
        wide.zero_()
    assert torch.equal(adjust_logits(z.t().contiguous().t(), **on), out)
    assert torch.equal(adjust_logits(z[:1].expand(4, -1)), z[:1].expand(4, -1))


def test_numbers_that_are_none(cuda):
    """NaN and infinite logits, biases of -inf, penalties that are no numbers, a mask past the last."""
    z = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, -1.0]] * 3, device=cuda)
    h = torch.tensor([[0, 1, 2, 3, 4]] * 3, device=cuda)
    nan = torch.tensor([math.nan, 0.0, -2.0], device=cuda)
    out = adjust_logits(z, history=h, repetition=nan, frequency=torch.full((3,), math.nan, device=cuda))
    assert torch.equal(out.nan_to_num(7.0), z.nan_to_num(7.0))
    out = adjust_logits(z, history=h, repetition=2.0, presence=1.0, bias_ids=h[:, 3:4], bias=torch.full((3, 1), -math.inf, device=cuda))
    assert bool(out[:, 0].isnan().all()) and out[0, 1:].tolist() == [math.inf, -math.inf, -math.inf, -3.0]
    allowed = pack_allowed(torch.ones(2, 5, dtype=torch.bool, device=cuda))
    out = adjust_logits(z, allowed=allowed, allowed_rows=int32([0, 2, 1], cuda))
    assert bool(out[1].isnan().all()) and torch.equal(out[2].nan_to_num(7.0), z[2].nan_to_num(7.0))


def test_drawn_from(cuda):
    """What the sampler draws: only allowed tokens, none of a mask that allows nothing, no banned ones."""
    g = torch.Generator(device=cuda).manual_seed(0)
    z = torch.randn(64, 3000, generator=g, device=cuda)
    allowed = torch.rand(64, 3000, generator=g, device=cuda) < 0.01
    allowed[5] = False
    best = z.masked_fill(~allowed, -math.inf).argmax(dim=1)
    out = adjust_logits(z, allowed=pack_allowed(allowed), bias_ids=best[:, None],
                        bias=torch.full((64, 1), -math.inf, device=cuda))
    tokens, _ = sample_tokens(out, torch.rand(64, generator=g, device=cuda), top_p=0.9)
    assert tokens[5] == -1
    rest = torch.arange(64, device=cuda) != 5
    assert bool(allowed[rest].gather(1, tokens[rest][:, None]).all()) and bool((tokens != best)[rest].all())


def test_captured(cuda):
    """A captured call replays with new logits, history and penalties; an eager one between replays."""
    g = torch.Generator(device=cuda).manual_seed(1)
    z = torch.randn(8, 5000, generator=g, device=cuda)
    h = torch.randint(0, 5000, (8, 100), generator=g, device=cuda)
    n, r = torch.full((8,), 10, dtype=torch.int32, device=cuda), torch.full((8,), 1.5, device=cuda)
    call = lambda: adjust_logits(z, history=h, lengths=n, repetition=r, presence=0.5)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        z.normal_(generator=g)
        n.fill_(20 * k)
        r.fill_(1.0 + k)
        graph.replay()
        want = call()
        assert torch.equal(out, want)


def dense(z, history, lengths, prompts, repetition, frequency, presence, bias_ids, bias, allowed):
    """(want, bound) in 64 bits, over whole rows at once."""
    b, v = z.shape
    x, spots = z.double(), torch.arange(history.shape[1], device=z.device)[None]
    fine = (spots < lengths[:, None]) & (history >= 0) & (history < v)
    ids = history.long().masked_fill(~fine, 0)
    zeros = torch.zeros(b, v, dtype=torch.float64, device=z.device)
    seen = zeros.scatter_add(1, ids, fine.double()) > 0
    counts = zeros.scatter_add(1, ids, (fine & (spots >= prompts[:, None])).double())
    x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - frequency * counts - presence * (counts > 0)
    there = (bias_ids >= 0) & (bias_ids < v)
    at, size = bias_ids.long().masked_fill(~there, 0), bias.double() * there
    x = x.scatter_add(1, at, size)
    size = zeros.scatter_add(1, at, size.abs() * max(1, bias.shape[1]))  # each of a token's biases may round the sum
    bound = ref.bound(z, x, frequency, presence, counts, size, z.dtype)
    return x.masked_fill(~allowed, -math.inf), bound


@pytest.mark.parametrize("dtype, rows, vocab, width, biases", [
    (torch.bfloat16, 131, 33001, 40, 0),        # long slices, rows that begin at odd places
    (torch.bfloat16, 131, 33001, 5000, 1024),   # lists that a thread does not hold at once, the most biases
    (torch.float16, 67, 65537, 16383, 3),       # the longest history that 16 bits count
    (torch.float16, 67, 65537, 16384, 700),     # and one more
    (torch.bfloat16, 1, 65537, 16384, 700),
    (torch.float32, 131, 33001, 5000, 1024),
])
def test_long_rows(cuda, dtype, rows, vocab, width, biases):
    g = torch.Generator(device=cuda).manual_seed(rows + vocab)
    draw = lambda high, *shape: torch.randint(-1, high, shape, generator=g, device=cuda)  # noqa: E731
    z = torch.randn(rows, vocab, generator=g, device=cuda).to(dtype)
    history = draw(vocab + 1, rows, width)
    history[:, ::3] = vocab - 1  # one token again and again
    history[0] = 5
    lengths = draw(width + 1, rows).to(torch.int32)
    lengths[0] = width
    prompts = draw(width + 1, rows).to(torch.int32)
    prompts[0] = 0
    ids, bias = draw(vocab + 1, rows, biases), torch.randn(rows, biases, generator=g, device=cuda)
    ids[:, 1::2] = 7
    allowed = torch.rand(rows, vocab, generator=g, device=cuda) < 0.7
    allowed[:, [5, 7, vocab - 1]] = True
    options = (1.25, 2.0 ** -10, 0.5)
    got = adjust_logits(z, history=history, lengths=lengths, prompt_lengths=prompts, repetition=options[0],
                        frequency=options[1], presence=options[2], bias_ids=ids, bias=bias, allowed=pack_allowed(allowed))
    want, bound = dense(z, history, lengths, prompts, *options, ids, bias, allowed)
    assert excess(got, want.cpu(), bound.cpu()) <= 0
    again = z.clone()
    adjust_logits(again, history=history.to(torch.int32), lengths=lengths, prompt_lengths=prompts, repetition=options[0],
                  frequency=options[1], presence=options[2], bias_ids=ids.to(torch.int32), bias=bias,
                  allowed=pack_allowed(allowed), out=again)
    assert torch.equal(again, got)
