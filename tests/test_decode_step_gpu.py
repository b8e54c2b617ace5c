"""A decoding step as a rollout runs it: embedding, append, attention, head, adjusted logits, sampling."""

from __future__ import annotations

import pytest
import torch

from oracle import paged as ref
from oracle import sampling as ref_sampling
from tests.paged_cases import excess, int32, offsets_of
from thundersync_amd.attention import causal_attention
from thundersync_amd.embedding import embedding
from thundersync_amd.logits import adjust_logits, pack_allowed
from thundersync_amd.paged import PagedCache, append_tokens, paged_attention, rotary_table
from thundersync_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class Decoder:
    """One attention layer between a table and a head."""

    def __init__(self, cuda, seqs, *, heads=4, kv_heads=2, dim=64, vocab=500, page=16, width=12, bits=8, seed=0):
        g = torch.Generator(device=cuda).manual_seed(seed)
        self.g, self.seqs, self.heads, self.kv_heads, self.dim, self.vocab = g, seqs, heads, kv_heads, dim, vocab
        self.table = torch.randn(vocab, 128, generator=g, device=cuda).to(BF)
        self.qkv = (torch.randn(128, (heads + 2 * kv_heads) * dim, generator=g, device=cuda) * 128 ** -0.5).to(BF)
        self.head = (torch.randn(heads * dim, vocab, generator=g, device=cuda) * 0.1).to(BF)
        self.cache = PagedCache.empty(seqs * width, page, kv_heads, dim, bits=bits, device=cuda)
        self.pages = torch.randperm(seqs * width, generator=g, device=cuda).to(torch.int32).view(seqs, width)
        self.rotary = rotary_table(page * width, dim, device=cuda)
        self.allowed = pack_allowed(torch.rand(seqs, vocab, generator=g, device=cuda) < 0.8)
        self.history = torch.full((seqs, page * width), -1, device=cuda)

    def layer(self, tokens, lengths, offsets=None):
        x = (embedding(tokens, self.table) @ self.qkv).view(-1, self.heads + 2 * self.kv_heads, self.dim)
        q, k, v = x.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        q = append_tokens(self.cache, self.pages, lengths, k, v, query=q, offsets=offsets, rotary=self.rotary)
        return q, paged_attention(q, self.cache, self.pages, lengths, self.dim ** -0.5, offsets=offsets)

    def draw(self, out, lengths, prompts, uniform):
        logits = out.flatten(1) @ self.head
        logits = adjust_logits(logits, history=self.history, lengths=lengths, prompt_lengths=prompts, repetition=1.2,
                               presence=0.3, allowed=self.allowed)
        return logits, *sample_tokens(logits, uniform, temperature=0.8, top_p=0.9)

    def dense(self, s, length):
        """Keys and values [1, length, kv_heads, dim] of sequence s, as the cache has them."""
        key, value = self.cache.values()
        pos = torch.arange(length, device=key.device)
        ids = self.pages[s].long()[pos // self.cache.page_size]
        return [x[ids, :, pos % self.cache.page_size].contiguous() for x in (key, value)]


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dim", [64, 128])
def test_rollout(cuda, bits, dim):
    """Prompts, then tokens: attention as the framework's own over the same keys, tokens as the sampler's oracle draws."""
    m = Decoder(cuda, 3, bits=bits, dim=dim)
    prompts = [33, 5, 70]
    ids = torch.randint(0, m.vocab, (sum(prompts),), generator=m.g, device=cuda)
    lengths = int32(prompts, cuda)
    start = lengths.clone()
    at = 0
    for s, n in enumerate(prompts):
        m.history[s, :n] = ids[at:at + n]
        at += n
    q, out = m.layer(ids, lengths, offsets_of(prompts, cuda))
    at = 0
    for s, n in enumerate(prompts):
        k, v = m.dense(s, n)
        whole = causal_attention(q[at:at + n].transpose(0, 1)[None], [k], [v], dim ** -0.5)[0].transpose(0, 1)
        want, bound = ref.attention(q[at:at + n].cpu(), k.cpu(), v.cpu(), dim ** -0.5, BF)
        assert excess(out[at:at + n], want, bound) <= 0
        assert excess(out[at:at + n], whole.double().cpu(), 2 * bound) <= 0
        at += n
    out = out[[prompts[0] - 1, prompts[0] + prompts[1] - 1, sum(prompts) - 1]]
    for step in range(40):
        u = torch.rand(3, generator=m.g, device=cuda)
        logits, tokens, _ = m.draw(out, lengths, start, u)
        for s in range(3):
            row = logits[s].double().cpu().numpy()
            if ref_sampling.border_distance(row, float(u[s]), 0.8, 0, 0.9) > 1e-9:
                assert int(tokens[s]) == ref_sampling.sample(row, float(u[s]), 0.8, 0, 0.9)[0]
        m.history.scatter_(1, lengths[:, None].long(), tokens[:, None])
        lengths = lengths + 1
        q, out = m.layer(tokens, lengths)
        for s in range(3):
            n = int(lengths[s])
            want, bound = ref.attention(q[s:s + 1].cpu(), *(x.cpu() for x in m.dense(s, n)), dim ** -0.5, BF)
            assert excess(out[s:s + 1], want, bound) <= 0, (step, s)


@pytest.mark.parametrize("bits", [8, 16])
def test_captured_step(cuda, bits):
    """One graph for every step of a rollout; an eager twin runs between the replays and gets the same tokens and pages."""
    a, b = (Decoder(cuda, 5, bits=bits, seed=4) for _ in range(2))
    state = []
    for m in (a, b):
        lengths, tokens, u = int32([1, 1, 1, 1, 0], cuda), torch.arange(5, device=cuda), torch.zeros(5, device=cuda)
        m.history[:, 0] = tokens
        state.append((lengths, tokens, u))

    def step(m, lengths, tokens, u):
        _, out = m.layer(tokens, lengths)
        return m.draw(out, lengths, torch.ones_like(lengths), u)

    step(a, *state[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(a, *state[0])
    for k in range(30):
        u = torch.rand(5, generator=a.g, device=cuda)
        for s in state:
            s[2].copy_(u)
        graph.replay()
        eager = step(b, *state[1])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured[:2], eager[:2])), k
        assert all(torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(a.cache.values(), b.cache.values()))
        for m, (lengths, tokens, _), got in zip((a, b), state, (captured, eager)):
            live = lengths > 0
            tokens.copy_(torch.where(live, got[1], tokens))
            m.history.scatter_(1, lengths[:, None].long(), tokens[:, None])
            lengths += live.int()


def test_on_other_streams(cuda):
    """Calls in flight on several streams at once, each with its own rows, over one cache."""
    g = torch.Generator(device=cuda).manual_seed(0)
    cache = PagedCache.empty(64, 64, 2, 128, bits=8, device=cuda)
    table = torch.arange(64, dtype=torch.int32, device=cuda).view(2, 32)
    x = torch.randn(4000, 2, 128, generator=g, device=cuda).to(BF)
    lengths = int32([2000, 2000], cuda)
    append_tokens(cache, table, lengths, x, x, offsets=int32([0, 2000, 4000], cuda))
    q = [torch.randn(2, 8, 128, generator=g, device=cuda).to(BF) for _ in range(4)]
    want = [paged_attention(y, cache, table, lengths, 0.1) for y in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    for _ in range(5):
        got = []
        for y, stream in zip(q, streams):
            with torch.cuda.stream(stream):
                got.append(paged_attention(y, cache, table, lengths, 0.1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_checked_batches(cuda, monkeypatch):
    monkeypatch.setenv("THUNDERSYNC_CHECK_TARGETS", "1")
    cache = PagedCache.empty(4, 16, 1, 64, device=cuda)
    x = torch.ones(2, 1, 64, dtype=BF, device=cuda)
    table, lengths = int32([[0, 1], [2, 3]], cuda), int32([17, 3], cuda)
    append_tokens(cache, table, lengths, x, x)
    paged_attention(x, cache, table, lengths, 1.0)
    for change, words in (({"table": int32([[0, 4], [2, 3]], cuda)}, "sequence 0"), ({"lengths": int32([17, 33], cuda)}, "sequence 1"),
                          ({"lengths": int32([-1, 3], cuda)}, "sequence 0"), ({"offsets": int32([0, 2, 1], cuda)}, "offsets"),
                          ({"offsets": int32([0, 1, 3], cuda)}, "offsets"),
                          ({"offsets": int32([0, 0, 2], cuda), "lengths": int32([5, 1], cuda)}, "sequence 1")):
        t, n, off = change.get("table", table), change.get("lengths", lengths), change.get("offsets")
        with pytest.raises(ValueError, match=words):
            append_tokens(cache, t, n, x, x, offsets=off)
        with pytest.raises(ValueError, match=words):
            paged_attention(x, cache, t, n, 1.0, offsets=off)
    with pytest.raises(ValueError, match="one block"):
        append_tokens(cache, int32([[0, 1], [1, 3]], cuda), int32([17, 3], cuda), x, x)


def test_availability(cuda, monkeypatch):
    from thundersync_amd import _lib, dispatch

    for dtype in (BF, torch.float16):
        for dim in (64, 72, 128, 256):
            assert dispatch.hip_paged_available(torch.zeros(2, 4, dim, device=cuda, dtype=dtype))
        assert dispatch.hip_adjust_logits_available(torch.zeros(2, 70, device=cuda, dtype=dtype))
    assert dispatch.hip_adjust_logits_available(torch.zeros(2, 1, device=cuda))
    for query in (torch.zeros(2, 4, 64, device=cuda), torch.zeros(2, 4, 64, dtype=BF),
                  torch.zeros(2, 4, 60, device=cuda, dtype=BF), torch.zeros(2, 4, 264, device=cuda, dtype=BF)):
        assert not dispatch.hip_paged_available(query)
    assert not dispatch.hip_adjust_logits_available(torch.zeros(2, 64))
    monkeypatch.setenv("THUNDERSYNC_HIP", "off")
    _lib.reset()
    try:
        assert not dispatch.hip_paged_available(torch.zeros(2, 4, 64, device=cuda, dtype=BF))
        assert not dispatch.hip_adjust_logits_available(torch.zeros(2, 64, device=cuda))
    finally:
        monkeypatch.undo()
        _lib.reset()
