"""Embedding lookup (bit-exact) and its gradient by sorted tokens against the oracle."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import embedding as ref
from thundersync_amd import _lib
from thundersync_amd.embedding import HipEmbedding, embedding, embedding_backward, use_hip_embedding

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def inputs(n, v, d, dtype, kind="skewed", seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(v, d, generator=g).to(dtype)
    if kind == "skewed":
        ids = (torch.rand(n, generator=g) ** 4 * v).long().clamp(max=v - 1)
    elif kind == "one":
        ids = torch.full((n,), v // 2)
    elif kind == "distinct":
        ids = torch.randperm(v, generator=g)[torch.arange(n) % v]
    else:
        ids = torch.randint(0, v, (n,), generator=g)
    return ids, w, torch.randn(n, d, generator=g).to(dtype)


def same_bits(a, b):
    a, b = a.detach().cpu(), b.detach().cpu()
    kind = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(
        torch.nan_to_num(a).contiguous().view(kind), torch.nan_to_num(b).contiguous().view(kind)) and torch.equal(
        a.isnan(), b.isnan())


def check_gradient(got, ids, dout, v, scale=1.0, padding_idx=None):
    want = ref.gradient(ids, dout, v, scale, padding_idx)
    bound = ref.gradient_bound(ids, dout, v, scale, padding_idx)
    off = (got.cpu().double() - want).abs()
    assert got.shape == want.shape and (off <= bound).all(), f"{(off - bound).max().item():.3g} past its bound"
    untouched = torch.bincount(ids.reshape(-1)[(ids.reshape(-1) >= 0) & (ids.reshape(-1) < v)], minlength=v) == 0
    assert got.cpu()[untouched].abs().sum() == 0


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("n, v, d, kind, scale", [
    (1, 1, 1, "any", 1.0),
    (1, 1000, 64, "any", 1.0),
    (2, 5, 7, "any", 0.5),            # a width of no whole vector
    (33, 500, 40, "one", 1.0),        # one token, one past a chunk of positions
    (64, 600, 128, "distinct", 11.3),
    (1000, 1023, 100, "skewed", math.sqrt(100)),
    (2049, 513, 64, "skewed", 1.0),   # one past a sort tile, two digits
    (5000, 3, 72, "any", 1.0),        # runs that cross many chunks
    (5000, 300000, 16, "any", 1.0),   # three digits
    (40000, 2000, 24, "skewed", 1.0),
    (4096, 4096, 8, "one", 1.0),
])
def test_lookup_and_gradient(cuda, n, v, d, kind, scale, dtype):
    print(f"embedding n={n} v={v} d={d} {kind} scale={scale} {dtype}", flush=True)
    ids, w, dout = inputs(n, v, d, dtype, kind, seed=n + v)
    wc = w.to(cuda).requires_grad_()
    out = embedding(ids.to(cuda), wc, scale=scale)
    assert same_bits(out, ref.lookup(ids, w, scale))
    (grad,) = torch.autograd.grad(out, wc, dout.to(cuda))
    assert grad.dtype == dtype
    check_gradient(grad, ids, dout, v, scale)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_shapes_strides_and_id_types(cuda, dtype):
    """ids of any shape and stride and of int32, a table with gaps between its rows, upstream gradients of every layout."""
    print(f"embedding strides {dtype}", flush=True)
    ids, w, dout = inputs(60, 50, 24, dtype)
    grid = ids.reshape(3, 4, 5)
    wide = torch.zeros(50, 31, dtype=dtype)
    wide[:, 5:29] = w
    wc = wide.to(cuda).requires_grad_()
    out = embedding(grid.to(cuda).permute(2, 0, 1).int(), wc[:, 5:29])
    assert same_bits(out, ref.lookup(grid.permute(2, 0, 1), w))
    up = dout.reshape(5, 3, 4, 24)
    (grad,) = torch.autograd.grad(out, wc, up.to(cuda))
    check_gradient(grad[:, 5:29].contiguous(), grid.permute(2, 0, 1), up, 50)
    assert grad[:, :5].abs().sum() == 0 and grad[:, 29:].abs().sum() == 0
    for layout in (dout.to(cuda).T.contiguous().T, torch.cat([dout, dout], 1).to(cuda)[:, 24:],
                   dout[:1].to(cuda).expand(60, 24), dout[:, :1].to(cuda).expand(60, 24)):
        got = embedding_backward(ids.to(cuda), layout, 50)
        check_gradient(got, ids, layout.cpu(), 50)
    scalar = embedding(torch.tensor(7, device=cuda), w.to(cuda))
    assert same_bits(scalar, ref.lookup(torch.tensor(7), w))
    misaligned = torch.zeros(60 * 24 + 1, dtype=dtype, device=cuda)[1:].view(60, 24)
    misaligned.copy_(dout)
    check_gradient(embedding_backward(ids.to(cuda), misaligned, 50), ids, dout, 50)


def test_no_tokens_and_sum(cuda):
    w = torch.randn(10, 16, device=cuda).to(BF16).requires_grad_()
    out = embedding(torch.zeros(2, 0, dtype=torch.int64, device=cuda), w)
    assert out.shape == (2, 0, 16)
    (grad,) = torch.autograd.grad(out.sum(), w)
    assert grad.shape == (10, 16) and grad.abs().sum() == 0
    ids = torch.tensor([3, 3, 9], device=cuda)
    (grad,) = torch.autograd.grad(embedding(ids, w).sum(), w)  # an expanded upstream gradient
    assert grad[3].eq(2).all() and grad[9].eq(1).all() and grad.sum() == 48


def test_padding_and_ids_outside_the_table(cuda, monkeypatch):
    """The padding row is looked up but not trained; ids outside the table give NaN rows and no gradient."""
    ids, w, dout = inputs(500, 40, 16, BF16)
    ids[::7] = 3
    wc = w.to(cuda).requires_grad_()
    out = embedding(ids.to(cuda), wc, padding_idx=3)
    assert same_bits(out, ref.lookup(ids, w))
    (grad,) = torch.autograd.grad(out, wc, dout.to(cuda))
    check_gradient(grad, ids, dout, 40, padding_idx=3)
    assert grad[3].abs().sum() == 0
    ids[5], ids[6], ids[7], ids[8] = -1, 40, 1 << 40, -(1 << 33)
    out = embedding(ids.to(cuda), wc)
    assert same_bits(out, ref.lookup(ids, w)) and out[5:9].isnan().all()
    dout[5:9] = math.nan
    (grad,) = torch.autograd.grad(out, wc, dout.to(cuda))
    clean = dout.clone()
    clean[5:9] = 0
    check_gradient(grad, ids, clean, 40)
    monkeypatch.setenv("THUNDERSYNC_CHECK_TARGETS", "1")
    with pytest.raises(ValueError, match=r"target\[5\] = -1 is outside"):
        embedding(ids.to(cuda), wc)


def test_tables_of_one_row_and_none(cuda):
    w = torch.randn(1, 24, device=cuda).to(BF16).requires_grad_()
    ids = torch.zeros(5000, dtype=torch.int64, device=cuda)
    out = embedding(ids, w)
    assert same_bits(out, ref.lookup(ids.cpu(), w.detach().cpu()))
    dout = torch.randn(5000, 24, device=cuda).to(BF16)
    (grad,) = torch.autograd.grad(out, w, dout)
    check_gradient(grad, ids.cpu(), dout.cpu(), 1)
    (grad,) = torch.autograd.grad(embedding(ids, w, padding_idx=0), w, dout)  # no token takes part
    assert grad.abs().sum() == 0
    empty = torch.zeros(0, 8, device=cuda, requires_grad=True)
    out = embedding(ids[:3], empty)
    assert out.shape == (3, 8) and out.isnan().all()
    assert torch.autograd.grad(out.sum(), empty)[0].shape == (0, 8)


def test_backward_twice(cuda):
    ids, w, dout = (t.to(cuda) for t in inputs(3000, 500, 40, FP16))
    w.requires_grad_()
    out = embedding(ids, w)
    one = torch.autograd.grad(out, w, dout, retain_graph=True)[0]
    assert torch.equal(one, torch.autograd.grad(out, w, dout)[0])


@pytest.mark.parametrize("n, v, d", [(300000, 1200, 16), (2048, 511, 8), (2049, 512, 8), (20000, 262143, 8)])
def test_sort_sizes(cuda, n, v, d):
    """Many tiles, exactly one, one more, and a vocabulary at a digit's edge."""
    print(f"embedding sort n={n} v={v}", flush=True)
    ids, w, dout = inputs(n, v, d, FP32, "any", seed=3)
    got = embedding_backward(ids.to(cuda), dout.to(cuda), v)
    check_gradient(got, ids, dout, v)


def test_gradient_against_differences(cuda):
    """The lookup is linear: <dW, X> = <dout, lookup(X)>."""
    ids, w, dout = (t.to(cuda) for t in inputs(300, 64, 32, FP32))
    x = torch.randn(64, 32, device=cuda)
    grad = embedding_backward(ids, dout, 64, scale=2.0)
    one = (grad.double() * x.double()).sum()
    two = (dout.double() * embedding(ids, x, scale=2.0).double()).sum()
    # every product is off by its two factors' roundings: 300 * 32 terms of about 2
    assert abs(one - two) <= 2.0 ** -22 * (dout.abs().double() * embedding(ids, x.abs(), scale=2.0)).sum()


@pytest.mark.parametrize("kind", ["one", "skewed"])
def test_the_same_bits_every_time(cuda, kind):
    ids, w, dout = (t.to(cuda) for t in inputs(20000, 3000, 64, BF16, kind))
    first = embedding_backward(ids, dout, 3000)
    for _ in range(3):
        assert torch.equal(first, embedding_backward(ids, dout, 3000))


@pytest.mark.parametrize("n", [100, 5000, 40000])
def test_in_a_graph_and_on_another_stream(cuda, n):
    print(f"embedding capture n={n}", flush=True)
    ids, w, dout = (t.to(cuda) for t in inputs(n, 700, 64, BF16))

    def step():
        leaf = w.detach().requires_grad_()
        out = embedding(ids, leaf, scale=3.0)
        return [out.detach(), *torch.autograd.grad(out, leaf, dout)]

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for shift in (0, 1, 17, 0):
        ids.add_(shift).remainder_(700)
        graph.replay()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        torch.cuda.synchronize()


def test_module_swap(cuda):
    """A swapped module's outputs and gradients, its tied head, and the types it leaves to torch."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Embedding(40, 16, padding_idx=2), torch.nn.Linear(16, 40, bias=False))
    model[1].weight = model[0].weight
    model = model.to(cuda, BF16)
    ids = torch.randint(0, 40, (4, 9), device=cuda)
    want = model[0](ids)
    assert use_hip_embedding(model) == 1 and isinstance(model[0], HipEmbedding)
    with _lib.KernelTimer() as timer:
        got = model[0](ids)
        torch.cuda.synchronize()
        assert timer.read("embedding.lookup_kernel")[1] == 1
    assert torch.equal(got, want) and model[0].weight is model[1].weight
    model(ids).float().square().sum().backward()
    assert model[0].weight.grad.isfinite().all()
    double = model.double()
    assert double[0](ids).dtype == torch.float64
