"""Distillation from a teacher's top logits against the fp64 oracle, within its per-element bounds (``oracle.distill
.bounds``: the roundings of the logits' sums, of the stored gradient block and of the results)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import distill as ref
from thundersync_amd.fused_distill import fused_distill

pytestmark = pytest.mark.gpu

BF16, FP16, FP32, FP64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def inputs(n, d, v, k, dtype, seed=0, ragged=True, wscale=None):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, d, generator=g, dtype=FP64).to(dtype)
    w = (torch.randn(v, d, generator=g, dtype=FP64) * (wscale or 1.5 / math.sqrt(d))).to(dtype)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] if v >= k else torch.randint(0, v, (k,), generator=g)
                       for _ in range(n)]) if n else torch.zeros(0, k, dtype=torch.int64)
    teacher = torch.randn(n, k, generator=g) * 2
    grad = torch.rand(n, generator=g) + 0.5
    if ragged and n:
        have = torch.randint(0, k + 1, (n,), generator=g)
        have[::3] = k
        absent = torch.arange(k) >= have[:, None]
        ids = torch.where(absent & (torch.arange(n) % 2 == 0)[:, None], -1, ids)  # either mark of an absent slot
        teacher = torch.where(absent, -math.inf, teacher)
    return h, w, ids, teacher, grad


def run(cuda, h, w, ids, teacher, grad, train, **options):
    hc, wc = h.to(cuda).requires_grad_(), w.to(cuda).requires_grad_(train)
    loss = fused_distill(hc, wc, ids.to(cuda), teacher.to(cuda), **options)
    grads = torch.autograd.grad(loss, [hc, wc] if train else [hc], grad.to(cuda).to(loss.dtype))
    return [loss.detach(), *grads]


def check(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN where the other has none"
    excess = torch.nan_to_num((got - want).abs() - bound)
    assert (excess <= 0).all(), f"{what}: {excess.max().item():.3g} past its bound, error " \
                                f"{(got - want).abs().nan_to_num().max().item():.3g}"


def compare(cuda, case, dtype, train, temperature=1.0, chunk=1024):
    want = ref.distill(*case[:4], case[4], temperature)
    bound = ref.bounds(want, dtype, case[2].shape[1], temperature)
    got = run(cuda, *case, train, temperature=temperature, chunk=chunk)
    assert got[0].dtype == (dtype if dtype in (FP32, FP64) else FP32) and got[1].dtype == dtype
    check(got[0], want["loss"], bound["loss"], "loss")
    check(got[1], want["dh"], bound["dh"], "dh")
    if train:
        check(got[2], want["dw"], bound["dw"], "dw")


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32, FP64])
@pytest.mark.parametrize("n, d, v, k, temperature, chunk", [
    (1, 8, 1, 1, 1.0, 1024),          # one of everything
    (1, 64, 300, 5, 1.0, 1024),
    (3, 24, 255, 20, 0.7, 1),
    (65, 128, 257, 33, 2.0, 16),      # one past a token tile, one past a vocabulary tile
    (130, 72, 1000, 64, 1.0, 64),
    (300, 64, 4099, 7, 1.3, 100),     # several blocks of rows, the last short
    (700, 40, 513, 100, 1.0, 128),
])
def test_values_and_gradients(cuda, n, d, v, k, temperature, chunk, dtype, train):
    print(f"distill n={n} d={d} v={v} k={k} T={temperature} chunk={chunk} {dtype} train={train}", flush=True)
    compare(cuda, inputs(n, d, v, k, dtype, seed=n + v), dtype, train, temperature, chunk)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("k", [2, 1024])
def test_tokens_named_twice(cuda, dtype, k):
    """Slots of one token add up, in the loss and in the gradient."""
    print(f"distill tokens named twice k={k} {dtype}", flush=True)
    h, w, _, teacher, grad = inputs(9, 32, 50, k, dtype, ragged=False)
    ids = torch.randint(0, 50 if k > 2 else 1, (9, k), generator=torch.Generator().manual_seed(1))
    compare(cuda, (h, w, ids, teacher, grad), dtype, True)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_padded_widths_strides_and_types(cuda, dtype):
    """A hidden dim that is no multiple of 8, rows with gaps, int32 ids, teacher logits of other types and strides."""
    print(f"distill strides {dtype}", flush=True)
    h, w, ids, teacher, grad = inputs(20, 50, 333, 6, dtype)
    want = ref.distill(h, w, ids, teacher.to(BF16), grad)
    bound = ref.bounds(want, dtype, 6)
    hc = torch.zeros(20, 131, dtype=dtype)
    hc[:, 3:53] = h
    wc = torch.zeros(333, 60, dtype=dtype)
    wc[:, :50] = w
    big, wbig = hc.to(cuda).requires_grad_(), wc.to(cuda).requires_grad_()
    tc = torch.zeros(20, 9, dtype=BF16)
    tc[:, 2:8] = teacher.to(BF16)
    loss = fused_distill(big[:, 3:53], wbig[:, :50], ids.to(cuda).int(), tc.to(cuda)[:, 2:8])
    dh, dw = torch.autograd.grad(loss, (big, wbig), grad.to(cuda))
    check(loss, want["loss"], bound["loss"], "loss")
    check(dh[:, 3:53], want["dh"], bound["dh"], "dh")
    check(dw[:, :50], want["dw"], bound["dw"], "dw")
    assert dh[:, :3].abs().max() == 0 and dh[:, 53:].abs().max() == 0
    t_teacher = teacher.to(cuda).T.contiguous().T  # column-major
    again = fused_distill(h.to(cuda), w.to(cuda), ids.to(cuda).T.contiguous().T, t_teacher.double())
    check(again, ref.distill(h, w, ids, teacher, grad)["loss"], bound["loss"], "loss, column-major")


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32, FP64])
def test_rows_without_a_teacher_hold_anything(cuda, dtype, train):
    """Loss 0 and gradient 0 where no slot is present, also of rows of NaN and infinities with NaN upstream; the
    other rows and the weight's gradient do not see them."""
    print(f"distill empty rows {dtype} train={train}", flush=True)
    h, w, ids, teacher, grad = inputs(70, 32, 300, 5, dtype)
    ids[:7], teacher[7:9], ids[69] = -1, -math.inf, -5
    dead = torch.zeros(70, dtype=torch.bool)
    dead[:9] = dead[69] = True
    want = ref.distill(h, w, ids, teacher, grad)
    bound = ref.bounds(want, dtype, 5)
    h[0], h[1], h[2, 3], h[69] = math.nan, math.inf, -math.inf, math.nan
    grad[0] = math.nan
    loss, *grads = run(cuda, h, w, ids, teacher, grad, train)
    assert loss[dead].abs().max() == 0 and grads[0][dead].abs().max() == 0
    check(loss, want["loss"], bound["loss"], "loss")
    check(grads[0], want["dh"], bound["dh"], "dh")
    if train:
        check(grads[1], want["dw"], bound["dw"], "dw")


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_no_row_has_a_teacher(cuda, dtype, train):
    h, w, ids, teacher, grad = inputs(5, 16, 40, 3, dtype)
    loss, *grads = run(cuda, h, w, torch.full_like(ids, -1), teacher, grad, train)
    assert loss.abs().max() == 0 and all(g.abs().max() == 0 for g in grads)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_a_token_past_the_vocabulary(cuda, dtype, train, monkeypatch):
    """Its row's loss is NaN and its slot has no gradient term; the other rows are as they are."""
    h, w, ids, teacher, grad = inputs(6, 16, 40, 3, dtype, ragged=False)
    ids[2, 1], ids[4, 0] = 40, 1 << 40
    want = ref.distill(h, w, ids, teacher, grad)
    bound = ref.bounds(want, dtype, 3)
    got = run(cuda, h, w, ids, teacher, grad, train)
    assert torch.isnan(got[0]).nonzero().flatten().tolist() == [2, 4]
    check(got[0], want["loss"], bound["loss"], "loss")
    check(got[1], want["dh"], bound["dh"], "dh")
    monkeypatch.setenv("THUNDERSYNC_CHECK_TARGETS", "1")
    with pytest.raises(ValueError, match=r"target\[2\] = 40 is outside the vocabulary"):
        fused_distill(h.to(cuda), w.to(cuda), ids.to(cuda), teacher.to(cuda))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_nan_and_infinite_logits_surface(cuda, dtype):
    h, w, ids, teacher, grad = inputs(6, 16, 600, 3, dtype, ragged=False)
    teacher[1, 0], h[3] = math.nan, math.nan
    w[599] = math.nan  # every row's last logit
    got = run(cuda, h, w, ids, teacher, grad, False)
    assert torch.isnan(got[0]).all()
    w[599] = 0.0
    got = run(cuda, h, w, ids, teacher, grad, False)
    assert torch.isnan(got[0]).nonzero().flatten().tolist() == [1, 3]
    assert torch.isnan(got[1]).any(dim=1).nonzero().flatten().tolist() == [1, 3]


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("chunk", [4, 64])
def test_gradcheck(cuda, n, chunk):
    """fp64 against central differences."""
    h, w, ids, teacher, _ = inputs(n, 6, 11, 3, FP64)
    hc, wc = h.to(cuda).requires_grad_(), w.to(cuda).requires_grad_()
    ic, tc = ids.to(cuda), teacher.to(cuda)
    assert torch.autograd.gradcheck(lambda a, b: fused_distill(a, b, ic, tc, temperature=1.5, chunk=chunk), (hc, wc),
                                    eps=1e-6, atol=1e-8)
    assert torch.autograd.gradcheck(lambda a: fused_distill(a, w.to(cuda), ic, tc, chunk=chunk), (hc,), eps=1e-6,
                                    atol=1e-8)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_repeated_rows(cuda, dtype):
    """One hidden row for every teacher's row, one teacher's row for every hidden row: expanded tensors."""
    h, w, ids, teacher, grad = inputs(12, 40, 300, 5, dtype, ragged=False)
    want = ref.distill(h[:1].expand(12, 40), w, ids[:1].expand(12, 5), teacher[:1].expand(12, 5), grad)
    bound = ref.bounds(want, dtype, 5)
    for train in (False, True):
        hc = h[:1].to(cuda).requires_grad_()
        wc = w.to(cuda).requires_grad_(train)
        loss = fused_distill(hc.expand(12, 40), wc, ids[:1].to(cuda).expand(12, 5), teacher[:1].to(cuda).expand(12, 5))
        (dh,) = torch.autograd.grad(loss, hc, grad.to(cuda))
        check(loss, want["loss"], bound["loss"], "loss")
        # twelve rounded gradients added by torch, in the element type
        u = torch.finfo(dtype).eps / 2
        total = want["dh"].sum(0, keepdim=True)
        check(dh, total, bound["dh"].sum(0, keepdim=True) + 12 * u * want["dh"].abs().sum(0, keepdim=True), "dh")
    one = fused_distill(h[:1].to(cuda).expand(1, 40), w.to(cuda), ids[:1].to(cuda), teacher[:1].to(cuda))
    check(one, want["loss"][:1], bound["loss"][:1], "one row")


def test_two_calls_at_once(cuda):
    """Calls on two streams, each with its own gradients, interleaved: neither sees the other."""
    case = [t.to(cuda) for t in inputs(200, 64, 2000, 9, BF16)]
    want = [run(cuda, *case, train) for train in (False, True)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(run(cuda, *case, bool(i)))
    torch.cuda.synchronize()
    for results, w in zip(got, want):
        assert all(torch.equal(a, b) for r in results for a, b in zip(r, w))


def test_no_rows(cuda):
    for dtype in (BF16, FP32):
        h, w, ids, teacher, grad = inputs(0, 16, 40, 3, dtype)
        loss, dh, dw = run(cuda, h, w, ids, teacher, grad, True)
        assert loss.shape == (0,) and dh.shape == (0, 16) and dw.shape == (40, 16) and dw.abs().max() == 0


@pytest.mark.parametrize("dtype, train", [(BF16, False), (BF16, True), (FP32, False), (FP32, True)])
def test_backward_twice_and_repeatable(cuda, dtype, train):
    """A graph that is kept can be walked again, with another upstream gradient; the same bits every time."""
    h, w, ids, teacher, grad = inputs(150, 48, 700, 9, dtype)
    hc, wc = h.to(cuda).requires_grad_(), w.to(cuda).requires_grad_(train)
    leaves = [hc, wc] if train else [hc]
    loss = fused_distill(hc, wc, ids.to(cuda), teacher.to(cuda))
    g = grad.to(cuda)
    one = torch.autograd.grad(loss, leaves, g, retain_graph=True)
    torch.autograd.grad(loss, leaves, 3 * g, retain_graph=True)
    two = torch.autograd.grad(loss, leaves, g)
    fresh = run(cuda, h, w, ids, teacher, grad, train)
    assert torch.equal(loss, fresh[0])
    for a, b, c in zip(one, two, fresh[1:]):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_without_gradients(cuda):
    """The same losses where no gradient is asked for."""
    h, w, ids, teacher, grad = inputs(100, 64, 900, 9, BF16)
    loss = run(cuda, h, w, ids, teacher, grad, False)[0]
    hc = h.to(cuda).requires_grad_()
    with torch.no_grad():
        assert torch.equal(fused_distill(hc, w.to(cuda), ids.to(cuda), teacher.to(cuda)), loss)
    plain = fused_distill(h.to(cuda), w.to(cuda), ids.to(cuda), teacher.to(cuda))
    assert torch.equal(plain, loss) and not plain.requires_grad


def test_gradient_of_the_weight_alone(cuda):
    h, w, ids, teacher, grad = inputs(100, 64, 900, 9, BF16)
    want = ref.distill(h, w, ids, teacher, grad)
    wc = w.to(cuda).requires_grad_()
    loss = fused_distill(h.to(cuda), wc, ids.to(cuda), teacher.to(cuda))
    (dw,) = torch.autograd.grad(loss, wc, grad.to(cuda))
    check(dw, want["dw"], ref.bounds(want, BF16, 9)["dw"], "dw")


@pytest.mark.parametrize("train", [False, True])
def test_in_a_graph_and_on_another_stream(cuda, train):
    """A captured forward and backward, replayed between eager work, against the eager result."""
    print(f"distill capture train={train}", flush=True)
    h, w, ids, teacher, grad = (t.to(cuda) for t in inputs(90, 64, 900, 9, BF16))

    def step():
        hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_(train)
        loss = fused_distill(hg, wg, ids, teacher)
        return [loss.detach(), *torch.autograd.grad(loss, [hg, wg] if train else [hg], grad)]

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
    first = h.clone()
    for shift in (0.0, 0.25, -0.5, 0.0):
        h.copy_(first + shift)
        graph.replay()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        torch.cuda.synchronize()


@pytest.mark.parametrize("n, k, dtype", [(48, 20, BF16), (281, 64, BF16), (600, 5, FP16)])
def test_full_vocabulary(cuda, n, k, dtype):
    """A wide head, against the formula in fp64 on the GPU on sampled rows (a row's loss and gradient are its own)."""
    print(f"distill full vocabulary n={n} k={k} {dtype}", flush=True)
    d, v = 1024, 151936
    g = torch.Generator(device=cuda).manual_seed(n)
    h = torch.randn(n, d, generator=g, device=cuda).to(dtype).requires_grad_()
    w = (torch.randn(v, d, generator=g, device=cuda) * 0.05).to(dtype)
    ids = torch.randint(0, v, (n, k), generator=g, device=cuda)
    ids[:, 0] = v - 1  # the last token of the last tile
    teacher = torch.randn(n, k, generator=g, device=cuda) * 2
    loss = fused_distill(h, w, ids, teacher)
    (dh,) = torch.autograd.grad(loss.sum(), h)
    rows = torch.tensor([0, 1, n // 2, n - 1])
    want = ref.distill(h.detach()[rows].cpu(), w.cpu(), ids[rows].cpu(), teacher[rows].cpu(), torch.ones(4))
    bound = ref.bounds(want, dtype, k)
    check(loss[rows], want["loss"], bound["loss"], "loss")
    check(dh[rows], want["dh"], bound["dh"], "dh")
