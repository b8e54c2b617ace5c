"""Operands whose rows are narrower than a stage of the matrix core (32 elements) at the very end of their memory: the
rows that a tile has past the last one are not read.  (Read, they lay up to 48 bytes past the operand, which faults
where a mapping ends there.)"""

from __future__ import annotations

import pytest
import torch

from thundersync_amd.fused_distill import fused_distill
from thundersync_amd.fused_logprob import fused_logprob

pytestmark = pytest.mark.gpu

SEGMENT = 32 << 20  # torch gives an allocation of this size a mapping of its own


def at_the_end(t):
    """``t`` in the last bytes of a mapping."""
    buffer = torch.empty(SEGMENT // t.element_size(), dtype=t.dtype, device=t.device)
    out = buffer[buffer.numel() - t.numel():].view(t.shape)
    return out.copy_(t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n, d, v", [(64, 8, 64), (1, 8, 1), (300, 16, 1000), (65, 24, 257), (128, 8, 2)])
def test_narrow_rows(cuda, n, d, v, dtype):
    print(f"narrow operands n={n} d={d} v={v} {dtype}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(n)
    h = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    w = torch.randn(v, d, generator=g, device=cuda).to(dtype)
    target = torch.randint(0, v, (n,), generator=g, device=cuda)
    teacher = torch.randn(n, 2, generator=g, device=cuda)

    def run(h, w, chunk):
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        lp = fused_logprob(h, w, target, chunk=chunk)
        out = [lp, *torch.autograd.grad(lp.sum(), (h, w))]
        loss = fused_distill(h, w, target[:, None].expand(n, 2), teacher, chunk=chunk)
        out += [loss, *torch.autograd.grad(loss.sum(), (h, w))]
        frozen = fused_distill(h, w.detach(), target[:, None].expand(n, 2), teacher, chunk=chunk)
        return [t.detach() for t in [*out, *torch.autograd.grad(frozen.sum(), h)]]

    for chunk in (1024, 32):
        got, want = run(at_the_end(h), at_the_end(w), chunk), run(h, w, chunk)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
