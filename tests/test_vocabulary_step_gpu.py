"""Sampling, embedding and distillation together, as an on-policy distillation step uses them."""

from __future__ import annotations

import pytest
import torch

from oracle import distill as ref_distill
from oracle import embedding as ref_embedding
from oracle import sampling as ref_sampling
from thundersync_amd import dispatch, forest
from thundersync_amd.embedding import embedding, use_hip_embedding
from thundersync_amd.fused_distill import fused_distill
from thundersync_amd.fused_logprob import fused_logprob
from thundersync_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n, v, d, k", [(40, 300, 48, 7), (300, 1025, 32, 20)])
def test_a_step_with_a_tied_table(cuda, n, v, d, k):
    """Tokens drawn from the head, looked up in the table that is also the head, distilled: the table's gradient is
    the lookup's and the head's, within the sum of their bounds."""
    print(f"vocabulary step n={n} v={v} d={d} k={k}", flush=True)
    g = torch.Generator().manual_seed(n)
    table = torch.randn(v, d, generator=g)
    mix = torch.randn(d, d, generator=g) / d ** 0.5
    start = torch.randn(n, d, generator=g)
    u = torch.rand(n, generator=g)
    teacher = torch.randn(n, k, generator=g)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    weight = table.to(cuda).requires_grad_()
    with torch.no_grad():
        logits = start.to(cuda) @ weight.T
    tokens, logprobs = sample_tokens(logits, u.to(cuda), temperature=0.9, top_k=50, top_p=0.95)
    want = [ref_sampling.sample(r, float(x), 0.9, 50, 0.95)[0] for r, x in zip(logits.cpu().double().numpy(), u)]
    assert tokens.tolist() == want
    # drawn without filters, a token's logprob is the fused logprob's: the two products' sums of D terms apart
    free, logprobs = sample_tokens(logits, u.to(cuda))
    scored = fused_logprob(start.to(cuda), weight.detach(), free)
    size = (start.abs() @ table.abs().T).max()
    assert (scored - logprobs).abs().max() <= 4 * (d + v + 8) * 2.0 ** -24 * (1 + size)

    x = embedding(tokens, weight, scale=d ** 0.5)
    h = x @ mix.to(cuda)
    h.retain_grad()
    loss = fused_distill(h, weight, ids.to(cuda), teacher.to(cuda))
    grad = torch.full((n,), 1.0 / n)
    loss.backward(grad.to(cuda))
    # the head's part from the hidden states that it saw, the lookup's from the gradient that came back to it
    ref = ref_distill.distill(h.detach().cpu(), table, ids, teacher, grad)
    bound = ref_distill.bounds(ref, torch.float32, k)
    assert ((loss.detach().cpu().double() - ref["loss"]).abs() <= bound["loss"]).all()
    assert ((h.grad.cpu().double() - ref["dh"]).abs() <= bound["dh"]).all()
    dx = h.grad.cpu().double() @ mix.double().T
    dx_bound = (d + 2) * 2.0 ** -24 * (h.grad.cpu().double().abs() @ mix.double().abs().T)
    scale = d ** 0.5
    looked = ref_embedding.gradient(tokens.cpu(), dx, v, scale)
    looked_bound = ref_embedding.gradient(tokens.cpu(), dx_bound, v, scale) + \
        ref_embedding.gradient_bound(tokens.cpu(), dx.float(), v, scale) * (1 + 2.0 ** -20)
    both, both_bound = ref["dw"] + looked, bound["dw"] + looked_bound
    assert ((weight.grad.cpu().double() - both).abs() <= both_bound + 2.0 ** -24 * both.abs()).all()


def test_forest_distillation_in_a_model(cuda):
    """A forest's losses are those of its scored hidden states, in logical order; a swapped embedding does not change
    them, and gradients reach the table."""
    transformers = pytest.importorskip("transformers")
    from thundersync_amd.attention import HIP_FOREST_ATTENTION_NAME, register_attention
    from thundersync_amd.step import forest_distillation, split_by_trajectory

    print("forest distillation", flush=True)
    cfg = transformers.Qwen3Config(vocab_size=96, hidden_size=256, intermediate_size=384, num_hidden_layers=1,
                                   num_attention_heads=4, num_key_value_heads=1, head_dim=128,
                                   tie_word_embeddings=True)
    torch.manual_seed(0)
    model = transformers.Qwen3ForCausalLM(cfg).to(cuda, torch.bfloat16)
    register_attention()
    model.set_attn_implementation(HIP_FOREST_ATTENTION_NAME)
    trajs = [forest.Trajectory([forest.Segment.prompt(list(range(1, 40))), forest.Segment.action(body)], group_id=0,
                               traj_id=t) for t, body in enumerate(([4, 5, 6], [4, 5, 7, 8], [9]))]
    plan = forest.compile_plan(forest.build_forest(trajs)).to(cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    s = plan.score_src.numel()
    ids = torch.randint(0, 96, (s, 5), generator=g, device=cuda)
    teacher = torch.randn(s, 5, generator=g, device=cuda)
    seen = {}

    def hidden_fn(tokens, pos):
        seen["h"] = model.model(input_ids=tokens[None], position_ids=pos[None], use_cache=False).last_hidden_state[0]
        return seen["h"]

    stock = forest_distillation(model, plan, ids, teacher, temperature=1.5, hidden_fn=hidden_fn)
    direct = fused_distill(seen["h"][plan.score_src], model.lm_head.weight, ids, teacher, temperature=1.5)
    assert torch.equal(stock, direct[plan.logical_to_slot])
    assert use_hip_embedding(model) == 1 and model.lm_head.weight is model.model.embed_tokens.weight
    swapped = forest_distillation(model, plan, ids, teacher, temperature=1.5)
    assert torch.equal(swapped, stock)
    assert [x.numel() for x in split_by_trajectory(plan, swapped).values()] == [3, 4, 1]
    swapped.sum().backward()
    assert model.model.embed_tokens.weight.grad.isfinite().all()
    with pytest.raises(ValueError, match="one row per scored position"):
        forest_distillation(model, plan, ids[1:], teacher[1:])


def test_availability(cuda, monkeypatch):
    from thundersync_amd import _lib

    for dtype in (torch.bfloat16, torch.float32):
        like = torch.zeros(2, 64, device=cuda, dtype=dtype)
        assert dispatch.hip_distill_available(like)
        assert dispatch.hip_embedding_available(like)
        assert dispatch.hip_sampling_available(like)
    assert not dispatch.hip_embedding_available(torch.zeros(2, 64, device=cuda, dtype=torch.float64))
    assert not dispatch.hip_sampling_available(torch.zeros(2, 64))
    monkeypatch.setenv("THUNDERSYNC_HIP", "off")
    _lib.reset()
    try:
        assert not dispatch.hip_distill_available(torch.zeros(2, 64, device=cuda))
        with pytest.raises(RuntimeError, match="switched off"):
            sample_tokens(torch.zeros(1, 4, device=cuda), torch.zeros(1, device=cuda))
    finally:
        monkeypatch.undo()
        _lib.reset()
