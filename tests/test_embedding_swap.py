"""The embedding swap keeps the modules themselves: hooks, attributes and every name they go by (CPU)."""

from __future__ import annotations

import copy

import torch

from thundersync_amd.embedding import HipEmbedding, use_hip_embedding


class Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.shared = torch.nn.Embedding(10, 4)
        self.encoder = torch.nn.Module()
        self.encoder.embed = self.shared
        self.other = torch.nn.Embedding(6, 4, padding_idx=2)


def test_hooks_of_a_frozen_table_stay():
    """A forward hook that makes a frozen table's rows ask for gradients, as checkpointing below adapters needs it."""
    model = Model().requires_grad_(False)
    model.shared.register_forward_hook(lambda module, args, out: out.requires_grad_())
    calls = []
    model.shared.register_forward_pre_hook(lambda module, args: calls.append("pre"))
    model.shared.register_state_dict_pre_hook(lambda module, prefix, keep: calls.append("state"))
    model.shared.note = "kept"
    ids = torch.tensor([1, 2])
    want = model.shared(ids)
    assert use_hip_embedding(model) == 2
    out = model.shared(ids)
    assert out.requires_grad and torch.equal(out, want) and model.shared.note == "kept"
    model.state_dict()
    assert calls[:2] == ["pre", "pre"] and "state" in calls[2:]


def test_a_module_of_two_names_is_one():
    model = Model()
    module = model.shared
    assert use_hip_embedding(model) == 2
    assert model.shared is module is model.encoder.embed and type(module) is HipEmbedding
    assert type(model.other) is HipEmbedding and model.other.padding_idx == 2
    assert use_hip_embedding(model) == 0


def test_the_swapped_module_is_copied_and_saved_as_torchs(tmp_path):
    model = Model()
    names = list(model.state_dict())
    use_hip_embedding(model)
    twin = copy.deepcopy(model)
    assert type(twin.other) is HipEmbedding and twin.shared is twin.encoder.embed
    assert list(twin.state_dict()) == names and repr(model.other) == "HipEmbedding(6, 4, padding_idx=2)"
    torch.save(model.state_dict(), tmp_path / "state.pt")
    Model().load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
