"""GPU: the results of a routing saved, loaded and kept, each by itself and all together."""

from __future__ import annotations

import copy
import dataclasses
import io

import pytest
import torch

import test_expert_calls_gpu as C
from piper_offload_b200 import routing

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("path", ["compiled", "written"])
def test_saved_and_loaded(path, cuda_device, monkeypatch):
    if path == "written":
        monkeypatch.setattr(routing, "calls", C.Declines)
    logits = torch.randn(50, 16, device=cuda_device, requires_grad=True)
    r = routing.route_tokens(logits, 4)
    kept = {f.name: getattr(r, f.name).detach() for f in dataclasses.fields(r)}
    file = io.BytesIO()
    torch.save(kept, file)
    file.seek(0)
    loaded = torch.load(file, weights_only=True)
    for name, t in kept.items():
        assert torch.equal(loaded[name], t) and loaded[name].dtype is t.dtype
        # nothing but its own values is saved, and kept alive, with a result
        assert t.untyped_storage().nbytes() == t.numel() * t.element_size() and t.storage_offset() == 0
    places = [t.untyped_storage().data_ptr() for t in kept.values()]
    assert len(set(places)) == len(places)
    again = copy.deepcopy(kept)
    assert all(torch.equal(again[name], t) for name, t in kept.items())
