"""CPU: how the INT8 and routing libraries and their compiled calls are built, with the compilers replaced; and which device
is current when those operators plan and launch."""

from __future__ import annotations

from pathlib import Path

import pytest
import torch

from piper_offload_b200 import build, int8, routing
from test_fp4_devices import Devices

OUTPUTS = ("OUT", "FP4_OUT", "CALLS_OUT", "INT8_OUT", "ROUTING_OUT", "EXPERT_CALLS_OUT")


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """The commands that a build runs, each of which leaves its output behind; outputs go to a folder of their own."""
    ran = []

    def run(cmd, **kwargs):
        ran.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("built")

    monkeypatch.setattr(build.subprocess, "run", run)
    for name in OUTPUTS:
        monkeypatch.setattr(build, name, tmp_path / getattr(build, name).name)
    return ran


def test_everything_is_built_once(commands):
    build.build(force=True)
    assert len(commands) == 6 and all(getattr(build, name).exists() for name in OUTPUTS)
    for cmd, source in zip(commands, ("merge.cu", "fp4.cu", "fp4_calls.cpp", "int8.cu", "routing.cu", "expert_calls.cpp")):
        assert any(part.endswith(source) for part in cmd)
        assert ("arch=compute_100a,code=sm_100a" in cmd) == source.endswith(".cu")
    for again in (build.build_int8, build.build_routing, build.build_expert_calls):
        again()
    assert len(commands) == 6


def test_calls_are_built_again_for_another_torch(commands, monkeypatch):
    build.build_expert_calls()
    build.build_expert_calls()
    assert len(commands) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.0")
    build.build_expert_calls()
    build.build_expert_calls()
    assert len(commands) == 2


def test_every_source_is_a_dependency():
    """What a source includes of this repository makes its library old when it changes."""
    import re

    for sources, deps in ((build.INT8_SOURCES, build.INT8_DEPS), (build.ROUTING_SOURCES, build.ROUTING_DEPS),
                          (build.EXPERT_CALLS_SOURCES, build.EXPERT_CALLS_DEPS)):
        seen, todo = set(), list(sources)
        while todo:
            path = todo.pop()
            if path in seen:
                continue
            seen.add(path)
            todo += [(path.parent / name).resolve() for name in re.findall(r'#include "([^"]+)"', path.read_text())]
        assert seen <= {p.resolve() for p in deps}, seen - set(deps)


@pytest.mark.parametrize("index", [0, 1])
def test_plans_and_launches_are_made_on_the_tensors_device(index, monkeypatch):
    devices, seen = Devices(), []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: devices.current)
    monkeypatch.setattr(torch.cuda, "device", devices.entered)
    monkeypatch.setattr(routing, "raw_stream", lambda i: i)

    def function(*args):
        seen.append((devices.current, args[0]))
        return int8.nat.OK

    device = torch.device("cuda", index)
    assert int8._workspace(function, device, 1, 2) is None
    int8._on(device, function, 1, 2)
    routing._call(function, device, 1)
    assert seen == [(index, 1)] * 3 and devices.current == 0
