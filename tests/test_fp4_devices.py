"""CPU: which device is current when the FP4 operators plan and launch, with the library and the devices replaced."""

from __future__ import annotations

import pytest
import torch

from piper_offload_b200 import fp4


class Devices:
    """Two devices, of which the first is current."""

    def __init__(self):
        self.current = 0

    def entered(self, device):
        devices, index = self, torch.device(device).index

        class Guard:
            def __enter__(self):
                self.before, devices.current = devices.current, index

            def __exit__(self, *exc):
                devices.current = self.before

        return Guard()


@pytest.mark.parametrize("index", [0, 1])
def test_plans_and_launches_are_made_on_the_tensors_device(index, monkeypatch):
    devices, seen = Devices(), []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: devices.current)
    monkeypatch.setattr(torch.cuda, "device", devices.entered)
    monkeypatch.setattr(fp4.nat, "raw_stream", lambda i: i)

    def function(*args):
        seen.append(devices.current)
        return fp4.nat.OK

    device = torch.device("cuda", index)
    assert fp4._workspace(function, device, 1, 2) is None
    fp4._call(function, device, 1, 2)
    assert seen == [index, index] and devices.current == 0
