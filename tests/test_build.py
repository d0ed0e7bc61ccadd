"""CPU: when the compiled calls are built again, with which headers, and in what order the libraries are; the compilers
are replaced."""

from __future__ import annotations

from pathlib import Path

import pytest
import torch

from piper_offload_b200 import build


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """The commands that a build runs, each of which leaves its output behind; outputs go to a folder of their own."""
    ran = []

    def run(cmd, **kwargs):
        ran.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("built")

    monkeypatch.setattr(build.subprocess, "run", run)
    for name in ("OUT", "FP4_OUT", "CALLS_OUT"):
        monkeypatch.setattr(build, name, tmp_path / getattr(build, name).name)
    return ran


def test_calls_are_built_again_for_another_torch(commands, monkeypatch):
    build.build_calls()
    assert len(commands) == 1 and build.CALLS_OUT.read_text() == "built"
    build.build_calls()
    assert len(commands) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.0")
    build.build_calls()
    assert len(commands) == 2
    build.build_calls()
    assert len(commands) == 2
    # one that came without its record fits nothing for certain
    for p in build.CALLS_OUT.parent.iterdir():
        if p != build.CALLS_OUT:
            p.unlink()
    build.build_calls()
    assert len(commands) == 3


def test_calls_are_built_again_for_another_interpreter(commands, monkeypatch):
    build.build_calls()
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399-other")
    build.build_calls()
    assert len(commands) == 2


def test_a_failed_build_is_tried_again(commands, monkeypatch):
    build.build_calls()
    monkeypatch.setattr(torch, "__version__", "0.0.0")

    def fails(cmd, **kwargs):
        raise build.subprocess.CalledProcessError(1, cmd)

    with monkeypatch.context() as m:
        m.setattr(build.subprocess, "run", fails)
        for _ in range(2):
            with pytest.raises(build.subprocess.CalledProcessError):
                build.build_calls()
    build.build_calls()
    assert len(commands) == 2


def test_cuda_headers_come_from_the_compiler_that_is_found(commands, monkeypatch, tmp_path):
    """With nvcc on PATH alone its headers are the toolkit's beside it, through links too."""
    toolkit = tmp_path / "toolkit"
    (toolkit / "bin").mkdir(parents=True)
    real = toolkit / "bin" / "nvcc"
    real.write_text("#!/bin/sh\n")
    real.chmod(0o755)
    links = tmp_path / "links"
    links.mkdir()
    (links / "nvcc").symlink_to(real)
    monkeypatch.setenv("NVCC", str(tmp_path / "none"))
    for folder in (toolkit / "bin", links):
        monkeypatch.setenv("PATH", str(folder))
        build.build_calls(force=True)
        assert f"-I{toolkit / 'include'}" in commands[-1]


def test_the_merges_do_not_wait_for_the_calls_compiler(commands, monkeypatch):
    """Without a host compiler for the FP4 calls the merges' library is built all the same, and the error is raised."""
    run = build.subprocess.run

    def only_nvcc(cmd, **kwargs):
        if "nvcc" not in cmd[0]:
            raise FileNotFoundError(cmd[0])
        run(cmd, **kwargs)

    monkeypatch.setattr(build.subprocess, "run", only_nvcc)
    with pytest.raises(FileNotFoundError):
        build.build(force=True)
    assert build.OUT.exists() and build.FP4_OUT.exists() and not build.CALLS_OUT.exists()
