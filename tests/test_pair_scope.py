"""CPU: what the sources say of waits and barriers and no run can show. Between the two blocks of a pair an arrival in the other's
shared memory releases over the cluster, and who waits for it acquires so."""

from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "piper_offload_b200" / "csrc"


def test_arrivals_in_another_block_release_over_the_cluster():
    found = [m for path in sorted(CSRC.glob("*.cu*")) for m in re.findall(r"mbarrier\.arrive[\w.:]*\.shared::cluster[\w.:]*", path.read_text())]
    assert found and all(".release.cluster." in m for m in found), found


def test_pairs_wait_over_the_cluster():
    tiles = (CSRC / "int8_tiles.cuh").read_text()
    assert "mbarrier.try_wait.parity.acquire.cluster." in tiles
    # all waits of the product's pairs; of the gradient's kernel, which has both forms, all but that for the block's own warps
    assert "pm::mbar_wait(" not in (CSRC / "int8_pair.cuh").read_text()
    plain = re.findall(r"pm::mbar_wait\((&?\w+)", (CSRC / "int8_grad.cuh").read_text())
    assert plain == ["&ready"], plain


def test_the_next_launch_begins_after_the_allocation():
    """A launch that follows may allocate tensor memory before it waits for the one before it."""
    for name in ("int8_linear.cuh", "int8_pair.cuh", "int8_grad.cuh"):
        text = (CSRC / name).read_text()
        kernel = text[text.index("__global__"):]
        assert kernel.count("grid_launch_dependents()") == 1
        assert max(m.start() for m in re.finditer(r"tmem_alloc(_pair)?\(", kernel)) < kernel.index("__syncthreads()") < kernel.index("grid_launch_dependents()")
