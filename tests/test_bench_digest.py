"""The digest that ties counter profiles to kernel sources: it changes with the profiled kernels' sources, and with
no others."""
import os
import shutil

import pytest

import bench

CSRC = os.path.join(os.path.dirname(os.path.abspath(bench.__file__)), "delta-block-lm_amd", "csrc")


@pytest.mark.parametrize("name,changes", [
    ("gdn2_chunk.hip", True), ("gdn2_chunk_f32.hip", True), ("gdn2_chunk_tile.h", True),
    ("gdn2_seq.hip", True), ("gdn2_api.hip", True), ("gdn2_mfma.h", True), ("gdn2_common.h", True),
    ("gdn2_linear.hip", False), ("gdn2_layernorm.hip", False), ("gdn2_q8.hip", False),
    ("gdn2_hola.hip", False), ("gdn2_of_its_own.hip", False)])
def test_what_the_digest_covers(tmp_path, monkeypatch, name, changes):
    root = tmp_path / "delta-block-lm_amd"
    shutil.copytree(CSRC, root / "csrc")
    monkeypatch.setattr(bench, "REPO", str(tmp_path))
    before = bench.sources_digest()
    with open(root / "csrc" / name, "a") as f:
        f.write("// changed\n")
    assert (bench.sources_digest() != before) == changes
