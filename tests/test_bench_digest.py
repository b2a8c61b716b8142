"""The digest that ties committed counter and power collections to kernel sources: it follows the measured steps' kernels, and nothing else."""
import os
import shutil

import bench


def test_digest_follows_the_steps_kernels_only(tmp_path, monkeypatch):
    for d in ("spurfies_amd/csrc", "include"):
        shutil.copytree(os.path.join(bench.ROOT, d), tmp_path / d)
    start = bench.csrc_digest()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    assert bench.csrc_digest() == start
    header = tmp_path / "include" / "spurfies_hip.h"
    text = header.read_text()
    assert text.count(bench.OTHER_SECTION) == 1
    for name in bench.OTHER_SOURCES:
        (tmp_path / "spurfies_amd/csrc" / name).write_text("// changed")
    header.write_text(text.replace("spf_wgrad8(", "spf_wgrad8_changed("))
    assert bench.csrc_digest() == start                                # operators that no measured step runs
    header.write_text(text.replace("spf_adam_step(", "spf_adam_step_changed("))
    assert bench.csrc_digest() != start
    header.write_text(text)
    (tmp_path / "spurfies_amd/csrc/grid.hip").write_text("// changed")
    assert bench.csrc_digest() != start


def test_other_sources_are_of_the_operators_alone():
    """No kernel of the measured steps includes them."""
    folder = os.path.join(bench.ROOT, "spurfies_amd", "csrc")
    for name in os.listdir(folder):
        if name not in bench.OTHER_SOURCES:
            text = open(os.path.join(folder, name)).read()
            assert not any(f'"{other}"' in text for other in bench.OTHER_SOURCES), name
