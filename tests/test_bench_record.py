"""bench.py quotes measured traffic for the build that it was measured on only."""
import os
import shutil

import bench


def test_hash_goes_by_sources_and_flags(tmp_path, monkeypatch):
    csrc = os.path.join("recommender_amd", "csrc")
    os.makedirs(tmp_path / csrc)
    for name in ("epoch.hip", "common.h", "Makefile"):
        shutil.copy(os.path.join(bench.ROOT, csrc, name), tmp_path / csrc / name)
    here = bench.kernel_source_hash()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    assert bench.kernel_source_hash() == here

    def changed(name, old, new):
        path = tmp_path / csrc / name
        was = path.read_text()
        assert old in was
        path.write_text(was.replace(old, new, 1))
        got = bench.kernel_source_hash()
        path.write_text(was)
        return got != here
    assert changed("Makefile", "-O3", "-O2") and changed("Makefile", "-Xclang -packed-fp32-ops", "")
    assert changed("Makefile", "ARCH ?= gfx950", "ARCH ?= gfx942") and changed("epoch.hip", "{", "{ ") and changed("common.h", "{", "{ ")
    assert not changed("Makefile", "SRCS := prep.hip", "SRCS := extra.hip prep.hip")         # other files, other targets, comments
