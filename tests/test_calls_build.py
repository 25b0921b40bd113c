"""The module of the 8-bit cache's common calls (``csrc/quantised_calls.cpp``): how it is built, and what happens where it cannot be."""

import threading

import pytest

from clockwork_b200.csrc import build


def _compiler(folder, body):
    path = folder / "cxx"
    path.write_text("#!/bin/sh\n" + body)
    path.chmod(0o755)
    return str(path)


def test_threads_that_build_at_once_write_files_of_their_own(tmp_path, monkeypatch):
    out = tmp_path / "out"
    out.mkdir()
    monkeypatch.setattr(build, "build_dir", lambda: out)
    # (a compiler that notes where it writes, and takes its time over it)
    monkeypatch.setenv("CXX", _compiler(tmp_path, f'while [ "$1" != "-o" ]; do shift; done\necho "$2" >> {tmp_path}/written\nprintf half > "$2"\nsleep 0.3\nprintf whole > "$2"\n'))
    monkeypatch.setattr(build, "find_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    threads = [threading.Thread(target=build.ensure_calls_built) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    written = (tmp_path / "written").read_text().split()
    assert len(written) == 3 and len(set(written)) == 3
    assert (out / f"{build.CALLS_NAME}.so").read_text() == "whole" and {p.name for p in out.iterdir()} == {f"{build.CALLS_NAME}.so", f"{build.CALLS_NAME}.so.digest"}
