"""The module of the 8-bit cache's common calls (``csrc/quantised_calls.cpp``): how it is built, and what happens where it cannot be."""

import threading

import pytest
import torch

from clockwork_b200.csrc import build
from clockwork_b200.ops import quantised


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


def _no_compiler(monkeypatch, tmp_path):
    out = tmp_path / "out"
    out.mkdir()
    monkeypatch.setattr(build, "build_dir", lambda: out)
    monkeypatch.setattr(quantised, "_calls_module", None)
    monkeypatch.setenv("CXX", _compiler(tmp_path, "exit 1\n"))


def test_without_a_compiler_calls_say_so_once(tmp_path, monkeypatch):
    _no_compiler(monkeypatch, tmp_path)
    monkeypatch.setattr(quantised, "library", lambda: None)
    monkeypatch.setattr(build, "find_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    with pytest.warns(RuntimeWarning, match="unavailable"):
        calls = quantised._calls()
    assert quantised._calls() is calls
    assert all(getattr(calls, name)(1, 2, 3) is None for name in ("store", "step", "decode", "read", "portions"))


@pytest.mark.gpu
def test_without_a_compiler_the_kernels_still_run(tmp_path, monkeypatch):
    from clockwork_b200 import ops

    ops.library()
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(3, 16 * 64, generator=g).bfloat16().cuda()
    at = torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda")
    outs = []
    for missing in (False, True):
        if missing:
            _no_compiler(monkeypatch, tmp_path)
        cache, status = quantised.allocate_pages(4, 16, 2, 64, "cuda"), ops.new_status("cuda")
        tables, ctx = torch.tensor([[0], [1], [2]], dtype=torch.int32, device="cuda"), at + 1
        slots = torch.tensor([0, 16 + 5, 32 + 9], dtype=torch.int32, device="cuda")

        def run():
            out = quantised.decode_step(qkv, at, slots, None, cache, tables, ctx, 12, 2, 64, 0.125, status)
            plan = quantised.plan_portions([1, 1, 1], [1, 6, 10], 12, 2, 64, 16, torch.device("cuda"), most_rows=0)
            back = [torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
            quantised.read_pages(cache, tables, ctx, *back, status)
            return [out, quantised.attention_portions(out, cache, tables, torch.arange(4, dtype=torch.int32, device="cuda"), ctx, plan, 12, 0.125, status), *back]

        if missing:
            with pytest.warns(RuntimeWarning, match="unavailable"):
                outs.append(run())
        else:
            outs.append(run())
        ops.raise_on_status(status)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
