"""When the host module is compiled again (nothing is compiled here)."""
import os
import subprocess

import pytest
import torch

from compressai_b200 import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A built host module that is newer than its sources, of this torch."""
    for name, value in (("HOST", tmp_path / "host.so"), ("HOST_STAMP", tmp_path / "key"), ("CSRC", tmp_path), ("INCLUDE", tmp_path)):
        monkeypatch.setattr(build, name, str(value))
    src = tmp_path / "attention_host.cpp"
    src.write_text("")
    os.utime(src, (1, 1))
    (tmp_path / "host.so").write_text("")
    (tmp_path / "key").write_text(build._host_key())
    runs = []

    def gxx(cmd, **kw):
        runs.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(build.subprocess, "run", gxx)
    return tmp_path, runs


def test_an_up_to_date_module_is_kept(tree):
    build._build_host(False)
    assert not tree[1]


def test_another_torch_rebuilds_it_once(tree, monkeypatch):
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build._build_host(False)
    build._build_host(False)
    assert len(tree[1]) == 1


@pytest.mark.parametrize("gone", ["key", "host.so"])
def test_a_missing_part_rebuilds_it(tree, gone):
    (tree[0] / gone).unlink()
    build._build_host(False)
    assert len(tree[1]) == 1


def test_a_newer_source_rebuilds_it(tree):
    os.utime(tree[0] / "attention_host.cpp", None)
    os.utime(tree[0] / "host.so", (2, 2))
    build._build_host(False)
    assert len(tree[1]) == 1
