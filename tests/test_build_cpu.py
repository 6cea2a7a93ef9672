"""Building the operators on torch tensors: left out where there is no CUDA
build of PyTorch, built again where another one has come."""
import os

import pytest

from snn_b200 import build


@pytest.fixture
def fake(tmp_path, monkeypatch):
    """A PyTorch with nothing but what the build looks for, and a compiler that only notes its calls."""
    t = tmp_path / "site" / "torch"
    (t / "include" / "ATen").mkdir(parents=True)
    (t / "include" / "ATen" / "ATen.h").write_text("")
    (t / "lib").mkdir()
    (t / "lib" / "libc10_cuda.so").write_text("")
    (t / "version.py").write_text("__version__ = '1'\n")
    (tmp_path / "obj").mkdir()
    calls = []

    def run(cmd, check):
        calls.append(cmd)
        with open(build.TORCH_OPS, "w") as f:
            f.write("")

    rest = [p for p in build.sys.path if not os.path.exists(os.path.join(p, "torch"))]
    monkeypatch.setattr(build.sys, "path", [str(tmp_path / "site")] + rest)
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "TORCH_OPS", str(tmp_path / "sequence_ops.so"))
    monkeypatch.setattr(build, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(build.subprocess, "run", run)
    return t, calls


def test_built_again_for_another_torch(fake, tmp_path):
    t, calls = fake
    build.build_torch_ops([], False, False)
    build.build_torch_ops([], False, False)
    assert len(calls) == 1 and os.path.join(str(t), "lib") in calls[0]
    (t / "version.py").write_text("__version__ = '2'\n")
    build.build_torch_ops([], False, False)
    assert len(calls) == 2
    os.rename(tmp_path / "site", tmp_path / "moved")
    build.sys.path[0] = str(tmp_path / "moved")
    build.build_torch_ops([], False, False)
    build.build_torch_ops([], False, False)
    assert len(calls) == 3
    build.build_torch_ops([], True, False)
    assert len(calls) == 4


@pytest.mark.parametrize("gone", ["include/ATen/ATen.h", "lib/libc10_cuda.so"])
def test_left_out_without_a_cuda_build_of_torch(fake, capsys, gone):
    t, calls = fake
    (t / gone).unlink()
    build.build_torch_ops([], False, False)
    build.build_torch_ops([], True, False)
    assert not calls
    assert "not built" in capsys.readouterr().err
