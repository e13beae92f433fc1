"""The torch binding of the feature operators: only they need it, and it is built
again when torch or Python changed under it."""

import os
import shutil
import subprocess
import sys

import pytest

from dot_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def without_binding(tmp_path, binding=None):
    """A copy of the package with the C-ABI library and, as its torch binding, `binding` or none."""
    shutil.copytree(os.path.join(ROOT, "dot_b200"), tmp_path / "dot_b200",
                    ignore=shutil.ignore_patterns("_lib", "csrc", "__pycache__"))
    os.makedirs(tmp_path / "dot_b200" / "_lib")
    os.symlink(build.LIB, tmp_path / "dot_b200" / "_lib" / "libdot_b200.so")
    if binding is not None:
        (tmp_path / "dot_b200" / "_lib" / "_torch_features.so").write_bytes(binding)


def run(tmp_path, code):
    env = {**os.environ, "PYTHONPATH": str(tmp_path)}
    return subprocess.run([sys.executable, "-c", code], cwd=tmp_path, env=env, capture_output=True, text=True,
                          timeout=600)


CODE = """
import torch, dot_b200
from dot_b200 import Sinkhorn, bidirectional_softmax, sinkhorn, sinkhorn_points, GroupNormAct, Rotary
assert dot_b200._lib.load().dot_abi_version() == 1
GroupNormAct(2, 8), Rotary((2, 2))
for call in (lambda: dot_b200.group_norm_act(torch.rand(2, 4, 8), 2),
             lambda: dot_b200.rotary(torch.rand(1, 2, 8), torch.zeros(1, 1), torch.zeros(4, 1))):
    try:
        call()
    except ImportError as e:
        assert "build.py" in str(e), e
    else:
        raise AssertionError("no binding, no error")
print("fine")
"""


@pytest.mark.parametrize("binding", [None, b"not a library"], ids=["missing", "broken"])
def test_the_rest_of_the_package_runs_without_it(tmp_path, binding):
    without_binding(tmp_path, binding)
    out = run(tmp_path, CODE)
    assert out.returncode == 0 and "fine" in out.stdout, out.stderr


def test_it_is_built_again_for_another_torch(tmp_path, monkeypatch):
    compiled = []

    def compiler(cmd, check):
        compiled.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_torch_features.so"))
    monkeypatch.setattr(build, "BINDING_STAMP", str(tmp_path / "_torch_features.built_for"))
    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build_binding()
    build.build_binding()
    assert len(compiled) == 1          # it is there, for this torch
    (tmp_path / "_torch_features.built_for").write_text("torch 1.0, cpython-27")
    build.build_binding()
    assert len(compiled) == 2
    build.build_binding()
    assert len(compiled) == 2
    os.remove(tmp_path / "_torch_features.built_for")
    build.build_binding()
    assert len(compiled) == 3
