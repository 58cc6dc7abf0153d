"""The build of the decoder operators' Python extension: where it cannot be built the library still is, another torch or
interpreter does not get a stale one."""
import subprocess
import sys
import sysconfig

import pytest
import torch

from dracomancer_llmengine_b200 import build


@pytest.fixture
def calls(monkeypatch, tmp_path):
    """Compiler calls, recorded instead of made."""
    made = []

    def run(cmd, **_):
        made.append(cmd)
        open(cmd[cmd.index("-o") + 1], "wb").close()

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "PKG", str(tmp_path))
    monkeypatch.setattr(build, "EXT", str(tmp_path / "_decoder.tag.so"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path))
    monkeypatch.setattr(build, "EXT_FOR", str(tmp_path / "torch"))
    return made


def test_torch_without_cuda(calls, monkeypatch, capsys):
    monkeypatch.setattr(torch.version, "cuda", None)
    assert build.build_decoder() is None and not calls
    assert "no CUDA" in capsys.readouterr().err


def test_no_python_headers(calls, monkeypatch, tmp_path):
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert build.build_decoder() is None and not calls


def test_rebuilt_for_another_torch(calls, monkeypatch, tmp_path):
    (tmp_path / "_decoder.so").touch()
    assert build.build_decoder() == build.EXT and len(calls) == 1
    assert not (tmp_path / "_decoder.so").exists()          # the untagged one of an earlier build
    assert build.build_decoder() == build.EXT and len(calls) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.build_decoder() == build.EXT and len(calls) == 2
    assert '-DDRACO_TORCH_VERSION="0.0.1"' in calls[1]


def test_name_has_the_interpreters_tag():
    assert build.EXT.endswith(sysconfig.get_config_var("EXT_SUFFIX")) and "cpython" in build.EXT


def test_extension_of_another_torch_is_refused():
    code = ("import torch\ntorch.__version__ = '0.0.1'\nimport dracomancer_llmengine_b200 as dm\n"
            "try:\n    from dracomancer_llmengine_b200 import decoder\nexcept dm.DracoError as e:\n    print(e)")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, check=True).stdout
    assert "built for torch" in out and "0.0.1" in out
