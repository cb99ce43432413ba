"""The build without what only the extension needs, and the extension beside another torch than it was built for."""

import os
import subprocess
import sys

import pytest

from redline_tiny_b200 import build as B


@pytest.fixture
def there(tmp_path, monkeypatch):
    """The extension's files under a temporary folder, its compiler replaced by one that writes the output."""
    monkeypatch.setattr(B, "EXT", str(tmp_path / "_rl_torch.so"))
    monkeypatch.setattr(B, "EXT_FOR", B.EXT + ".txt")
    monkeypatch.setattr(B, "OUT", str(tmp_path / "libredline_b200.so"))
    ran = []

    def run(cmd, verbose):
        ran.append(cmd[0])
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
    monkeypatch.setattr(B, "_run", run)
    return ran


@pytest.mark.parametrize("missing", ["torch", "compiler", "Python.h"])
def test_the_library_needs_nvcc_alone(there, monkeypatch, tmp_path, capsys, missing):
    with open(B.EXT, "w") as f:
        f.write("older")
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    elif missing == "compiler":
        monkeypatch.setenv("CXX", str(tmp_path / "no-compiler"))
    else:
        monkeypatch.setattr(B.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert B.build(force=True) == B.OUT
    assert len(there) == 1 and os.path.exists(B.OUT)
    assert not os.path.exists(B.EXT)                              # one that would not follow the library's interface
    assert "left out" in capsys.readouterr().err
    with pytest.raises(RuntimeError, match="extension"):
        B.build(need_extension=True)


def test_an_extension_for_another_torch_is_built_again(there, monkeypatch):
    torch = pytest.importorskip("torch")
    assert B.build_extension() == B.EXT and len(there) == 1
    assert B.build_extension() == B.EXT and len(there) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert B.build_extension() == B.EXT and len(there) == 2
    os.remove(B.EXT_FOR)
    assert B.build_extension() == B.EXT and len(there) == 3


def test_an_extension_for_another_torch_does_not_load():
    pytest.importorskip("torch")
    B.build()
    code = ("import torch.version; torch.version.__version__ = '0.0.1'\n"
            "from redline_tiny_b200 import ops; assert ops._fast is None\n"
            "import redline_tiny_b200._rl_torch")
    r = subprocess.run([sys.executable, "-c", code], cwd=B.ROOT, capture_output=True, text=True)
    assert r.returncode != 0 and "ImportError" in r.stderr and "built for torch" in r.stderr, r.stderr
