"""The builds of the library and of the Python module beside it, and what is imported without torch."""
import os
import subprocess
import sys
import warnings

import pytest

from kore_b200 import _build


class Runs:
    """stands for subprocess.run: notes the programs, writes the outputs, fails where told to"""

    def __init__(self, failing=()):
        self.programs, self.failing = [], failing

    def __call__(self, cmd, **kw):
        name = os.path.basename(cmd[0])
        self.programs.append(name)
        rc = int(name in self.failing)
        if not rc:
            open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, rc, "", "no")


@pytest.fixture
def sandbox(monkeypatch, tmp_path):
    """builds into an empty folder"""
    monkeypatch.setattr(_build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(_build, "LIB_PATH", str(tmp_path / "lib.so"))
    return tmp_path


@pytest.mark.parametrize("why", ["no compiler", "no torch"])
def test_the_library_is_built_without_the_module(monkeypatch, sandbox, why):
    """nvcc is all that the library needs"""
    runs = Runs(failing=("g++", "c++"))
    monkeypatch.setattr(_build.subprocess, "run", runs)
    if why == "no torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    with pytest.warns(RuntimeWarning, match="serving"):
        assert _build.build() == _build.LIB_PATH
    assert runs.programs[0] == "nvcc" and os.path.exists(_build.LIB_PATH)


def test_a_library_that_does_not_compile_is_an_error(monkeypatch, sandbox):
    monkeypatch.setattr(_build.subprocess, "run", Runs(failing=("nvcc",)))
    with pytest.raises(RuntimeError, match="nvcc"):
        _build.build()


def test_the_decoder_is_imported_without_torch():
    """its configuration and angle tables need numpy alone"""
    code = ("import sys; sys.modules['torch'] = None\n"
            "from kore_b200 import decoder\n"
            "assert decoder.rope_tables(decoder.DecoderConfig())[0].shape == (640, 50)")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def test_a_module_of_another_torch_is_not_taken_for_current(monkeypatch, sandbox):
    import torch

    runs = Runs()
    monkeypatch.setattr(_build.subprocess, "run", runs)
    first = _build.build_module()
    assert _build.build_module() == first and runs.programs == ["g++"]
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert _build.build_module() != first and runs.programs == ["g++", "g++"]


@pytest.mark.parametrize("broken", [False, True])
def test_calls_without_the_module_go_the_other_way(monkeypatch, tmp_path, broken):
    """one warning, then the Python layer's own checks and errors; asking for the module itself is an error"""
    import torch

    from kore_b200 import KoreError, serving

    path = tmp_path / "m.so"
    if broken:
        path.write_bytes(b"not a library")
    monkeypatch.setattr(_build, "module_path", lambda: str(path))
    monkeypatch.setattr(serving, "_native", None)
    with pytest.warns(RuntimeWarning, match="native module"), pytest.raises(KoreError, match="logits"):
        serving.sample(torch.zeros(2, 5), torch.zeros(2))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(KoreError, match="logits"):
            serving.sample(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(ImportError if broken else RuntimeError):
        serving.native()
