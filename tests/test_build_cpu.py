"""The build, with the compilers' calls recorded instead of run: the library does
not depend on torch or on the extension beside it."""

import builtins
import os
import subprocess
import warnings

import pytest


@pytest.fixture
def recorded(tmp_path, monkeypatch):
    """The build module with outputs of its own and the commands it ran; `fail` names a source that does not compile."""
    from sunshape_mlx_b200 import build

    done, fail = [], []

    class Popen:
        def __init__(self, cmd, **kw):
            self.rc = int(any(f in " ".join(cmd) for f in fail))
            done.append(cmd)
            if not self.rc:
                open(cmd[cmd.index("-o") + 1], "w").close()
            self.returncode = self.rc

        def wait(self, timeout=None):
            return self.rc

        def poll(self):
            return self.rc

        def communicate(self, *a, **kw):
            return None, None

        def __enter__(self):
            return self

        def __exit__(self, *a):
            return False

    monkeypatch.setattr(subprocess, "Popen", Popen)
    monkeypatch.setattr(build, "_nvcc", lambda: "/cuda/bin/nvcc")
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "FAST", str(tmp_path / "_fast.so"))
    return build, done, fail


def test_library_is_built_without_torch(recorded, monkeypatch):
    import sys

    build, done, _ = recorded
    real = builtins.__import__

    def no_torch(name, *a, **kw):
        if name.split(".")[0] == "torch":
            raise ImportError("no torch")
        return real(name, *a, **kw)

    monkeypatch.setattr(builtins, "__import__", no_torch)
    monkeypatch.delitem(sys.modules, "torch")
    monkeypatch.setattr("importlib.util.find_spec", lambda name, *a: None)
    assert build.build() == build.LIB and os.path.exists(build.LIB) and not os.path.exists(build.FAST)
    assert all(c[0] == "/cuda/bin/nvcc" for c in done)
    n = len(done)
    build.build()  # and is up to date then
    assert len(done) == n


def test_library_is_there_when_the_extension_fails(recorded):
    build, done, fail = recorded
    fail.append("binding.cpp")
    with pytest.raises(subprocess.CalledProcessError):
        build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.FAST)
    fail.clear()
    n = len(done)
    build.build()  # the extension alone
    assert os.path.exists(build.FAST) and all(c[0] == "g++" for c in done[n:])
    n = len(done)
    build.build()
    assert len(done) == n


def test_calls_go_through_their_wrappers_without_the_extension(monkeypatch):
    from sunshape_mlx_b200 import _lib as L, build

    build.build()

    def missing(name, package=None):
        raise ImportError("not built")

    monkeypatch.setattr(L, "_fast", None)
    monkeypatch.setattr(L.importlib, "import_module", missing)
    with pytest.warns(UserWarning, match="native call lane"):
        lane = L.fast()
    for f in ("plan_step", "append", "fetch", "attention", "logprobs"):
        assert getattr(lane, f)(1, 2, 3) is None
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert L.fast() is lane  # said once
