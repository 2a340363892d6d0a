"""When the library and its torch binding count as built from what stands there now."""

import os
import shutil
import types

import pytest

torch = pytest.importorskip("torch")

from verdict_b200 import build, ops  # noqa: E402


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """The build's files, copied, with stamps as a build leaves them."""
    def copy(path):
        to = tmp_path / os.path.basename(path)
        shutil.copy2(path, to)
        return str(to)

    for name in ("TORCH_SOURCE", "TORCH_LIB", "LIB"):
        monkeypatch.setattr(build, name, copy(getattr(build, name)))
    monkeypatch.setattr(build, "HEADERS", [copy(p) for p in build.HEADERS])
    monkeypatch.setattr(build, "TORCH_STAMP", str(tmp_path / "torch.stamp"))
    monkeypatch.setattr(build, "LIB_STAMP", str(tmp_path / "lib.stamp"))
    build._write(build.TORCH_STAMP, build._torch_digest())
    build._write(build.LIB_STAMP, build._digest(build.HEADERS))
    monkeypatch.setattr(build, "DEPS", [])
    return tmp_path


def test_a_binding_is_told_by_what_it_was_built_from(tree, monkeypatch):
    assert build.torch_up_to_date()
    for p in (build.TORCH_SOURCE, *build.HEADERS):  # a copy with new times is the same file
        os.utime(p, (2e9, 2e9))
    assert build.torch_up_to_date()
    for p in (build.TORCH_SOURCE, *build.HEADERS):
        text = open(p).read()
        with open(p, "a") as f:
            f.write("/* changed */\n")
        os.utime(p, (1, 1))  # however old it looks
        assert not build.torch_up_to_date(), p
        with open(p, "w") as f:
            f.write(text)
        assert build.torch_up_to_date()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", torch.__version__ + ".other")
        assert not build.torch_up_to_date()
    os.remove(build.TORCH_STAMP)
    assert not build.torch_up_to_date()
    build._write(build.TORCH_STAMP, build._torch_digest())
    os.remove(build.TORCH_LIB)
    assert not build.torch_up_to_date()


def test_a_stale_binding_that_cannot_be_rebuilt_is_not_used(tree, monkeypatch):
    def broken(*a, **k):
        raise RuntimeError("no compiler")

    monkeypatch.setattr(build, "build_torch_ops", broken)
    assert isinstance(ops._load(), types.ModuleType)  # as it stands
    with open(build.HEADERS[1], "a") as f:
        f.write("/* changed */\n")
    monkeypatch.setattr(build, "DEPS", [build.HEADERS[1]])
    os.utime(build.HEADERS[1], (4e9, 4e9))
    with pytest.raises(RuntimeError, match="other headers"):
        ops._load()
    monkeypatch.setattr(build, "DEPS", [])  # the library is rebuilt, the binding is not
    with pytest.raises(RuntimeError, match="no compiler"):
        ops._load()
