"""The binding module is an extra: without it the same calls go through ctypes, so its build never stops the library's."""
import os
import sysconfig

import pytest
import torch

from zeroplatform_b200 import build


@pytest.fixture
def place(tmp_path, monkeypatch):
    """A package folder of its own for the module, with an untagged one that an earlier build left."""
    monkeypatch.setattr(build, "PKG", str(tmp_path))
    monkeypatch.setattr(build, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(build, "DISPATCH", str(tmp_path / os.path.basename(build.DISPATCH)))
    (tmp_path / "_dispatch.so").write_bytes(b"old")
    return tmp_path


def test_the_module_is_named_for_its_interpreter(place):
    assert build.build_dispatch() == build.DISPATCH
    assert build.DISPATCH.endswith("_dispatch" + sysconfig.get_config_var("EXT_SUFFIX"))
    assert sorted(p.name for p in place.iterdir()) == sorted(["_build", os.path.basename(build.DISPATCH)])


@pytest.mark.parametrize("fault", ["compiler fails", "no compiler"])
def test_a_failed_compile_leaves_no_module_and_goes_on(place, monkeypatch, capfd, fault):
    build.build_dispatch()
    os.utime(build.DISPATCH, (0, 0))  # older than its source
    if fault == "no compiler":
        monkeypatch.setenv("PATH", str(place))
    else:
        monkeypatch.setattr(build, "ROOT", str(place / "nowhere"))
        monkeypatch.setattr(build, "CSRC", str(place))
        (place / "dispatch.c").write_text("#error no exchange table\n")
        (place / "nowhere" / "include").mkdir(parents=True)
        (place / "nowhere" / "include" / "zero_tensor_cuda.h").write_text("")
    assert build.build_dispatch() is None
    assert not list(place.glob("_dispatch*.so*"))
    err = capfd.readouterr().err
    assert "ctypes" in err and ("gcc" in err if fault == "no compiler" else "no exchange table" in err)


def test_another_pytorch_builds_it_again(place, monkeypatch):
    runs = []
    real = build.subprocess.run
    monkeypatch.setattr(build.subprocess, "run", lambda *a, **k: runs.append(a) or real(*a, **k))
    for version, count in ((torch.__version__, 1), (torch.__version__, 1), ("0.0", 2), ("0.0", 2)):
        monkeypatch.setattr(torch, "__version__", version)
        assert build.build_dispatch() == build.DISPATCH
        assert len(runs) == count
