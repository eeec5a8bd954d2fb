"""The build of the calls over torch tensors: left out where torch has no CUDA, a warning where it fails, made again for
another torch. No compiler runs: the torch, the module and the compiler of these tests are files in a temporary folder."""
import importlib.util
import os
import stat
import sys
import types

import pytest

BUILD = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mimizuku_b200", "build.py")


@pytest.fixture
def place(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("mmz_build_under_test", BUILD)
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    torch = tmp_path / "torch"
    (torch / "lib").mkdir(parents=True)
    (torch / "version.py").write_text("__version__ = '1'")
    (tmp_path / "serving.cpp").write_text("")
    os.utime(tmp_path / "serving.cpp", (1000, 1000))
    log = tmp_path / "log"
    cxx = tmp_path / "cxx"
    cxx.write_text(f"""#!{sys.executable}
import sys
open({str(log)!r}, "a").write("called\\n")
open(sys.argv[sys.argv.index("-o") + 1], "w").write("module")
""")
    cxx.chmod(cxx.stat().st_mode | stat.S_IXUSR)
    for name, value in (("SERVING", tmp_path / "_serving.so"), ("SERVING_SRC", tmp_path / "serving.cpp"), ("BUILD", tmp_path)):
        monkeypatch.setattr(b, name, str(value))
    monkeypatch.setenv("CXX", str(cxx))
    monkeypatch.setattr(b.importlib.util, "find_spec",
                        lambda name: types.SimpleNamespace(submodule_search_locations=[str(torch)]))
    calls = lambda: len(log.read_text().split()) if log.exists() else 0  # noqa: E731
    return types.SimpleNamespace(b=b, torch=torch, so=tmp_path / "_serving.so", calls=calls, go=lambda force=False: b._build_serving(
        force, 1000, False))


def test_a_torch_without_cuda_is_left_alone(place, monkeypatch):
    place.go()
    assert place.calls() == 0 and not place.so.exists()
    monkeypatch.setattr(place.b.importlib.util, "find_spec", lambda name: None)
    place.go(force=True)
    assert place.calls() == 0 and not place.so.exists()


def test_built_once_and_again_for_another_torch(place):
    (place.torch / "lib" / "libc10_cuda.so").write_text("")
    place.go()
    assert place.calls() == 1 and place.so.read_text() == "module"
    place.go()
    assert place.calls() == 1
    (place.torch / "version.py").write_text("__version__ = '2'")
    place.go()
    assert place.calls() == 2
    place.go()
    assert place.calls() == 2
    os.remove(place.so)
    place.go()
    place.go(force=True)
    assert place.calls() == 4


def test_a_failure_is_a_warning_and_leaves_no_old_module(place, monkeypatch, capfd):
    (place.torch / "lib" / "libc10_cuda.so").write_text("")
    place.go()
    (place.torch / "version.py").write_text("__version__ = '2'")
    monkeypatch.setenv("CXX", "false")
    place.go()
    assert not place.so.exists() and "_serving.so" in capfd.readouterr().err
    place.go()  # tried again
    assert "_serving.so" in capfd.readouterr().err


def test_a_module_that_does_not_load_says_how_to_build_it(tmp_path, monkeypatch):
    import mimizuku_b200
    (tmp_path / "_serving.so").write_text("no library")
    monkeypatch.setattr(mimizuku_b200, "__path__", [str(tmp_path)])
    for name in ("mimizuku_b200._serving", "mimizuku_b200.serving"):
        monkeypatch.delitem(sys.modules, name, raising=False)
    spec = importlib.util.spec_from_file_location("mimizuku_b200.serving", os.path.join(os.path.dirname(BUILD), "serving.py"))
    with pytest.raises(ImportError, match="build.py"):
        spec.loader.exec_module(importlib.util.module_from_spec(spec))
