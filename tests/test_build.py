"""What the build compiles, with the compilers replaced by a recorder."""
import importlib.util
import os

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxcpm-inference_b200")


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("vxb_build_under_test", os.path.join(PKG, "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    monkeypatch.setattr(m, "BUILD", str(tmp_path / "build"))
    monkeypatch.setattr(m, "LIB", str(tmp_path / "lib" / "libvxb.so"))
    monkeypatch.setattr(m, "NATIVE", str(tmp_path / "lib" / "_vxb_native.so"))
    m.ran = []

    def run(cmd, verbose):
        m.ran.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            return ""

    monkeypatch.setattr(m, "_run", run)
    return m


def outputs(m):
    done = sorted(os.path.basename(c[c.index("-o") + 1]) for c in m.ran)
    m.ran.clear()
    return done


def test_library_is_built_without_torch(build, monkeypatch):
    monkeypatch.setattr(build, "_torch", lambda: None)
    assert build.build() == build.LIB
    assert not any("torch" in a or "native" in a for c in build.ran for a in c)
    assert "libvxb.so" in outputs(build)
    build.build()
    assert outputs(build) == []


def test_without_torch_there_is_no_module(build, monkeypatch):
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    assert build._torch() is None


def test_module_is_built_again_for_another_torch(build, monkeypatch):
    if build._torch() is None:
        pytest.skip("needs torch and Python's headers")
    build.build()
    assert {"libvxb.so", "native.cpp.o", "_vxb_native.so"} <= set(outputs(build))
    build.build()
    assert outputs(build) == []
    made_for = build._made_for
    monkeypatch.setattr(build, "_made_for", lambda torch: made_for(torch) + "another")
    build.build()
    assert outputs(build) == ["_vxb_native.so", "native.cpp.o"]
    build.build()
    assert outputs(build) == []
