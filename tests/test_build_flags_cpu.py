"""What the build's own command lines make of the HIP sources (hipcc cross-compiles without a GPU): no library holds packed
fp32 instructions, some forms of which have given wrong results on the hardware now and then."""
import importlib.util
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def build():
    spec = importlib.util.spec_from_file_location("p3d_build", ROOT / "primitive3d_amd" / "_build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("step", ["build_capi", "build_capi_dev", "build_mt", "build_rc"])
def test_no_packed_fp32(build, step, tmp_path, monkeypatch):
    if not Path(build.HIPCC).exists() and not shutil.which(build.HIPCC):
        pytest.skip("hipcc not available")
    monkeypatch.delenv("P3D_CAPI_LIB", raising=False)
    commands = []
    monkeypatch.setattr(build, "PKG", tmp_path)   # (nothing is written beside the package)
    monkeypatch.setattr(build, "_write_stamp", lambda *a: None)
    with monkeypatch.context() as m:
        m.setattr(build.subprocess, "check_call", commands.append)
        getattr(build, step.removesuffix("_dev"))(force=True, **({"dev": True} if step.endswith("_dev") else {}))
    (cmd,) = commands
    out = tmp_path / "device.s"
    cmd = [c for c in cmd[:cmd.index("-o")] if c != "-shared"] + ["-S", "--cuda-device-only", "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    asm = out.read_text()
    assert ".amdhsa_kernel" in asm
    assert not re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", asm)


def test_build_compiles_where_libraries_are_there(built, tmp_path, monkeypatch):
    """__graft_entry__.build() is the check that the sources compile: a library that is already there does not answer it."""
    import __graft_entry__
    mod = __graft_entry__.load_build_module()
    commands = []
    monkeypatch.setattr(mod.subprocess, "check_call", commands.append)
    monkeypatch.setattr(mod, "_write_stamp", lambda *a: None)
    monkeypatch.setattr(mod, "_stale", lambda *a: False)
    monkeypatch.setattr(mod, "PKG", tmp_path)   # (nothing is written beside the package)
    monkeypatch.setattr(__graft_entry__, "load_build_module", lambda: mod)
    __graft_entry__.build()
    outs = sorted(Path(c[c.index("-o") + 1]).relative_to(mod.PKG).as_posix() for c in commands if "-o" in c)
    assert outs == sorted(["libp3dmc.so", "dev/libp3dmc.so", "libp3dmt.so", "libp3drc.so", mod.pybind_path().name])
