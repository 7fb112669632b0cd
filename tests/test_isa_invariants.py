"""Properties of the COMPILED kernels that their speed leans on and that the source cannot promise (hipcc cross-compiles
without a GPU, so this runs in the CPU suite):

  * the cursor atomic of k_fused is ONE returning vector atomic per wave-plane, and its result is awaited by a COUNTED
    wait that leaves the NU plane loads issued behind it in flight (a wait for everything would pay the memory latency and
    the arithmetic of every plane one after the other);
  * beside it and the spill area's cursor no other atomic lives in that kernel;
  * no kernel writes memory through the scalar unit: what it does there is load;
  * no k_fused / k_faces / k_face_count_walk variant uses scratch memory.
"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def device_asm(tmp_path_factory):
    if not Path(HIPCC).exists() and not shutil.which("hipcc"):
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("isa") / "p3d_mc.s"
    import importlib.util
    spec = importlib.util.spec_from_file_location("p3d_build", ROOT / "primitive3d_amd" / "_build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    cmd = [HIPCC if Path(HIPCC).exists() else "hipcc", *build.HIP_FLAGS, *build.CAPI_EXTRA_FLAGS, "-S",
           "--cuda-device-only", str(ROOT / "primitive3d_amd" / "csrc" / "p3d_mc.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    return out.read_text()


def _kernels(asm, name):
    """{mangled name: body} of the kernels whose mangled name contains `name`."""
    out = {}
    for m in re.finditer(r"^(_Z\w*%s\w*):\s*;.*?$" % name, asm, re.M):
        start = m.end()
        end = asm.index(".amdhsa_kernel", start)
        out[m.group(1)] = asm[start:end]
    return out


def _instructions(body):
    """Instruction lines of a kernel's text, without comments, labels and directives."""
    lines = (ln.split(";")[0].strip() for ln in body.split("\n"))
    return [ln for ln in lines if ln and not ln.endswith(":") and not ln.startswith(".")]


def _vregs(text):
    """Vector registers a line of assembly mentions: v7 -> {7}, v[16:17] -> {16, 17}."""
    regs = set()
    for a, b in re.findall(r"\bv\[(\d+):(\d+)\]", text):
        regs.update(range(int(a), int(b) + 1))
    regs.update(int(r) for r in re.findall(r"\bv(\d+)\b", text))
    return regs


def test_one_vector_atomic_per_wave_plane(device_asm):
    kernels = _kernels(device_asm, "k_fused")
    assert len(kernels) == 8   # 4 tile geometries x 2 sample types
    for name, body in kernels.items():
        atomics = [ins for ins in _instructions(body) if "atomic" in ins.split()[0]]
        # one cursor atomic per half of the unrolled plane loop, and behind each the spill area's (region-layout mode, the rare
        # wave-plane that does not fit): word 8 of a cursor line
        assert len(atomics) == 4, (name, atomics)
        assert all(re.fullmatch(r"global_atomic_add v\d+, v\d+, v\d+, s\[\d+:\d+\]( offset:64)? sc0", ins) for ins in atomics), (name, atomics)
        assert sum("offset:64" in ins for ins in atomics) == 2, (name, atomics)


def test_cursor_result_is_awaited_by_a_count(device_asm):
    """Between a cursor atomic and the first reader of its result stand exactly the NU row loads of the prefetched plane and
    a wait that leaves those NU in flight; nothing in between reads, copies or overwrites the register, and no wait in
    between is stricter."""
    for name, body in _kernels(device_asm, "k_fused").items():
        nc, ry = map(int, re.search(r"k_fusedI\w*?Li(\d+)ELi(\d+)E", name).groups())
        nu = (ry + 1) * nc
        ins = _instructions(body)
        cursors = [i for i, ln in enumerate(ins) if ln.startswith("global_atomic_add") and "offset:64" not in ln]
        assert len(cursors) == 2, name
        for i in cursors:
            dest = int(re.match(r"global_atomic_add v(\d+),", ins[i]).group(1))
            use = next(j for j in range(i + 1, len(ins)) if dest in _vregs(ins[j]))
            assert re.fullmatch(r"v_readfirstlane_b32 s\d+, v%d" % dest, ins[use]), (name, ins[i], ins[use])
            between = ins[i + 1:use]
            loads = sum(ln.startswith(("buffer_load", "global_load", "flat_load")) for ln in between)
            others = [ln for ln in between if re.match(r"(buffer|global|flat|scratch)_(store|atomic)", ln)]
            assert loads == nu and not others, (name, loads, others)
            waits = [int(m.group(1)) for ln in between for m in [re.search(r"\bvmcnt\((\d+)\)", ln)] if m]
            assert waits and min(waits) == waits[-1] == nu, (name, waits)


def test_scalar_unit_only_loads(device_asm):
    for ins in _instructions(device_asm):
        op = ins.split()[0]
        assert not (op.startswith("s_") and ("atomic" in op or "store" in op)), ins


def test_no_scratch_in_the_benchmarked_variants(device_asm):
    # kernel descriptors: .amdhsa_kernel <name> ... .amdhsa_private_segment_fixed_size N
    seen = 0
    for m in re.finditer(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", device_asm, re.S):
        name, desc = m.group(1), m.group(2)
        if "k_fused" not in name and "k_faces" not in name and "k_face_count_walk" not in name:
            continue
        size = int(re.search(r"\.amdhsa_private_segment_fixed_size (\d+)", desc).group(1))
        assert size == 0, (name, size)
        seen += 1
    assert seen >= 12
