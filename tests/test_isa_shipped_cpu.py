"""The kernels as they ship: the scans of test_isa_cpu.py on sources compiled with the Makefile's own flags, and the built library's code
objects -- no packed fp32 arithmetic anywhere, no scratch in the attention kernels but what their register budget's comment names."""
import glob
import os
import re
import shlex
import shutil
import subprocess

import pytest

import test_isa_cpu as isa

LIB = os.path.join(isa.ROOT, "indm_amd", "libindm_hip.so")
LLVM = "/opt/rocm/llvm/bin/"

needs_hipcc = pytest.mark.skipif(shutil.which("hipcc") is None, reason="needs hipcc")
needs_llvm = pytest.mark.skipif(not (os.path.exists(LLVM + "llvm-objdump") and os.path.exists(LIB)), reason="needs llvm-objdump and the built library")


def shipped_flags(source):
    """what the Makefile compiles a source with"""
    obj = source.replace(".hip", ".o")
    out = subprocess.run(["make", "-n", "-W", source, obj], cwd=isa.CSRC, check=True, capture_output=True, text=True).stdout
    (line,) = [x for x in out.splitlines() if " -c " + source in x]
    cmd = shlex.split(line)
    return cmd[1:cmd.index("-c")]


@needs_hipcc
@pytest.mark.parametrize("name", ["test_no_read_of_registers_with_a_load_in_flight", "test_fused_groupnorm_loads_its_arguments_before_its_first_barrier",
                                  "test_f16_kernels_keep_their_loads_in_flight", "test_lds_fold_matches_are_the_audited_kernels"])
def test_scans_with_the_shipped_flags(name, tmp_path, monkeypatch):
    run, seen = subprocess.run, []

    def as_shipped(cmd, **kw):
        if cmd[0] != "hipcc":
            return run(cmd, **kw)
        at = cmd.index("--cuda-device-only")
        flags = shipped_flags(os.path.basename(cmd[at + 2]))
        assert set(cmd[1:at]) <= set(flags) and "-packed-fp32-ops" in flags     # the scans' flags, and what was added to the build since
        seen.append(cmd[at + 2])
        return run([cmd[0]] + flags + cmd[at:], **kw)

    monkeypatch.setattr(isa.subprocess, "run", as_shipped)
    getattr(isa, name)(tmp_path)
    assert seen


def code_objects(tmp_path):
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([LLVM + "llvm-objdump", "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    files = sorted(glob.glob(str(tmp_path / "lib.so.*gfx950*")))
    assert len(files) == len(glob.glob(os.path.join(isa.CSRC, "*.hip")))
    return files


PACKED = re.compile(r"\bv_pk_(add|mul|fma)_f32\b")


@needs_llvm
def test_no_packed_fp32_in_the_library(tmp_path):
    assert PACKED.search("\tv_pk_fma_f32 v[2:3], v[4:5], v[6:7], v[2:3]") and not PACKED.search("\tv_pk_add_f16 v1, v2, v3")
    for f in code_objects(tmp_path):
        text = subprocess.run([LLVM + "llvm-objdump", "-d", f], check=True, capture_output=True, text=True).stdout
        assert "s_endpgm" in text and not PACKED.search(text), f


@needs_llvm
def test_scratch_of_the_attention_kernels(tmp_path):
    """bytes of scratch a lane, as the compiler recorded them with each kernel"""
    scratch = {}
    for f in code_objects(tmp_path):
        notes = subprocess.run([LLVM + "llvm-readelf", "--notes", f], check=True, capture_output=True, text=True).stdout
        for entry in re.split(r"\n  - ", notes):
            name, size = re.search(r"\.name:\s+(\S*wattn_\S+)", entry), re.search(r"\.private_segment_fixed_size:\s+(\d+)", entry)
            if name and size:
                scratch[name.group(1)] = int(size.group(1))
    assert len(scratch) > 100
    some = {k: v for k, v in scratch.items() if v}
    assert [k for k in some if "wattn_query_kernelItLi64ELi4ELb0ELb0E" not in k] == [] and max(some.values(), default=0) <= 16, some
