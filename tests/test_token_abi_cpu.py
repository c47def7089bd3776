"""The compiled layer above the token operators' C entry points takes their types from include/indm_hip.h: a changed signature does not
compile, and a changed header rebuilds it."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "indm_amd", "csrc")
HEADER = os.path.join("..", "..", "include", "indm_hip.h")

needs_make = pytest.mark.skipif(shutil.which("make") is None or shutil.which("g++") is None, reason="needs make and g++")


def command():
    """what make runs for the module once the header is newer than it"""
    out = subprocess.run(["make", "-n", "-W", HEADER, "../_token.so"], cwd=CSRC, check=True, capture_output=True, text=True).stdout
    lines = [x for x in out.splitlines() if "token_bind.cpp" in x]
    assert len(lines) == 1, out
    return shlex.split(lines[0])


@needs_make
def test_the_header_rebuilds_the_module():
    assert "token_bind.cpp" in command()


@needs_make
@pytest.mark.parametrize("change", [None, "layernorm_bwd_bf16", "wattn_fwd_f32"])
def test_a_changed_signature_does_not_compile(tmp_path, change):
    text = open(os.path.join(ROOT, "include", "indm_hip.h")).read()
    if change is not None:
        text, n = re.subn(r"(int indm_%s\()" % change, r"\1int one_more, ", text)
        assert n == 1
    (tmp_path / "indm_hip.h").write_text(text)
    cmd = command()
    at = cmd.index("-o")
    cmd = [cmd[0], "-I" + str(tmp_path), "-fsyntax-only"] + cmd[1:at] + cmd[at + 2:]
    run = subprocess.run(cmd, cwd=CSRC, capture_output=True, text=True, timeout=300)
    assert (run.returncode == 0) == (change is None), run.stderr[-2000:]
    assert change is None or "error" in run.stderr
