"""The compiled layer above the token operators' C entry points takes their types from include/indm_hip.h: a changed signature does not
compile, and a changed header rebuilds it."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

from indm_amd import hip

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


def test_layout_query():
    """few blocks are shared, many are not; bad sizes are refused"""
    f = hip.lib().indm_wattn_layout
    assert f(2, 1, 256, 4, 4, 64, 64, 64, 1, 0) == 1 | 2 | 1 << 4 | 1 << 16      # 8 key blocks; a sink block's 4 tiles of queries: one workgroup
    assert f(2, 8, 4096, 4, 4, 64, 256, 256, 0, 0) == 1 << 4                     # 1024 blocks of queries and of keys: nothing is shared
    assert f(2, 8, 4096, 4, 4, 64, 256, 256, 4, 0) & 0xffff == 4 | 1 << 4        # the sinks apart
    for bad in ((3, 1, 8, 1, 1), (2, 1, 8, 3, 2), (2, 0, 8, 1, 1), (2, 1, 0, 1, 1), (2, 1, 8, 0, 0)):
        assert f(*bad, 32, 1, 1, 0, 0) == -1
    assert f(2, 1, 8, 1, 1, 32, -1, 1, 0, 0) == f(2, 1, 8, 1, 1, 32, 1, 1, -1, 0) == f(2, 1, 8, 1, 1, 0, 1, 1, 0, 0) == -1
