"""The library's Makefile, by what `make -n` says it would run: nothing is compiled."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "recommender_amd", "csrc")
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"

pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="no make here")


def would_run(*args, **env):
    out = subprocess.run(["make", "-n", "-C", CSRC, *args], env={**os.environ, **env}, check=True, capture_output=True, text=True).stdout
    return [line for line in out.splitlines() if line.startswith("hipcc")]


def compiles(lines):
    return [line for line in lines if re.search(r"\.hip\b", line)]


@pytest.mark.parametrize("args, env", [((), {}), (("CXXFLAGS=-O1",), {}), ((), {"CXXFLAGS": "-O1"}), (("NO_PACKED_FP32=", "COMPILE=hipcc"), {}),
                                       ((), {"NO_PACKED_FP32": ""})])
@pytest.mark.parametrize("target", ["all", "fenced", "prof", "nowait", "dev", "devprof"])
def test_no_packed_fp32_whatever_the_flags(target, args, env):
    lines = compiles(would_run("-B", target, *args, **env))
    assert lines and all(FLAG in line for line in lines)


def test_other_flags_are_other_objects():
    """A changed Makefile compiles every source again."""
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
    again = {m for line in would_run("-W", "Makefile") if " -c " in line for m in re.findall(r"(\w+\.hip)\b", line)}
    assert sorted(again) == sources
