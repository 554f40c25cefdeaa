"""Calls of two threads on one stream over one workspace: a call's launches follow each other, since a launch of
the other call between them would overwrite what the first hands on to its second. On the CPU, the HIP launch
replaced by a stub that records the launching thread."""
import json
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
LIB = HERE.parent / "efficient-inference-system_amd" / "libpaged_hip.so"
CALLS = 4  # of each thread


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None or not LIB.exists() or not Path("/opt/rocm/include/hip/hip_runtime_api.h").exists():
        pytest.skip("needs g++, the HIP headers and the built library")
    out = tmp_path_factory.mktemp("stub") / "libstub.so"
    subprocess.run([gxx, "-shared", "-fPIC", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    str(HERE / "launch_order_stub.cpp"), "-o", str(out), "-pthread"], check=True, timeout=120)
    return out


@pytest.mark.parametrize("name, launches", [
    ("q4 chunk with totals", 2),
    ("q4 decode over ranges of keys", 2),
    ("q4 decode over ranges of keys, with totals", 2),
    ("split prefill", 2),
    ("split decode", 2),
    ("split decode in the library's scratch", 2),
])
def test_a_calls_launches_are_not_divided(stub, name, launches):
    run = subprocess.run([sys.executable, str(HERE / "launch_order_calls.py"), str(stub), name], capture_output=True,
                         text=True, timeout=120)
    assert run.returncode == 0, run.stderr[-2000:]
    got = json.loads(run.stdout)
    assert got["statuses"] == [0] * (2 * CALLS)
    order = got["order"]
    assert len(order) == 2 * CALLS * launches and order.count(0) == order.count(1)
    for at in range(0, len(order), launches):
        assert len(set(order[at:at + launches])) == 1, order
