"""Calls of two threads on one stream over one workspace: a call's launches follow each other, since a launch of
the other call between them would overwrite what the first hands on to its second. On the CPU, the HIP launch
replaced by a stub that records the launching thread."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

import launch_stub

HERE = Path(__file__).resolve().parent
CALLS = 4  # of each thread


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    return launch_stub.build(tmp_path_factory.mktemp("stub"))


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
