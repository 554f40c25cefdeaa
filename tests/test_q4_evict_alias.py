"""Evictions whose outputs lie over what their workgroups still read are refused. On the CPU, the HIP launch replaced by
a stub."""
import json
import subprocess
import sys
from pathlib import Path

import launch_stub
from q4_evict_alias_calls import PLACES

HERE = Path(__file__).resolve().parent


def test_outputs_over_inputs_are_refused(tmp_path):
    lens, table, new_table, kept = (PLACES[k] for k in ("lens", "table", "new_table", "kept"))
    good = [{}, {"new_lens": lens + 12}, {"new_lens": lens - 12}, {"kept": table + 4 * 30}]
    bad = [{"new_lens": lens}, {"new_lens": lens + 8}, {"new_lens": lens - 8},  # 3 lengths in, 3 out
           {"new_table": table}, {"new_lens": table + 4}, {"kept": lens}, {"kept": table + 4 * 29}, {"kept": new_table},
           {"new_lens": kept}]
    stub = launch_stub.build(tmp_path)
    run = subprocess.run([sys.executable, str(HERE / "q4_evict_alias_calls.py"), str(stub)], input=json.dumps(good + bad),
                         capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr[-2000:]
    assert json.loads(run.stdout) == [0] * len(good) + [1] * len(bad)
