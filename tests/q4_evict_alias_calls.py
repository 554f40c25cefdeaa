"""Run by test_q4_evict_alias.py in a process of its own: evictions whose outputs alias their inputs or do not, with the
HIP launch replaced by a stub (nothing reads the operands); prints the statuses."""
import ctypes
import json
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parents[1] / "efficient-inference-system_amd"
PLACES = {"lens": 1 << 40, "table": 2 << 40, "new_table": 3 << 40, "kept": 4 << 40, "new_lens": 5 << 40}


def main(stub_path: str) -> None:
    ctypes.CDLL(stub_path, mode=ctypes.RTLD_GLOBAL)
    lib = ctypes.CDLL(str(PKG / "libpaged_hip.so"))
    p, i64 = ctypes.c_void_p, ctypes.c_int64
    out = []
    for change in json.load(sys.stdin):
        at = {**PLACES, **change}
        out.append(lib.pa_q4_evict(p(6 << 40), p(7 << 40), p(8 << 40), i64(99), p(at["table"]), i64(10), 10, p(at["lens"]),
                                   p(at["new_table"]), i64(10), 10, 40, 8, p(at["kept"]), p(at["new_lens"]), 3, 2, 64, None))
    print(json.dumps(out))


if __name__ == "__main__":
    main(*sys.argv[1:])
