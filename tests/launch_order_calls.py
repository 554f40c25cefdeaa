"""Run by test_launch_order.py in a process of its own: two threads make the named call over one workspace, with
the HIP launch replaced by a stub; prints the launching threads in order. (Nothing here reads the operands.)"""
import ctypes
import json
import sys
import threading
from pathlib import Path

PKG = Path(__file__).resolve().parents[1] / "efficient-inference-system_amd"
CALLS = 4


def main(stub_path: str, name: str) -> None:
    stub = ctypes.CDLL(stub_path, mode=ctypes.RTLD_GLOBAL)
    lib = ctypes.CDLL(str(PKG / "libpaged_hip.so"))
    p, i64, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_float
    ops = p(1 << 30)  # an address that is never read
    room, ws = ctypes.c_size_t(1 << 40), p(1 << 32)

    T = 20

    def q4(T, pages, weights):
        strides = [i64(T * 512), i64(64), i64(512)]
        return lambda: lib.pa_q4_attention(ops, *strides, p(1 << 31), *strides, 0, ops, ops, i64(9), ops, i64(pages), pages, ops,
                                           ops, ops if weights else None, 2, 8, 8, T, 64, f32(0.125), ws, room, None)

    def attention(fn, strides, T, tail):
        s = [i64(x) for x in strides]
        query = [T] if T else []
        order = [] if T else [None]  # (decode's processing order)
        return lambda: fn(ops, *s, p(1 << 31), *s, 0, ops, ops, 0, i64(9), ops, i64(200), 200, ops, ops, *order, 2, 8, *query, 64,
                          16, f32(0.125), 16, *tail)

    call = {
        "split prefill": attention(lib.pa_prefill, (T * 512, 64, 512), T, (ws, room, None)),
        "split decode": attention(lib.pa_decode, (512, 64), 0, (ws, room, None)),
        "split decode in the library's scratch": attention(lib.pa_decode_noalloc, (512, 64), 0, (None,)),
        "q4 chunk with totals": q4(40, 8, True),
        "q4 decode over ranges of keys": q4(1, 4000, False),
        "q4 decode over ranges of keys, with totals": q4(1, 4000, True),
    }[name]
    start = threading.Barrier(2)
    statuses = []

    def work(me):
        stub.stub_thread(me)
        start.wait()
        statuses.extend(call() for _ in range(CALLS))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    out = (ctypes.c_int * 1000)()
    n = stub.stub_order(out, 1000)
    print(json.dumps({"statuses": statuses, "order": list(out[:n])}))


if __name__ == "__main__":
    main(*sys.argv[1:])
