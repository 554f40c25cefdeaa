"""Which layouts of q and out 4-bit attention refuses: every one whose rows share a byte, and none of the same
strides whose rows do not. On the CPU, the HIP launch replaced by a stub."""
import itertools
import json
import random
import subprocess
import sys
from pathlib import Path

import pytest

import launch_stub

HERE = Path(__file__).resolve().parent
HD = 64


@pytest.fixture(scope="module")
def statuses(tmp_path_factory):
    stub = launch_stub.build(tmp_path_factory.mktemp("stub"))

    def run(cases):
        done = subprocess.run([sys.executable, str(HERE / "q4_overlap_calls.py"), str(stub)], input=json.dumps(cases),
                              capture_output=True, text=True, timeout=120)
        assert done.returncode == 0, done.stderr[-2000:]
        return json.loads(done.stdout)

    return run


def _spans(case, strides, start):
    elem = 2 if case["dtype"] else 4
    for at in itertools.product(*map(range, case["sizes"])):
        first = start + elem * sum(i * s for i, s in zip(at, strides))
        yield first, first + elem * HD


def _meet(case):
    """Whether a byte is in a row of q and in one of out, row by row."""
    a, b = sorted(_spans(case, case["q"], 0)), sorted(_spans(case, case["out"], case["offset"]))
    return any(x0 < y1 and y0 < x1 for x0, x1 in a for y0, y1 in b)


def _cases():
    rng = random.Random(0)
    for dtype in (0, 1):
        elem = 2 if dtype else 4
        for _ in range(300):
            B, H, T = (rng.choice((1, 2, 3)) for _ in range(3))
            row = HD * rng.choice((1, 1, 2, 3)) + rng.choice((0, 0, 3))
            inner, outer = (H, T) if rng.random() < 0.5 else (T, H)
            s_in = row
            s_out = s_in * inner * rng.choice((1, 1, 2, 3))
            s_b = s_out * outer * rng.choice((1, 1, 2))
            strides = [s_b, s_in, s_out] if (inner, outer) == (H, T) else [s_b, s_out, s_in]
            other = list(strides)
            if rng.random() < 0.25:
                other = [s + HD * rng.choice((0, 1)) for s in strides]
            span = elem * (s_b * B + row)
            offset = rng.choice((0, elem * HD, elem * row, elem * s_out, elem * s_b, span, rng.randrange(-span, span)))
            offset = rng.choice((1, -1)) * offset // elem * elem
            yield dict(sizes=[B, H, T], q=strides, out=other, offset=offset, dtype=dtype)


def test_rows_that_share_a_byte_are_refused(statuses):
    cases = list(_cases())
    refused = accepted = 0
    for case, (status, message) in zip(cases, statuses(cases)):
        if _meet(case):
            assert status == 1 and "must not be q" in message, case
            refused += 1
        elif case["q"] == case["out"]:
            assert status == 0, (case, message)
            accepted += 1
        else:  # other strides: refused where the extents meet
            assert status == 0 or "must not be q" in message, case
    assert refused > 50 and accepted > 50


def test_layouts_that_programs_have(statuses):
    B, H, T = 3, 4, 5
    fused = [T * 3 * H * HD, HD, 3 * H * HD]  # [B, T, 3, H, HD]
    interleaved = [T * H * 2 * HD, 2 * HD, H * 2 * HD]  # [B, T, H, 2, HD]
    plain = [T * H * HD, HD, H * HD]
    of = lambda q, out, offset: dict(sizes=[B, H, T], q=q, out=out, offset=offset, dtype=0)  # noqa: E731
    good = [of(fused, fused, 4 * H * HD), of(interleaved, interleaved, 4 * HD), of(plain, plain, 4 * B * T * H * HD),
            of(plain, fused, 4 * B * T * H * HD), of(plain, plain, -4 * B * T * H * HD)]
    bad = [of(plain, plain, 0), of(plain, plain, 4), of(plain, plain, 4 * HD), of(plain, plain, -4 * T * H * HD),
           of(interleaved, interleaved, 4 * HD - 4), of(plain, plain, 4 * B * T * H * HD - 4)]
    got = statuses(good + bad)
    assert [s for s, _ in got] == [0] * len(good) + [1] * len(bad)
    huge = dict(sizes=[60000, 32, 1], q=[32 * HD, HD, 32 * HD], out=[32 * HD, HD, 32 * HD], offset=4 * HD * 32 * 59999, dtype=0)
    assert statuses([huge, dict(huge, offset=4 * HD * 32 * 60000)])[0][0] == 1
