"""The bound of bf16 attention over 4-bit pages tells right outputs from wrong ones: mistakes planted in the oracle, on
the CPU, pass it nowhere."""
import numpy as np
import pytest

from oracle import q4
from q4_bounds import attention
from q4_precision_cases import FLAT, ORDINARY, SHAPES, make

BLOCK = 16


def _oracle(c, **change):
    c = {**c, **change}
    kv = c.get("k", None)
    k = q4.values(c["kp"], c["hd"], True) if kv is None else kv
    v = q4.values(c["vp"], c["hd"], False) if "v" not in c else c["v"]
    return q4.attention(c["qd"], k, v, c["table"], c["lens"], c["cur"])


def _shorter(c):
    """The last key of every request is not seen. (Its rows' visibility with it: one more key than new rows is left.)"""
    out, added = np.zeros(c["qd"].shape), None
    for b, n in enumerate(c["lens"]):
        blk = c["table"][b, (n - 1) // BLOCK]
        vals = q4.values(c["kp"], c["hd"], True)
        vals[blk, :, (n - 1) % BLOCK] = -1e4 * np.sign(c["qd"][b, 0, -1])  # (one row's and head's score falls out)
        got, _ = q4.attention(c["qd"][b:b + 1, :1, -1:], vals[:, :1], q4.values(c["vp"], c["hd"], False)[:, :1],
                              c["table"][b:b + 1], [n], [1])
        out[b, 0, -1] = got[0, 0, 0]
    return out


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("name", SHAPES)
def test_mistakes_exceed_the_bound(name, hd):
    c = make(name, hd, FLAT)
    c["table"] = c["table"][:, :80]
    want, added, tol, off = attention(c["qd"], c["kp"], c["vp"], hd, c["table"], c["lens"], c["cur"])
    ref, ref_added = _oracle(c)
    # the bound's own outputs are the oracle's
    assert np.abs(want - ref).max() < 1e-12 and np.abs(added - ref_added).max() < 1e-12
    B = len(c["lens"])

    # the last row of head 0 without the request's last key
    lost = _shorter(c)
    for b in range(B):
        assert (np.abs(lost[b, 0, -1] - want[b, 0, -1]) > tol[b, 0, -1]).any()
    # a page in the middle, lost
    table = c["table"].copy()
    table[:, 1] = -1
    got, got_added = _oracle(c, table=table)
    for b in range(B):
        assert (np.abs(got[b] - want[b]) > tol[b]).any()
    # V's centres off by 0.02, in one group
    v = q4.values(c["vp"], hd, False)
    v[..., :64] += 0.02
    got, _ = _oracle(c, v=v)
    assert (np.abs(got - want) > tol)[..., :64].mean() > 0.5
    # V's scales off by a tenth
    v = q4.values(c["vp"], hd, False)
    v += 0.1 * (v - v.mean(-1, keepdims=True))
    got, _ = _oracle(c, v=v)
    assert (np.abs(got - want) > tol).any()
    # a row that sees one key more
    if c["cur"][0] > 1:
        got, _ = _oracle(c, cur=[n - 1 for n in c["cur"]])
        for b in range(B):
            assert (np.abs(got[b] - want[b]) > tol[b]).any()
    # a key's weight counted twice
    assert (2 * added - added > off)[added > 0].all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("name", SHAPES)
def test_wrong_scores_exceed_the_bound(name, hd):
    c = make(name, hd, ORDINARY)
    c["table"] = c["table"][:, :80]
    want, _, tol, _ = attention(c["qd"], c["kp"], c["vp"], hd, c["table"], c["lens"], c["cur"])
    # K's centres of every other token off by a tenth
    k = q4.values(c["kp"], hd, True)
    k[:, :, ::2, :64] += 0.1
    got, _ = _oracle(c, k=k)
    assert (np.abs(got - want) > tol).any()
    # the softmax's scale off by a fiftieth
    got, _ = _oracle(c, qd=c["qd"] * 1.02)
    assert (np.abs(got - want) > tol).any()
    # the neighbour's KV head
    if c["kp"].shape[1] > 1:
        got, _ = _oracle(c, k=q4.values(c["kp"], hd, True)[:, ::-1])
        assert (np.abs(got - want) > tol).mean() > 0.5
