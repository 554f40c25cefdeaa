"""bf16 attention over 4-bit pages within the bound that tells its outputs from those of small mistakes (a lost key, a
shifted centre: test_q4_precision_bounds.py plants them)."""
import numpy as np
import pytest
import torch

from q4_bounds import attention
from q4_precision_cases import FLAT, ORDINARY, SHAPES, make
from src.kernels import hip_q4_attention as kq

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_scale", [FLAT, ORDINARY])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("name", SHAPES)
def test_bf16_outputs_and_totals(device, name, hd, q_scale):
    c = make(name, hd, q_scale)
    want, added, tol, off = attention(c["qd"], c["kp"], c["vp"], hd, c["table"], c["lens"], c["cur"])
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    fn = kq.paged_attention_prefill_q4_hip if c["q"].shape[2] > 1 else kq.paged_attention_decode_q4_hip
    args = (c["q"].to(device), torch.from_numpy(c["kp"]).to(device), torch.from_numpy(c["vp"]).to(device), i32(c["table"]),
            i32(c["lens"]), i32(c["cur"]))
    totals = torch.zeros(*c["kp"].shape[:2], 16, device=device)
    for weights in (None, totals):
        got = fn(*args, weights=weights).double().cpu().numpy()
        assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    sums = totals.double().cpu().numpy()
    # additions in fp32, of at most 2^7 rows' weights in a lane and of few such sums
    assert (np.abs(sums - added) <= off + 2.0 ** -16 * added).all()
