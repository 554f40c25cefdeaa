"""4-bit attention on two streams at once, with totals: the records, scores and row operands of a call on one stream
are not those of a call on the other."""
import numpy as np
import pytest
import torch

from q4_cases import filled_pools, tables
from src.kernels import hip_q4_attention as kq

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads, T, width", [
    ((4, 2), 1, 44),   # totals from scores, in the first launch
    ((4, 2), 1, 300),  # records of several ranges, merged by a second launch, with totals
    ((4, 2), 3, 300),  # records, and totals from scores formed again
    ((2, 2), 40, 44),  # row operands handed to the totals' launch
    ((2, 2), 40, 260),  # those and records
], ids=str)
def test_calls_on_two_streams(device, dtype, heads, T, width):
    rng = np.random.default_rng(T + width)
    lens = [700, 90, 300, 41] if width < 100 else [16 * width - 9, 2000, 300, 41]
    blocks = sum(-(-n // 16) for n in lens) + 2
    kp, vp = filled_pools(rng, blocks, heads[1], 64)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)  # noqa: E731
    table, L, C = i32(tables(rng, lens, blocks, width=width)), i32(lens), i32([T] * 4)
    dk, dv = torch.from_numpy(kp).to(device), torch.from_numpy(vp).to(device)
    fn = kq.paged_attention_decode_q4_hip if T == 1 else kq.paged_attention_prefill_q4_hip
    qs = [torch.randn(4, heads[0], T, 64, generator=torch.Generator().manual_seed(i)).to(dtype).to(device) for i in range(2)]
    new = lambda: torch.zeros(blocks, heads[1], 16, device=device)  # noqa: E731
    wants = []
    for q in qs:
        totals = new()
        wants.append((fn(q, dk, dv, table, L, C, weights=totals), totals))
        torch.cuda.synchronize()
    assert not torch.equal(wants[0][0], wants[1][0]) and not torch.equal(wants[0][1], wants[1][1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    totals = [[new() for _ in range(12)] for _ in streams]
    gots = [[], []]
    torch.cuda.synchronize()
    for n in range(12):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                gots[i].append(fn(qs[i], dk, dv, table, L, C, weights=totals[i][n]))
    torch.cuda.synchronize()
    for i, (out, sums) in enumerate(wants):
        assert all(torch.equal(g, out) for g in gots[i])
        assert all(torch.equal(t, sums) for t in totals[i])  # (each slot gets one addition)
