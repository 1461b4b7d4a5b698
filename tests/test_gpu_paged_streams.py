"""The paged-cache operators next to work on other streams, where a call's CTAs
start at different times."""

import pytest

from test_gpu_paged import Cache, _cu, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
def test_ragged_forward_beside_other_streams(lib, cuda, D):
    """Single tokens behind long histories (units of few rows that several CTAs
    share) between chunks (row tiles), on two streams, while dense calls on a
    third hold part of the SMs: every row is written, with the bits of a call that
    has the GPU for itself."""
    import torch

    dtype = torch.bfloat16
    new = [1, 1, 90, 1, 2, 1, 300, 1, 1, 40]
    lens = [9000, 30, 700, 5000, 12000, 1, 2000, 0, 7000, 40]
    c = Cache(lens, 16, 2, D, dtype, 61)
    cu, sl = _cu(new), _i32(lens)
    qs = [_randn(c.gen, sum(new), 8, D, dtype=dtype) for _ in range(2)]
    args = (c.K, c.V, c.table, sl, cu)
    want = []
    for q in qs:
        want.append(lib.forward_paged(q, *args))
        torch.cuda.synchronize()
    dense = [_randn(c.gen, 1, 8, 1500, D, dtype=dtype) for _ in range(3)]
    dense_out = torch.empty_like(dense[0]), torch.empty(1, 8, 1500, device="cuda")
    side = torch.cuda.Stream()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [(torch.empty_like(O), torch.empty_like(L)) for O, L in want]
    torch.cuda.synchronize()
    for turn in range(40):
        for k in range(1 + turn % 3):
            lib.forward(*dense, causal=True, O=dense_out[0], L=dense_out[1], stream=side)
        for q, s, (O, L) in zip(qs, streams, got):
            with torch.cuda.stream(s):
                O.fill_(77.0)
                L.fill_(77.0)
                lib.forward_paged(q, *args, O=O, L=L)
        torch.cuda.synchronize()
        for (O, L), (O2, L2) in zip(got, want):
            assert torch.equal(O, O2) and torch.equal(L, L2), turn
    assert lib.device_status() == 0
