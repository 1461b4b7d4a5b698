"""The paged-cache operators next to work on other streams, where a call's CTAs
start at different times and inputs may arrive late."""

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


@pytest.mark.parametrize("captured", [False, True])
def test_appended_rows_from_another_stream(lib, cuda, captured):
    """Appends whose inputs another stream writes late: both caches end with the
    keys and values of the last step at every place, and the attention behind each
    append sees them."""
    import torch

    B, Hq, Hkv, D, ps = 6, 8, 2, 64, 16
    c = Cache([400] * B, ps, Hkv, D, torch.bfloat16, 43)
    start = c.K.clone(), c.V.clone()
    rounds = 8
    srcs = [(_randn(c.gen, B, Hq + 2 * Hkv, D, dtype=torch.bfloat16), _i32([40 * (i + 1)] * B))
            for i in range(rounds)]
    # the caches behind all appends, written by indexing
    K_want, V_want = (x.clone().view(-1, Hkv, D) for x in start)
    for qkv, lens in srcs:
        at = lens.long() - 1
        rows = c.table[torch.arange(B, device="cuda"), at // ps].long() * ps + at % ps
        K_want[rows], V_want[rows] = qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    qkv, lens, cu = torch.zeros_like(srcs[0][0]), _i32([1] * B), _cu([1] * B)
    burn = torch.zeros(1 << 25, device="cuda")
    side = torch.cuda.Stream()

    def step(src):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            burn.add_(1.0)
            qkv.copy_(src[0])
            lens.copy_(src[1])
        main.wait_stream(side)
        lib.kv_append_paged(qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], c.K, c.V, c.table, lens)
        return lib.forward_paged(qkv[:, :Hq].contiguous(), c.K, c.V, c.table, lens, cu)

    want = []
    for src in srcs:
        want.append(step(src))
        torch.cuda.synchronize()
    c.K.copy_(start[0])
    c.V.copy_(start[1])
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [step(src) for src in srcs]
        graph.replay()
    else:
        got = [step(src) for src in srcs]
    torch.cuda.synchronize()
    for (O, L), (O2, L2) in zip(got, want):
        assert torch.equal(O, O2) and torch.equal(L, L2)
    for have, wanted in ((c.K, K_want), (c.V, V_want)):
        assert torch.equal(have.view(torch.int16).view(-1), wanted.view(torch.int16).reshape(-1))
