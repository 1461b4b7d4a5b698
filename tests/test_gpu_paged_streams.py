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


def test_two_graphs_at_once(lib, cuda):
    """Captured steps replayed on two streams at the same time have their own
    workspaces, and a third step runs eagerly beside them."""
    import torch

    dtype = torch.bfloat16
    new, lens = [1, 200, 1, 3, 1], [6000, 900, 11000, 50, 3000]
    c = Cache([4000] + lens, 16, 2, 128, dtype, 62)
    table = c.table[1:].contiguous()
    cu, sl, plen = _cu(new), _i32(lens), _i32([4000])
    qs = [_randn(c.gen, sum(new), 8, 128, dtype=dtype) for _ in range(3)]

    def step(q):
        return (*lib.forward_paged(q, c.K, c.V, table, sl, cu),
                *lib.decode_shared_prefix(q[:5].unsqueeze(2), c.K, c.V, c.table[0], plen, table, sl))

    want = [[x.clone() for x in step(q)] for q in qs]
    torch.cuda.synchronize()
    graphs, got = [], []
    for q in qs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(step(q))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(20):
        for out in got:
            for x in out:
                x.fill_(33.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = step(qs[2])
        torch.cuda.synchronize()
        for have, wanted in zip([*got, eager], want):
            assert all(torch.equal(x, y) for x, y in zip(have, wanted)), turn
    assert lib.device_status() == 0


def test_calls_from_two_threads(lib, cuda):
    """Host threads that call at the same time, each on a stream of its own."""
    import threading

    import torch

    dtype = torch.float16
    new, lens = [1, 60, 1], [5000, 700, 90]
    c = Cache(lens, 32, 2, 64, dtype, 63)
    cu, sl = _cu(new), _i32(lens)
    qs = [_randn(c.gen, sum(new), 8, 64, dtype=dtype) for _ in range(2)]
    want = [lib.forward_paged(q, c.K, c.V, c.table, sl, cu) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                O, L = lib.forward_paged(qs[k], c.K, c.V, c.table, sl, cu)
                stream.synchronize()
                if not (torch.equal(O, want[k][0]) and torch.equal(L, want[k][1])):
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_very_many_sequences(lib, cuda):
    """70000 sequences of up to 20 keys and one token each, through both forms (a
    thread of the division of work has 183 of them), against a padded 64-bit form."""
    import torch

    import paged_ref as ref

    B, Hq, D, ps, dtype = 70000, 2, 64, 16, torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(64)
    pages = 2 * 600
    K, V = (torch.randn(pages, ps, 1, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    table = torch.randint(0, pages, (B, 2), generator=gen, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, 21, (B,), generator=gen, device="cuda", dtype=torch.int32)
    q = torch.randn(B, Hq, D, generator=gen, device="cuda").to(dtype)
    prefix, plen = _i32([7, 3, 500]), _i32([37])
    O, L = lib.forward_paged(q, K, V, table, lens,
                             torch.arange(B + 1, dtype=torch.int32, device="cuda"))
    O2, L2 = lib.decode_shared_prefix(q.unsqueeze(2), K, V, prefix, plen, table, lens)
    at = torch.arange(20, device="cuda")
    rows = table[:, at // ps].long() * ps + at % ps
    live = at < lens[:, None]
    k, v = K.view(-1, D)[rows].double(), V.view(-1, D)[rows].double()
    pre = prefix[torch.arange(37, device="cuda") // ps].long() * ps + torch.arange(37, device="cuda") % ps
    kp, vp = (x.view(-1, D)[pre].double().expand(B, 37, D) for x in (K, V))
    for keys, vals, seen, o, l in (
            (k, v, live, O, L),
            (torch.cat([kp, k], 1), torch.cat([vp, v], 1),
             torch.cat([torch.ones(B, 37, dtype=torch.bool, device="cuda"), live], 1),
             O2.squeeze(2), L2)):
        n = keys.shape[1]
        s = (q.double() @ keys.transpose(1, 2)) * D ** -0.5
        s = s.masked_fill(~seen[:, None], -float("inf"))
        mag = ((q.double().abs() @ keys.abs().transpose(1, 2)) * D ** -0.5).amax(2)
        dead = ~seen.any(1)[:, None].expand(B, Hq)
        want_l = torch.logsumexp(s, 2)
        p = torch.exp(s - want_l.masked_fill(dead, 0.0)[..., None])
        want_o = p @ vals
        # the terms of paged_ref.attend: scores, sums over n keys, P and O rounded
        e_s = D * 2 * ref.EPS32 * mag + 8 * ref.EPS32 * (mag + 1)
        acc = (n + 64) * 2 * ref.EPS32
        u = ref.half_step(dtype)
        bound_o = u * want_o.abs() + (p @ vals.abs()) * (u + 2 * e_s + 2 * acc)[..., None]
        bound_l = e_s + acc + 4 * ref.EPS32 * (want_l.masked_fill(dead, 0.0).abs() + 1)
        ref.check(o, want_o.masked_fill(dead[..., None], 0.0),
                  bound_o.masked_fill(dead[..., None], 0.0), "O")
        ref.check(l, want_l, bound_l, "L")
