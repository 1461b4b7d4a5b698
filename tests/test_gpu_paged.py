"""Paged-cache serving on the GPU: append with rotation, ragged forward and
shared-prefix decode, against plain 64-bit forms (tests/paged_ref.py, which
derives the bounds).  Cache places that belong to no live token hold NaN, and
table entries behind a sequence's last page name no page, so that a read of
either shows."""

import math

import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": "bfloat16", "f16": "float16"}


def _dtype(name):
    import torch

    return getattr(torch, DT[name])


def _gen(seed):
    import torch

    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype):
    import torch

    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


class Cache:
    """A pool of NaN pages with shuffled pages handed to lists of lengths."""

    def __init__(self, lens, page_size, hkv, D, dtype, seed, fill=True, extra=3):
        import torch

        g = torch.Generator().manual_seed(seed)
        self.gen = _gen(seed)
        need = [(n + page_size - 1) // page_size for n in lens]
        self.num_pages = sum(need) + extra
        order = torch.randperm(self.num_pages, generator=g).to(torch.int32)
        width = max(1, max(need))
        table = torch.full((len(lens), width), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table.cuda()
        self.page_size = page_size
        self.K = torch.full((self.num_pages, page_size, hkv, D), float("nan"), dtype=dtype,
                            device="cuda")
        self.V = self.K.clone()
        self.lens = list(lens)
        if fill:
            for b, n in enumerate(lens):
                self.put(b, _randn(self.gen, n, hkv, D, dtype=dtype),
                         _randn(self.gen, n, hkv, D, dtype=dtype))

    def rows(self, b, n):
        import torch

        return ref.cache_rows(self.table[b], torch.arange(n, device="cuda"), self.page_size)

    def put(self, b, k, v):
        r = self.rows(b, k.shape[0])
        self.K.view(-1, *self.K.shape[2:])[r] = k
        self.V.view(-1, *self.V.shape[2:])[r] = v

    def get(self, b, n=None):
        r = self.rows(b, self.lens[b] if n is None else n)
        return self.K.view(-1, *self.K.shape[2:])[r], self.V.view(-1, *self.V.shape[2:])[r]


def _i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return _i32(out)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 32, 8), (64, 14, 2), (32, 3, 3), (128, 1, 1)])
@pytest.mark.parametrize("page_size", [1, 4, 16, 128])
@pytest.mark.parametrize("rotary,interleaved", [(0, False), (16, False), (None, False),
                                                (16, True), (None, True)])
def test_append_ragged(lib, cuda, dt, D, Hq, Hkv, page_size, rotary, interleaved):
    """Ragged sequences, one without new tokens, slices of one projection's
    output; every other place of the cache stays as it was."""
    import torch

    import cuflash_attn as cf

    dtype = _dtype(dt)
    new = [3, 0, 1, 37, 130]
    old = [5, 40, 0, 16, 1]
    lens = [a + b for a, b in zip(new, old)]
    c = Cache(lens, page_size, Hkv, D, dtype, 1, fill=False)
    T = sum(new)
    qkv = _randn(c.gen, T, (Hq + 2 * Hkv) * D, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
    rotary = D if rotary is None else rotary
    rope = cf.rope_table(max(lens), rotary) if rotary else None
    want_k, want_v = c.K.clone(), c.V.clone()
    pos = torch.cat([torch.arange(o, n, device="cuda") for o, n in zip(old, lens)])
    rows = torch.cat([c.rows(b, lens[b])[old[b]:] for b in range(len(new))])
    out = lib.kv_append_paged(k, v, c.K, c.V, c.table, _i32(lens), _cu(new), Q=q, rope_table=rope,
                              interleaved=interleaved)
    kf, vf = c.K.view(-1, Hkv, D), c.V.view(-1, Hkv, D)
    if rope is None:
        assert torch.equal(out, q)
        assert torch.equal(kf[rows], k)
    else:
        for name, x, y in (("Q", q, out), ("K", k, kf[rows])):
            w, mag = ref.rotate(x, rope, pos, interleaved)
            ref.check(y, w, ref.rotate_bound(w, mag, dtype), name)
            assert torch.equal(y[..., rotary:], x[..., rotary:])
    assert torch.equal(vf[rows], v)
    want_k.view(-1, Hkv, D)[rows] = kf[rows]
    want_v.view(-1, Hkv, D)[rows] = vf[rows]
    assert torch.equal(c.K.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(c.V.view(torch.int16), want_v.view(torch.int16))


def test_append_one_token_each_and_padding(lib, cuda):
    """Without cu_seqlens token b belongs to sequence b; a sequence of length 0
    (a padded batch entry) and one whose page is not in the pool store nothing."""
    import torch

    import cuflash_attn as cf

    lens = [1, 17, 0, 64, 33]
    c = Cache(lens, 16, 2, 64, torch.bfloat16, 2, fill=False)
    c.table[4, 2] = c.num_pages  # the last page of sequence 4
    before = c.K.clone(), c.V.clone()
    k, v = (_randn(c.gen, 5, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    q = _randn(c.gen, 5, 4, 64, dtype=torch.bfloat16)
    rope = cf.rope_table(64, 64)
    out = lib.kv_append_paged(k, v, c.K, c.V, c.table, _i32(lens), Q=q, rope_table=rope)
    pos = torch.tensor([0, 16, 0, 63, 32], device="cuda")
    w, mag = ref.rotate(q, rope, pos, False)
    ref.check(out, w, ref.rotate_bound(w, mag, torch.bfloat16), "Q")
    for b in (0, 1, 3):
        r = c.rows(b, lens[b])[-1]
        assert torch.equal(c.V.view(-1, 2, 64)[r], v[b])
        before[1].view(-1, 2, 64)[r] = v[b]
        w, mag = ref.rotate(k[b:b + 1], rope, pos[b:b + 1], False)
        ref.check(c.K.view(-1, 2, 64)[r][None], w, ref.rotate_bound(w, mag, torch.bfloat16), "K")
        before[0].view(-1, 2, 64)[r] = c.K.view(-1, 2, 64)[r]
    assert torch.equal(c.K.view(torch.int16), before[0].view(torch.int16))
    assert torch.equal(c.V.view(torch.int16), before[1].view(torch.int16))


def test_append_positions_in_place_and_tail(lib, cuda):
    """Explicit positions (behind a shared prefix), out-of-table positions
    clamped, queries rotated in place, tokens behind the last sequence and
    tokens whose index is negative left out."""
    import torch

    import cuflash_attn as cf

    new, lens = [4, 3], [9, 2]  # sequence 1: its first token would sit at index -1
    c = Cache([9, 16], 8, 1, 32, torch.float16, 3, fill=False)
    T = 9  # two tokens behind the last sequence
    k, v = (_randn(c.gen, T, 1, 32, dtype=torch.float16) for _ in range(2))
    q = _randn(c.gen, T, 2, 32, dtype=torch.float16)
    q0 = q.clone()
    rope = cf.rope_table(100, 32)
    positions = _i32([50, 51, 52, 99, 7, 1000, -5, 3, 3])
    out = lib.kv_append_paged(k, v, c.K, c.V, c.table, _i32(lens), _cu(new), Q=q, Q_out=q,
                              rope_table=rope, positions=positions)
    assert out.data_ptr() == q.data_ptr()
    pos = positions.long().clamp(0, 99)
    w, mag = ref.rotate(q0, rope, pos, False)
    ref.check(q[:7], w[:7], ref.rotate_bound(w, mag, torch.float16)[:7], "Q")
    assert torch.equal(q[7:], q0[7:])
    r = torch.cat([c.rows(0, 9)[5:], c.rows(1, 2)])
    kept = torch.tensor([0, 1, 2, 3, 5, 6], device="cuda")
    assert torch.equal(c.V.view(-1, 1, 32)[r], v[kept])
    left = torch.ones(c.K.shape[0] * 8, dtype=torch.bool, device="cuda")
    left[r] = False
    assert bool(torch.isnan(c.K.view(-1, 32)[left]).all())
    # keys and values only
    c.V.fill_(float("nan"))
    assert lib.kv_append_paged(k, v, c.K, c.V, c.table, _i32(lens), _cu(new)) is None
    assert torch.equal(c.K.view(-1, 1, 32)[r], k[kept])
    assert torch.equal(c.V.view(-1, 1, 32)[r], v[kept])


def test_append_many_sequences(lib, cuda):
    """More sequences than one round of the look-up probes, many of them empty."""
    import torch

    g = torch.Generator().manual_seed(4)
    new = (torch.randint(0, 4, (2500,), generator=g) * torch.randint(0, 2, (2500,), generator=g))
    new = new.tolist()
    lens = [n + 2 for n in new]
    c = Cache(lens, 2, 1, 32, torch.bfloat16, 5, fill=False)
    k = _randn(c.gen, sum(new), 1, 32, dtype=torch.bfloat16)
    lib.kv_append_paged(k, k, c.K, c.V, c.table, _i32(lens), _cu(new))
    at = 0
    want = torch.full_like(c.K, float("nan")).view(-1, 1, 32)
    rows, toks = [], []
    table = c.table.cpu()
    for b, n in enumerate(new):
        for i in range(n):
            p = lens[b] - n + i
            rows.append(int(table[b, p // 2]) * 2 + p % 2)
            toks.append(at + i)
        at += n
    want[torch.tensor(rows, device="cuda")] = k[torch.tensor(toks, device="cuda")]
    assert torch.equal(c.K.view(torch.int16).view(-1), want.view(torch.int16).view(-1))
    assert torch.equal(c.V.view(torch.int16).view(-1), want.view(torch.int16).view(-1))


# ----------------------------------------------------------- ragged forward
def _check_forward(lib, new, lens, Hq, Hkv, D, page_size, dt, causal, seed=0, tail=0, ramp=None,
                   scale=None):
    import torch

    dtype = _dtype(dt)
    c = Cache(lens, page_size, Hkv, D, dtype, seed)
    if ramp is not None:
        for b, n in enumerate(lens):
            k, v = c.get(b)
            k = (k.float() * torch.linspace(1.0, ramp, max(n, 1), device="cuda")[:n, None, None])
            c.put(b, k.to(dtype), v)
    T = sum(new) + tail
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q = _randn(c.gen, T, Hq, D, dtype=dtype)
    O = torch.full_like(q, 7.0)
    L = torch.full((T, Hq), 7.0, device="cuda")
    lib.forward_paged(q, c.K, c.V, c.table, _i32(lens), _cu(new), causal=causal, scale=scale, O=O,
                      L=L)
    torch.cuda.synchronize()
    assert lib.device_status() == 0
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        k, v = c.get(b)
        vis = None
        if causal:
            i = torch.arange(n, device="cuda")[:, None]
            vis = torch.arange(m, device="cuda")[None] <= i + (m - n)
        O64, L64, bO, bL = ref.attend(q[at:at + n], k, v, scale, vis, dtype)
        ref.check(O[at:at + n], O64, bO, f"O of sequence {b}")
        ref.check(L[at:at + n], L64, bL, f"L of sequence {b}")
        at += n
    assert bool((O[at:] == 7.0).all()) and bool((L[at:] == 7.0).all())
    return O, L


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (7, 1), (6, 2)])
@pytest.mark.parametrize("page_size", [1, 4, 8, 16, 64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_forward_paged_ragged(lib, cuda, dt, D, Hq, Hkv, page_size, causal):
    """Sequences of no, one and several new tokens, lengths of zero and one and
    around tile and page borders, more new tokens than keys, and rows behind
    the last sequence."""
    _check_forward(lib, [0, 1, 5, 1, 129, 64, 1, 3], [10, 1, 5, 0, 300, 128, 255, 1], Hq, Hkv, D,
                   page_size, dt, causal, tail=3)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_forward_paged_long(lib, cuda, causal, D):
    """A long prompt chunk over a long history: units split over several CTAs."""
    _check_forward(lib, [700, 1, 90], [2900, 4111, 90], 4, 2, D, 16, "bf16", causal, seed=6)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 127, 128, 129, 255, 256, 257, 511])
@pytest.mark.parametrize("group", [1, 4, 5])
def test_forward_paged_one_sequence(lib, cuda, n, group):
    """One sequence, query counts around the row tiles' borders, causal."""
    _check_forward(lib, [n], [n + 77], 2 * group, 2, 64, 16, "bf16", True, seed=7)


def test_forward_paged_wide_groups(lib, cuda):
    """More query heads per key head than a tile has rows."""
    _check_forward(lib, [3, 1], [200, 150], 160, 1, 64, 16, "bf16", True, seed=8)
    _check_forward(lib, [2], [140], 256, 2, 32, 8, "f16", True, seed=8)


def test_forward_paged_growing_scores(lib, cuda):
    """Scores that grow along the cache: the running maximum rises block by
    block and the output is rescaled."""
    for dt in ("bf16", "f16"):
        _check_forward(lib, [40, 200], [1500, 900], 8, 2, 128, 32, dt, True, seed=9, ramp=8.0)


def test_forward_paged_zero_scale(lib, cuda):
    """Scale 0: the mean of the visible values."""
    _check_forward(lib, [5, 70], [300, 70], 4, 2, 64, 16, "bf16", True, seed=10, scale=0.0)


def test_forward_paged_matches_dense_forward(lib, cuda):
    """A prompt without history equals forward_gqa on the same keys."""
    import torch

    N, Hq, Hkv, D = 517, 8, 2, 128
    c = Cache([N], 16, Hkv, D, torch.bfloat16, 11)
    q = _randn(c.gen, N, Hq, D, dtype=torch.bfloat16)
    O, L = lib.forward_paged(q, c.K, c.V, c.table, _i32([N]), _cu([N]))
    k, v = (x.transpose(0, 1)[None].contiguous() for x in c.get(0))
    O2, L2 = lib.forward_gqa(q.transpose(0, 1)[None].contiguous(), k, v, causal=True)
    torch.cuda.synchronize()
    # both round P and O once: two half steps each of values up to max |V|
    assert float((O.float() - O2[0].transpose(0, 1).float()).abs().max()) <= 4 * 2.0 ** -8 * float(
        v.abs().max())
    assert float((L - L2[0].transpose(0, 1)).abs().max()) < 1e-4


@pytest.mark.parametrize("group", [1, 2, 3, 8, 15, 16, 17, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_forward_paged_few_rows(lib, cuda, group, D):
    """One to four new tokens per sequence over short and long histories: the
    forms of few rows, their borders to the row tiles, keys split over CTAs."""
    new = [1, 1, 2, 1, 4, 3, 1, 1, 5]
    lens = [3000, 1, 129, 5, 700, 3, 0, 6500, 260]
    _check_forward(lib, new, lens, 2 * group, 2, D, 16, "bf16", True, seed=31)
    _check_forward(lib, new, lens, group, 1, D, 64, "f16", False, seed=32)


def test_forward_paged_many_sequences(lib, cuda):
    """More sequences than threads of a CTA, the kinds of units mixed."""
    new = [(b % 5 == 0) * (1 + b % 9) for b in range(1300)]
    lens = [(n > 0) * (n + (17 * b) % 41) for b, n in enumerate(new)]
    _check_forward(lib, new, lens, 4, 2, 64, 8, "bf16", True, seed=33, tail=5)


@pytest.mark.parametrize("page_size", [2, 16])
@pytest.mark.parametrize("D", [32, 128])
def test_forward_paged_not_a_number(lib, cuda, page_size, D):
    """A NaN in a key that rows see makes those rows' O and L NaN, and no other
    row's; in a key that causality hides from a row it leaves the row alone.  A
    NaN in a value reaches O only."""
    import torch

    new, lens = [3, 1, 140, 1], [30, 200, 150, 400]
    c = Cache(lens, page_size, 2, D, torch.bfloat16, 34)
    q = _randn(c.gen, sum(new), 4, D, dtype=torch.bfloat16)
    args = (c.table, _i32(lens), _cu(new))
    want, want_l = lib.forward_paged(q, c.K, c.V, *args)
    nan = float("nan")
    K = c.K.clone()
    K.view(-1, 2, D)[c.rows(0, 30)[28], 0, 1] = nan    # hidden from token 0 of sequence 0
    K.view(-1, 2, D)[c.rows(1, 200)[77], 1, 0] = nan
    K.view(-1, 2, D)[c.rows(2, 150)[149], 0, 3] = nan  # seen by the last token alone
    O, L = lib.forward_paged(q, K, c.V, *args)
    hit = torch.zeros((sum(new), 4), dtype=torch.bool, device="cuda")
    hit[1:3, :2] = True
    hit[3, 2:] = True
    hit[143, :2] = True
    assert torch.equal(torch.isnan(L), hit)
    assert torch.equal(torch.isnan(O).all(-1), hit) and torch.equal(torch.isnan(O).any(-1), hit)
    assert torch.equal(O[~hit], want[~hit]) and torch.equal(L[~hit], want_l[~hit])
    V = c.V.clone()
    V.view(-1, 2, D)[c.rows(3, 400)[300], 0, 5] = nan
    O, L = lib.forward_paged(q, c.K, V, *args)
    assert torch.equal(L, want_l) and bool(torch.isnan(O[144, :2, 5]).all())
    O[144, :2, 5] = want[144, :2, 5]
    assert torch.equal(O, want)
    # the same through the prefix decode: prefix 0's keys, own keys of 1 and 3
    qd = q[:2].unsqueeze(2).contiguous()
    own = c.table[[1, 3]].contiguous()
    O, L = lib.decode_shared_prefix(qd, K, c.V, c.table[2], _i32([140]), own, _i32([200, 400]))
    hit = torch.tensor([[False, False, True, True], [False] * 4], device="cuda")
    assert torch.equal(torch.isnan(L), hit) and torch.equal(torch.isnan(O).any(-1)[..., 0], hit)
    O, L = lib.decode_shared_prefix(qd, K, c.V, c.table[2], _i32([150]), own, _i32([200, 400]))
    hit[:, :2] = True
    assert torch.equal(torch.isnan(L), hit) and torch.equal(torch.isnan(O).any(-1)[..., 0], hit)


@pytest.mark.parametrize("page_size", [4, 32])
def test_lengths_and_pages_out_of_range(lib, cuda, page_size):
    """Lengths beyond the table count as the table's, negative ones as zero; a
    page outside the pool gives some page's rows and touches nothing else."""
    import torch

    new, lens = [2, 1, 9, 1], [128, 96, 128, 60]
    c = Cache(lens, page_size, 1, 64, torch.bfloat16, 35)
    q = _randn(c.gen, sum(new), 4, 64, dtype=torch.bfloat16)
    want = lib.forward_paged(q, c.K, c.V, c.table, _i32(lens), _cu(new))
    far = lib.forward_paged(q, c.K, c.V, c.table, _i32([1 << 30, 96, 1 << 20, 60]), _cu(new))
    for x, y in zip(want, far):
        assert torch.equal(x, y)
    O, L = lib.forward_paged(q, c.K, c.V, c.table, _i32([128, -5, 128, 60]), _cu(new))
    assert bool((O[2] == 0).all()) and bool(torch.isneginf(L[2]).all())
    rest = [0, 1] + list(range(3, 13))
    assert torch.equal(O[rest], want[0][rest]) and torch.equal(L[rest], want[1][rest])
    bad = c.table.clone()
    bad[1, 1], bad[3, 0] = -3, c.num_pages + 1000
    O, L = lib.forward_paged(q, c.K, c.V, bad, _i32(lens), _cu(new))
    rest = [0, 1] + list(range(3, 12))
    assert torch.equal(O[rest], want[0][rest]) and torch.equal(L[rest], want[1][rest])
    assert lib.device_status() == 0


def test_sequences_that_share_pages(lib, cuda):
    """The same pages in several rows of the table, and twice in one."""
    import torch

    c = Cache([200], 16, 2, 128, torch.bfloat16, 36)
    row = c.table[0].clone()
    row[5] = row[4]
    table = torch.stack([c.table[0], c.table[0], row])
    q = _randn(c.gen, 3, 8, 128, dtype=torch.bfloat16)
    q[1] = q[0]
    O, L = lib.forward_paged(q, c.K, c.V, table, _i32([200] * 3), _cu([1] * 3))
    assert torch.equal(O[0], O[1]) and torch.equal(L[0], L[1])
    r = ref.cache_rows(row, torch.arange(200, device="cuda"), 16)
    k, v = c.K.view(-1, 2, 128)[r], c.V.view(-1, 2, 128)[r]
    O64, L64, bO, bL = ref.attend(q[2:], k, v, 128 ** -0.5, None, torch.bfloat16)
    ref.check(O[2:], O64, bO, "O")
    ref.check(L[2:], L64, bL, "L")


# ----------------------------------------------------- shared-prefix decode
def _check_prefix(lib, prefix, lens, Hq, Hkv, D, page_size, dt, seed=0, ramp=None):
    import torch

    dtype = _dtype(dt)
    c = Cache([prefix] + list(lens), page_size, Hkv, D, dtype, seed)
    if ramp is not None:
        for b, n in enumerate(c.lens):
            k, v = c.get(b)
            k = k.float() * torch.linspace(1.0, ramp, max(n, 1), device="cuda")[:n, None, None]
            c.put(b, k.to(dtype), v)
    B = len(lens)
    q = _randn(c.gen, B, Hq, 1, D, dtype=dtype)
    table = c.table[1:].contiguous()
    O, L = lib.decode_shared_prefix(q, c.K, c.V, c.table[0], _i32([prefix]), table, _i32(lens))
    torch.cuda.synchronize()
    assert lib.device_status() == 0
    kp, vp = c.get(0)
    for b in range(B):
        k, v = c.get(1 + b)
        O64, L64, bO, bL = ref.attend(q[b].transpose(0, 1), torch.cat([kp, k]),
                                      torch.cat([vp, v]), 1.0 / math.sqrt(D), None, dtype)
        ref.check(O[b].transpose(0, 1), O64, bO, f"O of sequence {b}")
        ref.check(L[b][None], L64, bL, f"L of sequence {b}")
    return O, L


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (7, 1)])
@pytest.mark.parametrize("page_size", [1, 8, 16, 64, 256])
@pytest.mark.parametrize("prefix", [0, 1, 300])
def test_shared_prefix(lib, cuda, dt, D, Hq, Hkv, page_size, prefix):
    _check_prefix(lib, prefix, [0, 1, 130, 16, 257], Hq, Hkv, D, page_size, dt)


@pytest.mark.parametrize("B", [1, 2, 32, 33, 64, 65, 200])
def test_shared_prefix_batches(lib, cuda, B):
    """Batches around the row tiles' borders (group 4: 32 sequences a tile)."""
    _check_prefix(lib, 700, [(37 * b) % 190 for b in range(B)], 8, 2, 64, 16, "bf16", seed=B)


def test_shared_prefix_long(lib, cuda):
    """A prefix and own tokens long enough to be split over many CTAs."""
    _check_prefix(lib, 9001, [2000, 3, 0, 1111], 8, 2, 128, 16, "bf16", seed=12)
    _check_prefix(lib, 4096, [500] * 20, 16, 4, 128, 64, "f16", seed=13, ramp=6.0)


def test_shared_prefix_wide_groups(lib, cuda):
    _check_prefix(lib, 333, [5, 0, 140], 160, 1, 64, 16, "bf16", seed=14)
    _check_prefix(lib, 200, [9, 150], 256, 2, 32, 8, "f16", seed=15)


@pytest.mark.parametrize("group", [1, 8, 16, 17])
def test_shared_prefix_groups(lib, cuda, group):
    _check_prefix(lib, 1500, [900, 0, 3, 129, 5000], 2 * group, 2, 128, 16, "bf16", seed=17)


def test_shared_prefix_no_key_at_all(lib, cuda):
    import torch

    O, L = _check_prefix(lib, 0, [0, 0, 3], 4, 2, 64, 16, "bf16")
    assert bool((O[:2] == 0).all()) and bool(torch.isneginf(L[:2]).all())


def test_shared_prefix_many_short_sequences(lib, cuda):
    """More sequences than threads of a CTA, most of them empty."""
    lens = [(b % 7 == 0) * (b % 40) for b in range(900)]
    _check_prefix(lib, 50, lens, 2, 1, 64, 16, "bf16", seed=16)


# -------------------------------------------------- as they are used together
def test_serving_chain(lib, cuda):
    """A shared prompt enters the cache and is attended to, every request's own
    prompt follows behind it, then tokens are decoded one by one, each append
    followed by the attention over what is there; every output against 64-bit
    attention over the rotated keys of the whole sequence."""
    import torch

    import cuflash_attn as cf

    dtype, Hq, Hkv, D, ps = torch.bfloat16, 8, 2, 64, 16
    P, own, steps = 150, [40, 1, 17], 3
    B = len(own)
    c = Cache([P] + [n + steps for n in own], ps, Hkv, D, dtype, 20, fill=False)
    rope = cf.rope_table(P + max(own) + steps, D)
    seen = [[], []], [[[], []] for _ in range(B)]
    scale = 1.0 / math.sqrt(D)

    def tokens(n):
        qkv = _randn(c.gen, n, (Hq + 2 * Hkv) * D, dtype=dtype)
        return [x.unflatten(1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], 1)]

    def rotated(k, first):
        pos = torch.arange(first, first + k.shape[0], device="cuda")
        return ref.rotate(k, rope, pos, False)[0].to(dtype)

    def check(O, L, q, k, v, vis, what):
        # keys rounded twice may differ by one step from the cache's: the keys
        # compared are the cache's own, checked against the rotation above
        O64, L64, bO, bL = ref.attend(q, k, v, scale, vis, dtype)
        ref.check(O, O64, bO, what)
        ref.check(L, L64, bL, what)

    # the prompt
    q, k, v = tokens(P)
    qr = lib.kv_append_paged(k, v, c.K, c.V, c.table[:1].contiguous(), _i32([P]), _cu([P]), Q=q,
                             rope_table=rope)
    O, L = lib.forward_paged(qr, c.K, c.V, c.table[:1].contiguous(), _i32([P]), _cu([P]))
    kp, vp = c.get(0, P)
    assert float((kp.double() - rotated(k, 0).double()).abs().max()) <= 2.0 ** -7 * 8
    tri = torch.ones(P, P, device="cuda").tril().bool()
    check(O, L, qr, kp, vp, tri, "prompt")
    # the requests' own prompts: positions behind the shared one
    table = c.table[1:].contiguous()
    q, k, v = tokens(sum(own))
    pos = torch.cat([torch.arange(P, P + n) for n in own]).to(torch.int32).cuda()
    qr = lib.kv_append_paged(k, v, c.K, c.V, table, _i32(own), _cu(own), Q=q, rope_table=rope,
                             positions=pos)
    # their attention reads the prefix's pages too: tables of the whole sequence
    # need the prefix to end with its last page; it does not here (150 of 160),
    # so the last prompt token of each request is decoded instead
    last = torch.tensor([sum(own[:b + 1]) - 1 for b in range(B)], device="cuda")
    lens = list(own)
    O, L = lib.decode_shared_prefix(qr[last].unsqueeze(2), c.K, c.V, c.table[0], _i32([P]), table,
                                    _i32(lens))
    for step in range(steps + 1):
        for b in range(B):
            ko, vo = c.get(1 + b, lens[b])
            check(O[b].transpose(0, 1), L[b][None], q_now(qr, last, b) if step == 0 else
                  qr[b:b + 1], torch.cat([kp, ko]), torch.cat([vp, vo]), None,
                  f"step {step}, request {b}")
        if step == steps:
            break
        lens = [n + 1 for n in lens]
        q, k, v = tokens(B)
        qr = lib.kv_append_paged(k, v, c.K, c.V, table, _i32(lens), Q=q, rope_table=rope,
                                 positions=_i32([P + n - 1 for n in lens]))
        O, L = lib.decode_shared_prefix(qr.unsqueeze(2), c.K, c.V, c.table[0], _i32([P]), table,
                                        _i32(lens))
    assert lib.device_status() == 0


def q_now(qr, last, b):
    return qr[last[b]:last[b] + 1]


def test_agrees_with_paged_decode(lib, cuda):
    """Single tokens without a prefix: ragged forward, shared-prefix decode and
    the library's paged decode compute the same attention."""
    import torch

    lens = [1, 40, 700, 129]
    c = Cache([0] + lens, 16, 2, 128, torch.bfloat16, 21)
    table = c.table[1:].contiguous()
    q = _randn(c.gen, 4, 8, 1, 128, dtype=torch.bfloat16)
    O0, L0 = lib.decode_paged(q, c.K, c.V, table, _i32(lens))
    O1, L1 = lib.forward_paged(q.squeeze(2), c.K, c.V, table, _i32(lens), _cu([1] * 4))
    O2, L2 = lib.decode_shared_prefix(q, c.K, c.V, c.table[0], _i32([0]), table, _i32(lens))
    torch.cuda.synchronize()
    step = 4 * 2.0 ** -8 * float(c.V.nan_to_num().abs().max())
    for O, L in ((O1.unsqueeze(2), L1), (O2, L2)):
        assert float((O.float() - O0.float()).abs().max()) <= step
        assert float((L - L0).abs().max()) < 1e-4


def test_captured_step_follows_lengths(lib, cuda):
    """One captured decode step (append, then attention), replayed as the
    lengths in device memory grow, beside a second graph of the same calls;
    equal to the same calls made eagerly, bit by bit."""
    import torch

    import cuflash_attn as cf

    dtype, Hq, Hkv, D, P, B = torch.bfloat16, 8, 2, 128, 333, 5
    start = [0, 3, 15, 16, 200]
    c = Cache([P] + [n + 40 for n in start], 16, Hkv, D, dtype, 22)
    table = c.table[1:].contiguous()
    rope = cf.rope_table(P + 300, D)
    lens = _i32(start)
    plen = _i32([P])
    pos = lens + P - 1
    cu = _cu([1] * B)
    q, k, v = (_randn(c.gen, B, h, D, dtype=dtype) for h in (Hq, Hkv, Hkv))

    def step():
        qr = lib.kv_append_paged(k, v, c.K, c.V, table, lens, Q=q, rope_table=rope, positions=pos)
        O, L = lib.decode_shared_prefix(qr.unsqueeze(2), c.K, c.V, c.table[0], plen, table, lens)
        O2, L2 = lib.forward_paged(qr, c.K, c.V, table, lens, cu)
        return O, L, O2, L2

    lens += 1
    pos += 1
    step()  # binds the failure word before the capture
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for it in range(6):
        lens += 5
        pos += 5
        graphs[it % 2].replay()
        graphs[(it + 1) % 2].replay()
        want = step()
        torch.cuda.synchronize()
        for o in outs:
            for x, y in zip(o, want):
                assert torch.equal(x, y)
    assert lib.device_status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_entries_with_single_arguments(lib, cuda, dt):
    """The C entries that take their arguments one by one do what the binding's
    packed ones do."""
    import torch

    dtype, Hq, Hkv, D, ps = _dtype(dt), 8, 2, 64, 16
    new, lens, T = [3, 1, 20], [40, 7, 150], 24
    packed, single = (Cache(lens, ps, Hkv, D, dtype, 27) for _ in range(2))
    qkv = _randn(packed.gen, T, Hq + 2 * Hkv, D, dtype=dtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    rope = torch.randn(160, 32, device="cuda")
    cu, sl = _cu(new), _i32(lens)
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 5

    def ptr(t):
        return t.data_ptr()

    def call(entry, *args):
        stream = torch.cuda.current_stream().cuda_stream
        assert getattr(lib.lib, f"cuflash_{entry}_{dt}")(*args, stream) == 0

    want_q = lib.kv_append_paged(k, v, packed.K, packed.V, packed.table, sl, cu, Q=q,
                                 rope_table=rope, positions=pos, interleaved=True)
    got_q, c = torch.empty_like(want_q), single
    row = (Hq + 2 * Hkv) * D
    geometry = (ps, c.table.shape[1], c.num_pages)
    call("kv_append_paged", ptr(q), ptr(k), ptr(v), ptr(got_q), ptr(c.K), ptr(c.V), ptr(rope),
         ptr(pos), ptr(c.table), ptr(sl), ptr(cu), T, 3, Hq, Hkv, D, *geometry, row, row, row, 32,
         160, True)
    assert torch.equal(want_q, got_q)
    for x, y in ((packed.K, c.K), (packed.V, c.V)):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    want = lib.forward_paged(want_q, packed.K, packed.V, packed.table, sl, cu, causal=False,
                             scale=0.2)
    got = [torch.empty_like(x) for x in want]
    call("attention_forward_paged", ptr(got_q), ptr(c.K), ptr(c.V), ptr(c.table), ptr(sl), ptr(cu),
         ptr(got[0]), ptr(got[1]), T, 3, Hq, Hkv, D, *geometry, 0.2, False)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    qd, plen = want_q[:2].unsqueeze(2).contiguous(), _i32([40])
    table, own = c.table[1:].contiguous(), _i32(lens[1:])
    want = lib.decode_shared_prefix(qd, packed.K, packed.V, packed.table[0], plen, table, own,
                                    scale=0.2)
    got = [torch.empty_like(x) for x in want]
    call("attention_decode_shared_prefix", ptr(qd), ptr(c.K), ptr(c.V), ptr(c.table[0]), ptr(plen),
         ptr(table), ptr(own), ptr(got[0]), ptr(got[1]), 2, Hq, Hkv, D, ps, c.table.shape[1],
         c.table.shape[1], c.num_pages, 0.2)
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_two_streams_at_once(lib, cuda):
    """Calls on two streams whose kernels may overlap have their own workspaces."""
    import torch

    lens = [(61 * b) % 500 for b in range(40)]
    c = Cache([1000] + lens, 16, 2, 64, torch.bfloat16, 23)
    table = c.table[1:].contiguous()
    qs = [_randn(c.gen, 40, 8, 1, 64, dtype=torch.bfloat16) for _ in range(2)]
    args = (c.K, c.V, c.table[0], _i32([1000]), table, _i32(lens))
    want = [lib.decode_shared_prefix(q, *args) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [lib.decode_shared_prefix(q, *args, stream=s) for q, s in zip(qs, streams)]
        torch.cuda.synchronize()
        for (O, L), (O2, L2) in zip(got, want):
            assert torch.equal(O, O2) and torch.equal(L, L2)


@pytest.mark.parametrize("captured", [False, True])
def test_inputs_from_another_stream(lib, cuda, captured):
    """Calls back to back, each after a wait for a stream that writes its inputs
    (queries, keys, lengths) late: the kernels start behind the one before them,
    but read nothing before what they wait for is there."""
    import torch

    B, Hq, Hkv, D = 6, 8, 2, 64
    c = Cache([400] * B, 16, Hkv, D, torch.bfloat16, 41)
    k0 = c.K.clone()
    rounds = 8
    srcs = [(_randn(c.gen, B, Hq + 2 * Hkv, D, dtype=torch.bfloat16), _i32([40 * (i + 1)] * B))
            for i in range(rounds)]
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
    c.K.copy_(k0)
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


def test_first_call_is_captured(cuda):
    """In a new process, the first calls may be captured ones."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch, cuflash_attn as cf
lib = cf.CuFlashAttn()
t = lambda *s: torch.randn(*s, device="cuda").bfloat16()
K, V, q, k = t(8, 16, 2, 64), t(8, 16, 2, 64), t(2, 4, 64), t(2, 2, 64)
table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
lens = torch.tensor([60, 17], dtype=torch.int32, device="cuda")
cu = torch.arange(3, dtype=torch.int32, device="cuda")
plen = torch.tensor([16], dtype=torch.int32, device="cuda")
rope = cf.rope_table(64, 64)
def step():
    r = lib.kv_append_paged(k, k, K, V, table, lens, Q=q, rope_table=rope)
    return (*lib.forward_paged(r, K, V, table, lens, cu),
            *lib.decode_shared_prefix(r.unsqueeze(2), K, V, table[0, :1].contiguous(), plen, table, lens))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
want = step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want)) and lib.device_status() == 0
"""
    root = Path(__file__).resolve().parents[1]
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root / "cuflash-attn_b200")


@pytest.mark.parametrize("reserve", [1, 147])
def test_reserved_sms(lib, cuda, reserve):
    """Fewer CTAs cut the work into fewer pieces."""
    import cuflash_attn as cf

    option = lib.lib.cuflash_set_option
    assert option(b"CUFLASH_RESERVE_SMS", reserve) == cf.SUCCESS
    try:
        _check_forward(lib, [1, 300, 1, 7], [900, 1000, 40, 7], 8, 2, 64, 16, "bf16", True, seed=25)
        _check_prefix(lib, 700, [5, 0, 400], 8, 2, 64, 16, "bf16", seed=26)
    finally:
        assert option(b"CUFLASH_RESERVE_SMS", -1) == cf.SUCCESS


def test_offsets_beyond_32_bits(lib, cuda):
    """A pool of more than 2^31 elements: pages at its far end."""
    import torch

    dtype, Hq, Hkv, D, ps = torch.bfloat16, 4, 2, 128, 64
    pages = (1 << 31) // (ps * Hkv * D) + 40
    if torch.cuda.mem_get_info()[0] < 2 * pages * ps * Hkv * D * 2 + (4 << 30):
        pytest.skip("needs 13 GB of device memory")
    c = Cache([200, 300], ps, Hkv, D, dtype, 24, fill=False)
    K = torch.empty((pages, ps, Hkv, D), dtype=dtype, device="cuda")
    V = torch.empty_like(K)
    far = c.table.clone()
    far[c.table >= 0] += pages - c.num_pages
    k, v = (_randn(c.gen, 500, Hkv, D, dtype=dtype) for _ in range(2))
    lens = [200, 300]
    lib.kv_append_paged(k, v, K, V, far, _i32(lens), _cu(lens))
    q = _randn(c.gen, 500, Hq, D, dtype=dtype)
    O, L = lib.forward_paged(q, K, V, far, _i32(lens), _cu(lens))
    O2, L2 = lib.decode_shared_prefix(q[-1:].unsqueeze(2), K, V, far[0], _i32([200]), far[1:],
                                      _i32([300]))
    scale = 1.0 / math.sqrt(D)
    at = 0
    for n in lens:
        vis = torch.ones(n, n, device="cuda").tril().bool()
        sl = slice(at, at + n)
        O64, L64, bO, bL = ref.attend(q[sl], k[sl], v[sl], scale, vis, dtype)
        ref.check(O[sl], O64, bO, "O")
        ref.check(L[sl], L64, bL, "L")
        at += n
    O64, L64, bO, bL = ref.attend(q[-1:], k, v, scale, None, dtype)
    ref.check(O2.squeeze(2), O64, bO, "prefix O")
    ref.check(L2, L64, bL, "prefix L")
