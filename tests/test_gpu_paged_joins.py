"""Attention over a paged cache where a unit is shared by many CTAs: joins of more
than 16 partials, with partials in which a row sees no key and with NaN in some,
and groups between the sizes of the forms for few rows.  The bounds are those of
tests/paged_ref.py."""

import pytest

from test_gpu_paged import Cache, _check_forward, _check_prefix, _cu, _dtype, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [9, 10, 11, 12, 13, 14, 15])
def test_prefix_groups_between_8_and_16(lib, cuda, group):
    _check_prefix(lib, 700, [90, 0, 3, 129], 2 * group, 2, 64 if group % 2 else 128, 16, "bf16",
                  seed=80 + group)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_many_partials(lib, cuda, dt, D):
    """About 140 partials of one unit; in the causal one the last of them hold keys
    that its first rows do not see."""
    _check_forward(lib, [256], [20000], 1, 1, D, 16, dt, True, seed=90)
    _check_forward(lib, [1], [30000], 4, 1, D, 64, dt, True, seed=91)
    _check_prefix(lib, 20000, [700, 0, 5], 4, 1, D, 16, dt, seed=92)


@pytest.mark.parametrize("D", [32, 64, 128])
def test_not_a_number_among_many_partials(lib, cuda, D):
    import torch

    dtype = _dtype("bf16")
    nan = float("nan")

    def same_but(got, want, hit):
        (O, L), (O0, L0) = got, want
        assert torch.equal(torch.isnan(L), hit)
        assert torch.equal(torch.isnan(O).any(-1), hit) and torch.equal(torch.isnan(O).all(-1), hit)
        assert torch.equal(O[~hit], O0[~hit]) and torch.equal(L[~hit], L0[~hit])

    for new, n, key in ((1, 30000, 20000), (40, 30000, 29990), (40, 30000, 5)):
        c = Cache([n], 16, 2, D, dtype, 93)
        q = _randn(c.gen, new, 8, D, dtype=dtype)
        args = (c.table, _i32([n]), _cu([new]))
        want = lib.forward_paged(q, c.K, c.V, *args)
        K = c.K.clone()
        K.view(-1, 2, D)[c.rows(0, n)[key], 1, 2] = nan
        hit = torch.zeros((new, 8), dtype=torch.bool, device="cuda")
        hit[max(0, key - (n - new)):, 4:] = True
        same_but(lib.forward_paged(q, K, c.V, *args), want, hit)
        q2 = q.clone()
        q2[new // 2, 3, 0] = nan  # one row's query
        hit[:] = False
        hit[new // 2, 3] = True
        same_but(lib.forward_paged(q2, c.K, c.V, *args), want, hit)

    c = Cache([30000, 900, 20], 16, 2, D, dtype, 94)
    q = _randn(c.gen, 3, 8, 1, D, dtype=dtype)
    own = torch.zeros((3, c.table.shape[1]), dtype=torch.int32, device="cuda")
    own[0], own[2] = c.table[1], c.table[2]
    args = (c.table[0], _i32([30000]), own, _i32([900, 0, 20]))

    def prefix(q, K):
        O, L = lib.decode_shared_prefix(q, K, c.V, *args)
        return O[:, :, 0], L

    want = prefix(q, c.K)
    K = c.K.clone()
    K.view(-1, 2, D)[c.rows(0, 30000)[12345], 0, 1] = nan
    K.view(-1, 2, D)[c.rows(1, 900)[899], 1, 1] = nan
    hit = torch.zeros((3, 8), dtype=torch.bool, device="cuda")
    hit[:, :4] = True
    hit[0, 4:] = True
    same_but(prefix(q, K), want, hit)
