"""Failure detection of the attention over a paged cache, without a GPU fault: the
first CTA's first keys never count as landed (a test option; every load is issued
and lands), the waits for them run out after a limit of 50 ms, the kernel tears
down and returns, and the failure is reported by the next call of any entry and
then cleared.  The joining kernels behind the failed one write nothing."""

import time

import pytest

import cuflash_attn as cf
from test_gpu_paged import Cache, _cu, _i32, _randn

pytestmark = pytest.mark.gpu

WAIT_TIMEOUT = 1  # kStatusWaitTimeout


def _tiles(lib, D, dtype):
    """Row tiles only."""
    new, lens = [300, 70, 200], [900, 2000, 200]
    c = Cache(lens, 16, 2, D, dtype, 71)
    q = _randn(c.gen, sum(new), 8, D, dtype=dtype)
    args = (c.K, c.V, c.table, _i32(lens), _cu(new))
    return lambda **out: lib.forward_paged(q, *args, **out)


def _few(lib, D, dtype):
    """Single tokens only, on enough keys that every CTA has some."""
    lens = [20000] * 8
    c = Cache(lens, 64, 2, D, dtype, 72)
    q = _randn(c.gen, 8, 8, D, dtype=dtype)
    args = (c.K, c.V, c.table, _i32(lens), _cu([1] * 8))
    return lambda **out: lib.forward_paged(q, *args, **out)


def _prefix(lib, D, dtype):
    lens = [150] * 30
    c = Cache([4000] + lens, 16, 2, D, dtype, 73)
    q = _randn(c.gen, 30, 8, 1, D, dtype=dtype)
    args = (c.K, c.V, c.table[0], _i32([4000]), c.table[1:].contiguous(), _i32(lens))
    return lambda **out: lib.decode_shared_prefix(q, *args, **out)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("make", [_tiles, _few, _prefix])
def test_wait_timeout_is_reported_then_cleared(lib, cuda, make, D):
    import torch

    call = make(lib, D, torch.bfloat16)
    # a normal call first (it also binds the host-visible status word)
    O_ref, L_ref = call()
    torch.cuda.synchronize()
    assert lib.device_status() == 0
    O, L = torch.full_like(O_ref, 55.0), torch.full_like(L_ref, 55.0)
    lib.set_option("CUFLASH_TEST_WAIT_LIMIT_MS", 50)
    lib.set_option("CUFLASH_TEST_SKIP_K_LOAD", 1)
    try:
        t0 = time.monotonic()
        call(O=O, L=L)  # the launch itself is fine
        torch.cuda.synchronize()  # the kernel returns: its waits are bounded
        elapsed = time.monotonic() - t0
    finally:
        lib.set_option("CUFLASH_TEST_WAIT_LIMIT_MS", -1)
        lib.set_option("CUFLASH_TEST_SKIP_K_LOAD", -1)
    assert elapsed < 3.0, elapsed
    try:
        with pytest.raises(cf.CuFlashError) as e:
            call(O=O, L=L)
        assert e.value.code == cf.CUDA_ERROR
        with pytest.raises(cf.CuFlashError):
            lib.forward(*[O_ref.view(1, -1, 8, D).transpose(1, 2).contiguous()] * 3)
    finally:
        code = lib.device_status()  # reads and clears
    assert code == WAIT_TIMEOUT
    assert lib.device_status() == 0
    # a row is whole or untouched: nothing was joined from missing partials
    same, kept = (O == O_ref).all(-1), (O == 55.0).all(-1)
    assert bool((same | kept).all()) and bool(kept.any())
    # the library works again, with the same results as before
    O2, L2 = call(O=O, L=L)
    torch.cuda.synchronize()
    assert lib.device_status() == 0
    assert torch.equal(O2, O_ref) and torch.equal(L2, L_ref)
