"""Plain 64-bit forms of the paged-cache operators and the error bounds their
tests use.  Everything is torch float64 on the device of its inputs.

Bounds (u = half a step of the 16-bit type, torch.finfo(t).eps / 2):

* rotation: x c + w s in fp32 is one rounded product and one fused
  multiply-add, each off by at most 2^-24 of its magnitude; the result is
  rounded once to the type (u relative, or half the smallest subnormal).
* scores: products of 16-bit values are exact in fp32; a sum of D of them is
  off by at most D 2^-23 of the sum of magnitudes (2^-23: the tensor core may
  truncate); scaling, the maximum's subtraction and ex2 add 2^-21 of the
  largest score magnitude (plus 1) in the exponent.
* output: numerator and denominator both carry the scores' error; P is rounded
  to the type (u, or half the smallest f16 subnormal per key: the running
  maximum never exceeds the true one, so the sum of P is at least 1); the
  sums over n keys add n 2^-23; the result is rounded once.
"""

import torch

EPS32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half of the smallest subnormal."""
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def cache_rows(table_row, idx, page_size):
    return table_row[idx // page_size].long() * page_size + idx % page_size


def rotate(x, rope, pos, interleaved):
    """x [n, heads, D] -> (rotated, magnitude of the terms), float64."""
    half = rope.shape[1] // 2
    c, s = rope[pos, :half].double()[:, None], rope[pos, half:].double()[:, None]
    x = x.double()
    y, mag = x.clone(), x.abs()
    i = torch.arange(half, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    mag[..., lo], mag[..., hi] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, mag


def rotate_bound(y, mag, dtype):
    return half_step(dtype) * y.abs() + smallest(dtype) + 2 * 1.01 * EPS32 * mag


def attend(q, k, v, scale, visible, dtype):
    """q [n, hq, D], k and v [m, hkv, D] (16-bit), visible bool [n, m] or None.
    Returns O, L in float64 and their bounds."""
    n, hq, D = q.shape
    m, hkv, _ = k.shape
    g = hq // hkv
    dev = q.device
    O = torch.zeros((n, hq, D), dtype=torch.float64, device=dev)
    L = torch.full((n, hq), -float("inf"), dtype=torch.float64, device=dev)
    bO, bL = torch.zeros_like(O), torch.zeros_like(L)
    if m == 0:
        return O, L, bO, bL
    u = half_step(dtype)
    for h in range(hq):
        qh, kh, vh = q[:, h].double(), k[:, h // g].double(), v[:, h // g].double()
        s = qh @ kh.T * scale
        mag = qh.abs() @ kh.abs().T * scale
        if visible is not None:
            s = s.masked_fill(~visible, -float("inf"))
            mag = mag.masked_fill(~visible, 0.0)
        top = s.amax(1, keepdim=True)
        dead = torch.isneginf(top)
        p = torch.exp(s - torch.where(dead, torch.zeros_like(top), top))
        l = p.sum(1, keepdim=True)
        ls = l.clamp_min(1e-300)
        O[:, h] = torch.where(dead, 0.0, p @ vh / ls)
        L[:, h] = torch.where(dead, -float("inf"), top + torch.log(ls))[:, 0]
        mass = p @ vh.abs() / ls
        e_s = D * 2 * EPS32 * mag.amax(1, keepdim=True) + 8 * EPS32 * (
            mag.amax(1, keepdim=True) + 1)
        acc = (m + 64) * 2 * EPS32
        bO[:, h] = (u * O[:, h].abs() + smallest(dtype) + mass * (u + 2 * e_s + 2 * acc) +
                    smallest(dtype) * vh.abs().sum(0) / ls.clamp_min(1.0))
        bL[:, h] = (e_s + acc)[:, 0] + 4 * EPS32 * torch.where(
            dead[:, 0], 0.0, L[:, h].abs().nan_to_num(0.0, 0.0, 0.0) + 1)
        bO[:, h] = torch.where(dead, 0.0, bO[:, h])
        bL[:, h] = torch.where(dead[:, 0], 0.0, bL[:, h])
    return O, L, bO, bL


def check(got, want, bound, what):
    """Elementwise |got - want| <= bound; infinities have to agree."""
    got = got.double().reshape(want.shape)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    err = (got - want)[~inf].abs()
    over = err > bound[~inf]
    assert not bool(torch.isnan(got).any()), f"{what}: NaN"
    assert not bool(over.any()), (
        f"{what}: {int(over.sum())} of {over.numel()} beyond the bound, worst "
        f"{float(err[over].max())} against {float(bound[~inf][over].min())}")
