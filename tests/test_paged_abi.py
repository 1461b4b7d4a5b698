"""Refusals of the paged-cache entries (append, ragged forward, shared-prefix
decode): every invalid call returns its code before any CUDA call, so these
run without a GPU.  The pointers are never dereferenced."""

import ctypes

import pytest

import cuflash_attn as cf

P = ctypes.c_void_p(0x1000)
NUL = ctypes.c_void_p(0)


def _append(lib, sfx="bf16", Q=P, K=P, V=P, Q_out=P, Kc=P, Vc=P, rope=P, positions=NUL, table=P,
            lens=P, cu=P, tokens=4, B=2, Hq=4, Hkv=2, D=64, ps=16, max_pages=4, num_pages=8, qs=0,
            ks=0, vs=0, rotary=64, max_pos=128, interleaved=False):
    return getattr(lib.lib, f"cuflash_kv_append_paged_{sfx}")(
        Q, K, V, Q_out, Kc, Vc, rope, positions, table, lens, cu, tokens, B, Hq, Hkv, D, ps,
        max_pages, num_pages, qs, ks, vs, rotary, max_pos, interleaved, NUL)


def _forward(lib, sfx="bf16", Q=P, Kc=P, Vc=P, table=P, lens=P, cu=P, O=P, L=P, tokens=4, B=2,
             Hq=4, Hkv=2, D=64, ps=16, max_pages=4, num_pages=8, scale=0.125, causal=True):
    return getattr(lib.lib, f"cuflash_attention_forward_paged_{sfx}")(
        Q, Kc, Vc, table, lens, cu, O, L, tokens, B, Hq, Hkv, D, ps, max_pages, num_pages, scale,
        causal, NUL)


def _prefix(lib, sfx="bf16", Q=P, Kc=P, Vc=P, ptab=P, plen=P, table=P, lens=P, O=P, L=P, B=2, Hq=4,
            Hkv=2, D=64, ps=16, max_prefix=4, max_pages=4, num_pages=8, scale=0.125):
    return getattr(lib.lib, f"cuflash_attention_decode_shared_prefix_{sfx}")(
        Q, Kc, Vc, ptab, plen, table, lens, O, L, B, Hq, Hkv, D, ps, max_prefix, max_pages,
        num_pages, scale, NUL)


APPEND = [
    (dict(K=NUL), cf.NULL_POINTER), (dict(V=NUL), cf.NULL_POINTER),
    (dict(Q=NUL), cf.NULL_POINTER), (dict(Q_out=NUL), cf.NULL_POINTER),
    (dict(Kc=NUL), cf.NULL_POINTER), (dict(Vc=NUL), cf.NULL_POINTER),
    (dict(table=NUL), cf.NULL_POINTER), (dict(lens=NUL), cf.NULL_POINTER),
    (dict(tokens=0), cf.INVALID_DIMENSION), (dict(B=0), cf.INVALID_DIMENSION),
    (dict(Hq=0), cf.INVALID_DIMENSION), (dict(Hkv=0), cf.INVALID_DIMENSION),
    (dict(D=0), cf.INVALID_DIMENSION), (dict(D=96), cf.UNSUPPORTED_HEAD_DIM),
    (dict(ps=0), cf.INVALID_DIMENSION), (dict(ps=24), cf.INVALID_DIMENSION),
    (dict(max_pages=0), cf.INVALID_DIMENSION), (dict(num_pages=0), cf.INVALID_DIMENSION),
    (dict(num_pages=1 << 28), cf.INVALID_DIMENSION),
    (dict(max_pages=1 << 28), cf.INVALID_DIMENSION),
    (dict(cu=NUL), cf.DIMENSION_MISMATCH),  # 4 tokens, 2 sequences
    (dict(rotary=0), cf.INVALID_DIMENSION), (dict(rotary=24), cf.INVALID_DIMENSION),
    (dict(rotary=80), cf.INVALID_DIMENSION), (dict(max_pos=0), cf.INVALID_DIMENSION),
    (dict(qs=128), cf.INVALID_DIMENSION), (dict(qs=260), cf.INVALID_DIMENSION),
    (dict(ks=64), cf.INVALID_DIMENSION), (dict(vs=-128), cf.INVALID_DIMENSION),
    (dict(qs=512), cf.INVALID_DIMENSION),  # in place (Q == Q_out) but not contiguous
    (dict(Hkv=1 << 30), cf.INVALID_DIMENSION),
    (dict(K=ctypes.c_void_p(0x1008)), cf.CUDA_ERROR),  # 16-byte alignment
]

FORWARD = [
    *[({k: NUL}, cf.NULL_POINTER) for k in ("Q", "Kc", "Vc", "table", "lens", "cu", "O", "L")],
    (dict(tokens=0), cf.INVALID_DIMENSION), (dict(B=-1), cf.INVALID_DIMENSION),
    (dict(Hq=0), cf.INVALID_DIMENSION), (dict(Hkv=0), cf.INVALID_DIMENSION),
    (dict(Hq=3), cf.DIMENSION_MISMATCH), (dict(D=48), cf.UNSUPPORTED_HEAD_DIM),
    (dict(ps=12), cf.INVALID_DIMENSION), (dict(max_pages=0), cf.INVALID_DIMENSION),
    (dict(num_pages=0), cf.INVALID_DIMENSION), (dict(num_pages=1 << 28), cf.INVALID_DIMENSION),
    (dict(scale=float("nan")), cf.INVALID_DIMENSION), (dict(scale=-1.0), cf.INVALID_DIMENSION),
    (dict(scale=float("inf")), cf.INVALID_DIMENSION),
    (dict(tokens=1 << 30, Hq=4), cf.INVALID_DIMENSION),
    (dict(Q=ctypes.c_void_p(0x1004)), cf.CUDA_ERROR),
]

PREFIX = [
    *[({k: NUL}, cf.NULL_POINTER)
      for k in ("Q", "Kc", "Vc", "ptab", "plen", "table", "lens", "O", "L")],
    (dict(B=0), cf.INVALID_DIMENSION), (dict(max_prefix=0), cf.INVALID_DIMENSION),
    (dict(max_prefix=1 << 28), cf.INVALID_DIMENSION), (dict(ps=3), cf.INVALID_DIMENSION),
    (dict(Hq=5), cf.DIMENSION_MISMATCH), (dict(D=256), cf.UNSUPPORTED_HEAD_DIM),
    (dict(scale=-0.5), cf.INVALID_DIMENSION),
    (dict(Vc=ctypes.c_void_p(0x1002)), cf.CUDA_ERROR),
]


@pytest.mark.parametrize("sfx", ["bf16", "f16"])
@pytest.mark.parametrize("kw,code", APPEND, ids=lambda x: str(x)[:40])
def test_append_refusals(lib, sfx, kw, code):
    assert _append(lib, sfx, **kw) == code


@pytest.mark.parametrize("sfx", ["bf16", "f16"])
@pytest.mark.parametrize("kw,code", FORWARD, ids=lambda x: str(x)[:40])
def test_forward_paged_refusals(lib, sfx, kw, code):
    assert _forward(lib, sfx, **kw) == code


@pytest.mark.parametrize("sfx", ["bf16", "f16"])
@pytest.mark.parametrize("kw,code", PREFIX, ids=lambda x: str(x)[:40])
def test_shared_prefix_refusals(lib, sfx, kw, code):
    assert _prefix(lib, sfx, **kw) == code


def _ptr(x):
    return x.value or 0 if isinstance(x, ctypes.c_void_p) else x


class _Packed:
    """The entries as their plain forms are called, through the packed ones."""

    def __init__(self, lib):
        self.raw, self.lib = lib.lib, self

    def __getattr__(self, name):
        entry, sfx = name.rsplit("_", 1)
        fn = getattr(self.raw, f"{entry}_args_{sfx}")

        def call(*a):
            a = [_ptr(x) for x in a]
            if entry == "cuflash_kv_append_paged":
                return fn(cf.APPEND_ARGS.pack(*a[:11], *a[19:22], *a[11:19], *a[22:]))
            if entry == "cuflash_attention_forward_paged":
                return fn(cf.PAGED_ARGS.pack(*a[:3], 0, 0, *a[3:14], 0, *a[14:16], a[17], a[16],
                                             a[18]))
            return fn(cf.PAGED_ARGS.pack(*a[:7], 0, *a[7:9], a[9], *a[9:17], 0, *a[17:]))

        return call


@pytest.mark.parametrize("sfx", ["bf16", "f16"])
def test_packed_arguments_refuse_alike(lib, sfx):
    """Each field arrives in its place: every refusal, through the struct."""
    packed = _Packed(lib)
    for call, cases in ((_append, APPEND), (_forward, FORWARD), (_prefix, PREFIX)):
        for kw, code in cases:
            assert call(packed, sfx, **kw) == code, kw
    for entry in ("kv_append_paged", "attention_forward_paged", "attention_decode_shared_prefix"):
        assert getattr(lib.lib, f"cuflash_{entry}_args_{sfx}")(None) == cf.NULL_POINTER


def test_packed_arguments_layout(tmp_path):
    """The binding's formats have the sizes and offsets of the header's structs."""
    import shutil
    import subprocess
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    cuda = Path(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc").resolve().parents[1] / "include"
    if not shutil.which("g++") or not (cuda / "cuda_runtime.h").exists():
        pytest.skip("needs g++ and the CUDA headers")
    src = tmp_path / "layout.cpp"
    src.write_text("""
#include <cstddef>
#include <cstdio>
#include "cuflash/flash_attention.h"
#define AT(S, F) offsetof(S, F)
int main() {
    using A = CuflashKvAppendArgs;
    using P = CuflashPagedAttentionArgs;
    std::printf("%zu %zu %zu %zu %zu %zu %zu %zu", sizeof(A), AT(A, q_stride), AT(A, num_tokens),
                AT(A, stream), sizeof(P), AT(P, num_tokens), AT(P, scale), AT(P, stream));
}
""")
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", "-I", str(root / "include"), "-I", str(cuda), str(src),
                    "-o", str(exe)], check=True)
    import struct

    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    a, p = cf.APPEND_ARGS, cf.PAGED_ARGS
    assert got == [a.size, struct.calcsize("@11P"), struct.calcsize("@11P3q"), a.size - 8,
                   p.size, struct.calcsize("@10P"), struct.calcsize("@10P10i"), p.size - 8]


def test_binding_refuses_before_the_library(lib):
    """Shapes, types and devices are checked by the binding (CPU tensors)."""
    import torch

    bf, i32 = torch.bfloat16, torch.int32
    K = torch.zeros(3, 2, 64, dtype=bf)
    cache = torch.zeros(4, 16, 2, 64, dtype=bf)
    table, lens = torch.zeros(3, 2, dtype=i32), torch.ones(3, dtype=i32)
    cu = torch.zeros(4, dtype=i32)
    call = lib.kv_append_paged
    with pytest.raises(ValueError):  # not CUDA tensors
        call(K, K, cache, cache, table, lens)
    with pytest.raises(cf.CuFlashError):
        call(K, K[:, :1], cache, cache, table, lens)
    with pytest.raises(cf.CuFlashError):
        call(K, K, cache, cache.half(), table, lens)
    with pytest.raises(cf.CuFlashError):
        call(K, K, cache, cache, table.long(), lens)
    with pytest.raises(cf.CuFlashError):
        call(K, K, cache, cache, table, lens, cu_seqlens=cu[:3])
    with pytest.raises(ValueError):
        call(K, K, cache, cache, table, lens, Q_out=K)
    with pytest.raises(ValueError):  # one row for every token
        call(K[:1].expand(3, 2, 64), K, cache, cache, table, lens)
    Q = torch.zeros(3, 4, 64, dtype=bf)
    with pytest.raises(cf.CuFlashError):
        lib.forward_paged(Q, cache, cache, table, lens, cu[:2])
    with pytest.raises(ValueError):
        lib.forward_paged(Q, cache, cache, table, lens, cu,
                          L=torch.zeros(3, 4, dtype=torch.float64))
    with pytest.raises(cf.CuFlashError):
        lib.decode_shared_prefix(Q.view(3, 4, 1, 64), cache, cache, table[0], lens, table, lens)


def test_rope_table_angles():
    import math

    import torch

    t = cf.rope_table(70000, 32, base=10000.0, device="cpu")
    assert t.shape == (70000, 32) and t.dtype == torch.float32
    for pos, i in ((0, 0), (1, 0), (69999, 0), (69999, 7), (12345, 15)):
        a = pos * 10000.0 ** (-i / 16)
        assert abs(t[pos, i].item() - math.cos(a)) <= 2.0 ** -24 + 1e-10
        assert abs(t[pos, 16 + i].item() - math.sin(a)) <= 2.0 ** -24 + 1e-10
