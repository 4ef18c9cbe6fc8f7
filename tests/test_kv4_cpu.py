"""The paged cache's entry points refuse what they cannot run before anything reaches a GPU, and the 64-bit restatement
that the GPU tests compare with holds what the header says of the format."""
import ctypes

import pytest
import torch

import kv4_ref as ref
from oumu_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


P = ctypes.c_void_p(1 << 20)    # never dereferenced: every check comes before any work
ODD = ctypes.c_void_p((1 << 20) + 2)
INVALID, UNSUPPORTED, WORKSPACE = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE


def test_page_bytes(lib):
    assert lib.oumu_kv4_page_bytes(2, 128) == 2 * 64 * 160
    assert lib.oumu_kv4_page_bytes(3, 64) == 3 * 64 * 80
    assert lib.oumu_kv4_page_bytes(2, 96) == 0 and lib.oumu_kv4_page_bytes(0, 128) == 0


@pytest.mark.parametrize("args,status", [
    ((None, P, P, P, P, 1, 1, 16, 2, 128, 4, 4), INVALID),
    ((P, P, None, P, P, 1, 1, 16, 2, 128, 4, 4), INVALID),
    ((P, P, P, P, P, 1, -1, 16, 2, 128, 4, 4), INVALID),
    ((P, P, P, P, P, 0, 1, 16, 2, 128, 4, 4), INVALID),
    ((P, P, P, P, P, 1, 1, 16, 0, 128, 4, 4), INVALID),
    ((P, P, P, P, P, 1, 1, 16, 2, 128, 0, 4), INVALID),
    ((P, P, P, P, P, 1, 1, 16, 2, 96, 4, 4), UNSUPPORTED),
    ((P, P, P, P, P, 4097, 1, 16, 2, 128, 4, 4), UNSUPPORTED),
    ((P, P, P, P, P, 1, 1, 16, 2, 128, 4, 1 << 25), UNSUPPORTED),
    ((ODD, P, P, P, P, 1, 1, 16, 2, 128, 4, 4), INVALID),
    ((P, P, P, None, None, 1, 257, 16, 2, 128, 4, 4), INVALID),  # more rows than the table has room for
    ((P, P, P, P, P, 1, 0, 16, 2, 128, 4, 4), _lib.OK),
])
def test_write_refusals(lib, args, status):
    assert lib.oumu_kv4_write(*args, None) == status


@pytest.mark.parametrize("args,status", [
    ((P, P, None, None, P, P, 1, 2, 128, 4, 4, 256), INVALID),
    ((P, P, P, None, None, P, 1, 2, 128, 4, 4, 256), INVALID),
    ((P, P, P, None, P, P, 1, 2, 128, 4, 4, 0), INVALID),
    ((P, P, P, None, P, P, 1, 2, 32, 4, 4, 256), UNSUPPORTED),
    ((P, P, P, None, P, ODD, 1, 2, 128, 4, 4, 256), INVALID),
])
def test_read_refusals(lib, args, status):
    assert lib.oumu_kv4_read(*args, None) == status


def test_attention_refusals(lib):
    def attn(qkv=P, pool=P, out=P, ws=P, n=1 << 24, table=P, pos=None, lens=P, B=4, nq=16, nk=2, hd=128, npages=8,
             maxpages=8, scale=0.1):
        return lib.oumu_attn_decode_kv4(qkv, pool, out, ws, n, table, pos, lens, B, nq, nk, hd, npages, maxpages, scale,
                                        None)

    for k in ("qkv", "pool", "out", "ws", "table", "lens"):
        assert attn(**{k: None}) == INVALID, k
    for k in ("qkv", "pool", "out", "ws"):
        assert attn(**{k: ODD}) == INVALID, k
    assert attn(nq=15) == INVALID and attn(scale=0.0) == INVALID and attn(scale=float("nan")) == INVALID
    assert attn(nq=18) == UNSUPPORTED and attn(hd=96) == UNSUPPORTED and attn(B=4097) == UNSUPPORTED
    assert attn(B=4096, maxpages=1 << 18) == UNSUPPORTED  # more tiles than the kernel counts
    assert attn(n=256) == WORKSPACE
    step = lib.oumu_attn_decode_kv4_step
    assert step(P, P, P, ODD, P, 1 << 24, P, P, 512, P, None, P, 4, 16, 2, 128, 8, 8, 0.1, None) == INVALID
    assert step(P, P, P, None, P, 1 << 24, P, None, 512, P, None, P, 4, 16, 2, 128, 8, 8, 0.1, None) == INVALID
    assert step(P, P, P, None, P, 1 << 24, P, P, 0, P, None, P, 4, 16, 2, 128, 8, 8, 0.1, None) == INVALID
    assert lib.oumu_attn_decode_kv4_workspace(4, 18, 2, 128, 8) == 0
    assert lib.oumu_attn_decode_kv4_workspace(4, 16, 2, 128, 0) == 0
    assert lib.oumu_attn_decode_kv4_workspace(4, 16, 2, 128, 8) > 0


def test_page_refusals(lib):
    assert lib.oumu_pages_extend(P, P, P, -1, P, 4, 8, 8, None) == INVALID
    assert lib.oumu_pages_extend(P, P, P, 0, P, 4097, 8, 8, None) == UNSUPPORTED
    fork = lib.oumu_pages_fork
    assert fork(None, 0, 1, 16, P, P, P, P, P, 1, P, 4, 8, 8, None) == INVALID
    assert fork(P, 0, 1, 24, P, P, P, P, P, 1, P, 4, 8, 8, None) == INVALID  # page bytes not a multiple of 16
    assert fork(P, 64, 2, 16, P, P, P, P, P, 1, P, 4, 8, 8, None) == INVALID  # layers overlap
    assert fork(P, 0, 1, 16, P, P, P, None, P, 1, P, 4, 8, 8, None) == INVALID
    assert fork(P, 0, 1, 16, P, P, P, P, P, 4097, P, 4, 8, 8, None) == UNSUPPORTED
    assert lib.oumu_pages_free(P, P, P, None, 1, 4, 8, 8, None) == INVALID
    assert lib.oumu_pages_free(P, P, P, None, 0, 4, 8, 8, None) == _lib.OK
    need = lib.oumu_pages_workspace(8)
    assert need > 0 and lib.oumu_pages_workspace(0) == 0
    assert lib.oumu_pages_compact(P, 128, 1, 16, P, P, P, need - 1, P, 4, 8, 8, None) == WORKSPACE
    assert lib.oumu_pages_compact(P, 128, 1, 16, P, P, ODD, need, P, 4, 8, 8, None) == INVALID


def test_refusals_of_tables_and_pools_that_int_cannot_count(lib):
    for npages, B, maxpages in (((1 << 30) + 1, 4, 8), ((1 << 31) - 1, 1, 8), (8, 4096, 1 << 19), (8, 64, 1 << 25)):
        assert lib.oumu_pages_extend(P, P, P, 0, P, B, npages, maxpages, None) == UNSUPPORTED
        assert lib.oumu_pages_fork(P, 0, 1, 16, P, P, P, P, P, 1, P, B, npages, maxpages, None) == UNSUPPORTED
        assert lib.oumu_pages_free(P, P, P, P, 1, B, npages, maxpages, None) == UNSUPPORTED
        assert lib.oumu_pages_compact(P, 1 << 40, 1, 16, P, P, P, 1 << 40, P, B, npages, maxpages, None) == UNSUPPORTED
        assert lib.oumu_kv4_write(P, P, P, None, None, B, 4, 16, 2, 128, npages, maxpages, None) == UNSUPPORTED
        assert lib.oumu_kv4_read(P, P, P, None, P, P, B, 2, 128, npages, maxpages, 64, None) == UNSUPPORTED
    assert lib.oumu_pages_workspace((1 << 30) + 1) == 0
    assert lib.oumu_pages_workspace(1 << 30) == 4 * (4 + 2 * ((1 << 29) + 1) + (1 << 30))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["k", "v"])
def test_every_code_has_a_place_of_its_own(hd, kind):
    seen = {(at, sh) for p in range(64) for c in range(hd) for at, sh, *_ in [ref.where(hd, kind, p, c)]}
    assert len(seen) == 64 * hd


@pytest.mark.parametrize("size", [1e-38, 1e-3, 1.0, 1e30])
def test_held_values_are_within_half_a_scale(size):
    x = (torch.randn(300, 64, generator=torch.Generator().manual_seed(5)) * size).bfloat16().double()
    n, s, z, v = ref.held(x)
    assert int(n.max()) <= 15 and int(n.min()) == 0
    assert bool(((v - x).abs().unflatten(-1, (-1, 32)) <= s[..., None] / 2).all())
    assert bool((s * 15 >= (x.unflatten(-1, (-1, 32)).amax(-1) - z)).all())
