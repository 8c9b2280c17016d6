"""Calls on the 8-bit cache that are refused, checked through the C entry points without a device: nothing is launched."""
import ctypes as C

import pytest

BAD, ALIGN, SCRATCH = -1, -2, -3
P = 1 << 20  # stands for a device address: a refused call never follows it


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as g
    g.build()
    from teenygrad_b200 import _lib
    return _lib


def shape(lib, slots=4, heads=2, cap=100, dim=64, vdim=64, block=32):
    return lib.Cache8Shape(slots, heads, cap, dim, vdim, block)


def host(*entries):
    return (C.c_int * (4 * len(entries)))(*[x for e in entries for x in e])


def append(lib, sh, table=None, n=1, rows=8, longest=8, k=P, kn=P, ldk=None, ks=P):
    ld = sh.kv_heads * sh.dim if ldk is None else ldk
    return lib.lib.teeny_cache8_append(0, C.addressof(sh), k, P, ks, P, None, kn, ld, P, sh.kv_heads * sh.vdim, rows, P, table, n, longest, None)


def attention(lib, sh, table=None, n=1, rows=8, longest=8, heads=4, q=P, out=P, weights=None, softcap=0.0, scratch=P, size=1 << 40, gate=None, ldg=0, ldq=None,
              scale=0.1):
    return lib.lib.teeny_cache8_attention(0, C.addressof(sh), P, P, P, P, weights, 0.5, q, heads * sh.dim if ldq is None else ldq, out, heads * sh.vdim, rows, heads,
                                          scale, softcap, None, gate, ldg, None, scratch, size, P, table, n, longest, None)


def evict(lib, sh, table=None, n=1, keep=10, recent=2, weights=P, kept=P, scratch=P, size=1 << 40):
    return lib.lib.teeny_cache8_evict(C.addressof(sh), P, P, P, P, weights, keep, recent, kept, scratch, size, P, table, n, None)


@pytest.mark.parametrize("change", [dict(slots=0), dict(heads=0), dict(cap=0), dict(dim=0), dict(dim=72), dict(dim=144), dict(vdim=8), dict(vdim=256),
                                    dict(block=0), dict(block=48), dict(block=256), dict(block=-16)])
def test_shapes(lib, change):
    sh = shape(lib, **change)
    assert append(lib, sh) == BAD and attention(lib, sh, heads=4) == BAD and evict(lib, sh) == BAD
    assert lib.lib.teeny_cache8_attention_scratch_bytes(C.addressof(sh), 0, 4, 8, 1, 8, 1) == 0 and lib.lib.teeny_cache8_evict_scratch_bytes(C.addressof(sh), 1, 10) == 0


@pytest.mark.parametrize("table", [[(4, 0, 0, 1)], [(-1, 0, 0, 1)], [(0, -1, 0, 1)], [(0, 100, 0, 1)], [(0, 98, 0, 3)], [(0, 0, 8, 1)], [(0, 0, 6, 3)],
                                   [(0, 0, -1, 1)], [(0, 0, 0, 9)], [(0, 0, 0, -1)], [(0, 2 ** 31 - 1, 0, 1)], [(1, 0, 0, 1), (1, 5, 1, 1)], [(0, 101, 0, 0)]], ids=str)
def test_tables(lib, table):
    sh = shape(lib)
    assert append(lib, sh, host(*table), len(table)) == BAD
    assert attention(lib, sh, host(*table), len(table), weights=P) == BAD
    if len(table) == 1:  # (reading the same slot twice is fine)
        assert attention(lib, sh, host(*table), len(table)) == BAD


@pytest.mark.parametrize("table", [[(0, 0, 0, 2), (1, 0, 1, 2)], [(0, 0, 4, 2), (1, 0, 0, 5)], [(0, 0, 3, 1), (1, 5, 3, 1)], [(0, 0, 6, 2), (1, 0, 0, 0), (2, 0, 0, 7)]], ids=str)
def test_rows_of_two_entries(lib, table):
    assert attention(lib, shape(lib), host(*table), len(table)) == BAD


@pytest.mark.parametrize("table", [[(0, 0, 0, 2), (1, 0, 2, 2)], [(0, 0, 4, 2), (1, 0, 0, 4)], [(0, 0, 3, 1), (1, 5, 3, 0)], [(0, 0, 6, 2), (1, 0, 7, 0), (2, 0, 0, 6)]], ids=str)
def test_rows_apart_in_any_order(lib, table):
    """(Scratch is asked for behind the table.)"""
    assert attention(lib, shape(lib), host(*table), len(table), weights=P, size=3) == SCRATCH


def test_arguments(lib):
    sh = shape(lib)
    assert append(lib, sh, kn=None) == BAD and append(lib, sh, k=None) == BAD and append(lib, sh, ks=None) == BAD and append(lib, sh, ldk=127) == BAD
    assert append(lib, sh, k=P + 8) == ALIGN and append(lib, sh, n=0) == BAD and append(lib, sh, n=65536) == BAD and append(lib, sh, longest=0) == BAD
    assert append(lib, sh, rows=0) == BAD
    assert attention(lib, sh, heads=3) == BAD and attention(lib, sh, heads=0) == BAD and attention(lib, sh, q=None) == BAD and attention(lib, sh, out=None) == BAD
    assert attention(lib, sh, ldq=255) == BAD and attention(lib, sh, softcap=-1.0) == BAD and attention(lib, sh, softcap=float("nan")) == BAD
    assert attention(lib, sh, softcap=1e-39) == BAD and attention(lib, sh, softcap=float("inf")) == BAD
    assert attention(lib, sh, gate=P, ldg=100) == BAD and attention(lib, sh, scale=float("nan")) == BAD
    assert attention(lib, sh, weights=P, scratch=None, size=0) == SCRATCH and attention(lib, sh, weights=P, size=3) == SCRATCH
    assert attention(lib, sh, weights=P, scratch=P + 4) == ALIGN
    assert evict(lib, sh, weights=None) == BAD and evict(lib, sh, kept=None) == BAD and evict(lib, sh, keep=0) == BAD and evict(lib, sh, keep=101) == BAD
    assert evict(lib, sh, recent=11) == BAD and evict(lib, sh, recent=-1) == BAD
    assert evict(lib, sh, host((0, 101, 0, 0))) == BAD and evict(lib, sh, host((0, 5, 0, 0), (0, 6, 0, 0)), 2) == BAD and evict(lib, sh, host((4, 5, 0, 0))) == BAD


def test_scratch_for_a_bound_that_nothing_reaches(lib):
    """max_len may be anything above the longest entry, which has to fit the rows and the cache."""
    size = lambda rows, longest, f32: lib.lib.teeny_cache8_attention_scratch_bytes(C.addressof(shape(lib)), f32, 4, rows, 2, longest, 1)  # noqa: E731
    for f32 in (0, 1):
        assert size(8, 2 ** 31 - 1, f32) == size(8, 8, f32) and size(900, 2 ** 31 - 1, f32) == size(900, 100, f32)


def test_the_wrappers_checks(lib):
    import torch
    from teenygrad_b200 import ops
    z = lambda *s: torch.zeros(*s)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA"):
        ops.Cache8(z(1, 1, 16, 16).to(torch.float8_e4m3fn), z(1, 1, 16, 16).to(torch.float8_e4m3fn), z(1, 1, 1), z(1, 1, 1), 16)
    with pytest.raises(ValueError, match="step table"):
        ops.step_table([], "cpu")
    with pytest.raises(ValueError, match="step table"):
        ops.step_table([(0, 1, 2)], "cpu")
    with pytest.raises(ValueError, match="side by side"):
        ops._head_rows(z(3, 4, 16).transpose(0, 1), 3, 16, "q")
    with pytest.raises(ValueError, match="side by side"):
        ops._head_rows(z(3, 4, 32)[..., ::2], 4, 16, "q")
    assert ops._head_rows(z(5, 100)[:, 8:72].unflatten(1, (4, 16)), 4, 16, "q") == 100
    t = ops.step_table([(0, 3, 0, 2), (1, 0, 2, 5)], "cpu")
    assert (t.n, t.longest, list(t.host)) == (2, 5, [0, 3, 0, 2, 1, 0, 2, 5]) and t.seqs.tolist() == [[0, 3, 0, 2], [1, 0, 2, 5]]


@pytest.mark.parametrize("f32,longest", [(0, 8), (0, 600), (1, 600)])
def test_scratch_off_its_alignment(lib, f32, longest):
    """Prompts' tokens are widened into scratch by stores of 32 bytes: scratch that begins in the middle of 32 is refused, whatever the call's lengths."""
    sh = shape(lib, cap=1000)
    for off in (4, 8, 16, 24, 48, 112):
        assert lib.lib.teeny_cache8_attention(f32, C.addressof(sh), P, P, P, P, None, 0.0, P, 256, P, 256, 700, 4, 0.1, 0.0, None, None, 0, None,
                                              P + off, 1 << 40, P, host((0, 3, 0, longest)), 1, longest, None) == ALIGN
