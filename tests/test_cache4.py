"""The 4-bit K / V cache's entry points without a GPU: what they refuse, and the size query."""
import ctypes

import numpy as np
import pytest
import torch

import asr_amd
from asr_amd import _lib, ops


def cache(*lead, T=8):
    return ops.Cache4(torch.zeros(*lead, T, 32, dtype=torch.uint8), torch.zeros(*lead, T, 2, dtype=torch.bfloat16))


def test_cache4_shapes_and_views():
    c = ops.Cache4.empty(6, 3, 4, 8, "cpu")
    assert c.shape == (6, 3, 4, 8) and len(c) == 6 and c[5].shape == (1, 3, 4, 8) and len(c[5]) == 1
    c[2].codes.fill_(7)
    assert int(c.codes[2].min()) == 7 and int(c.codes[3].max()) == 0        # views of the stack's memory
    assert ops.Cache4.empty(None, 3, 4, 8, "cpu").shape == (1, 3, 4, 8)
    with pytest.raises(IndexError):
        c[0][0]
    assert c[2:4].shape == (2, 3, 4, 8) and c[2:4].codes.data_ptr() == c[2].codes.data_ptr()


@pytest.mark.parametrize("index", [[0, 2], torch.tensor([0, 2]), torch.tensor([True] * 2 + [False] * 4), (0, 1), None, ...])
def test_cache4_indices_that_would_copy_are_refused(index):
    """a list or a mask would make another cache: what is put there would not be in this one"""
    with pytest.raises(TypeError):
        ops.Cache4.empty(6, 3, 4, 8, "cpu")[index]


def test_cache4_whole_number_indices():
    c = ops.Cache4.empty(6, 3, 4, 8, "cpu")
    for i in (-1, torch.tensor(5), np.int64(5)):
        assert c[i].codes.data_ptr() == c.codes[5].data_ptr()
    assert len([k for k in c]) == 6


@pytest.mark.parametrize("codes,meta,err", [
    (torch.zeros(2, 3, 8, 32, dtype=torch.int8), torch.zeros(2, 3, 8, 2, dtype=torch.bfloat16), TypeError),
    (torch.zeros(2, 3, 8, 32, dtype=torch.uint8), torch.zeros(2, 3, 8, 2), TypeError),
    (torch.zeros(2, 3, 8, 64, dtype=torch.uint8), torch.zeros(2, 3, 8, 2, dtype=torch.bfloat16), ValueError),
    (torch.zeros(2, 3, 8, 32, dtype=torch.uint8), torch.zeros(2, 3, 9, 2, dtype=torch.bfloat16), ValueError),
    (torch.zeros(3, 8, 32, dtype=torch.uint8), torch.zeros(3, 8, 2, dtype=torch.bfloat16), ValueError),
    (torch.zeros(2, 8, 3, 32, dtype=torch.uint8).transpose(1, 2), torch.zeros(2, 3, 8, 2, dtype=torch.bfloat16), ValueError),
])
def test_cache4_refuses(codes, meta, err):
    with pytest.raises(err):
        ops.Cache4(codes, meta)


def test_cpu_tensors_are_refused():
    c = cache(2, 3, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.cache4_put(c, torch.zeros(2, 3, 4, 1, 64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.cache4_get(c)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.cache4_attention(torch.zeros(3, 4, 1, 64), c[0], c[1])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.cache4_reorder(cache(2, 6, 4), torch.zeros(6, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), 3)


def test_argument_checks():
    c = cache(2, 3, 4)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    for x in (torch.zeros(2, 3, 4, 1, 32), torch.zeros(3, 4, 1, 64), torch.zeros(2, 3, 5, 1, 64), torch.zeros(2, 3, 4, 64, 2).transpose(3, 4)):
        with pytest.raises(ValueError):
            ops.cache4_put(c, x)
    x = torch.zeros(2, 3, 4, 1, 64)
    for kw in (dict(pos=i32(0, 0)), dict(pos=torch.zeros(3)), dict(pos=torch.zeros(3, dtype=torch.int64)), dict(n_new=i32(1)), dict(pos=torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            ops.cache4_put(c, x, **kw)
    with pytest.raises(ValueError):
        ops.cache4_get(c, L=-1)
    q = torch.zeros(3, 8, 1, 64)
    for args in ((torch.zeros(3, 8, 64), c[0], c[1]), (torch.zeros(3, 8, 1, 32), c[0], c[1]), (torch.zeros(2, 8, 1, 64), c[0], c[1]), (torch.zeros(3, 6, 1, 64), c[0], c[1]),
                 (q, c, c), (q, c[0], cache(3, 4, T=9)), (q.transpose(2, 3), c[0], c[1])):
        with pytest.raises(ValueError):
            ops.cache4_attention(*args)
    for k_len in (i32(1, 1), torch.ones(3, dtype=torch.int64), torch.ones(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            ops.cache4_attention(q, c[0], c[1], k_len=k_len)
    with pytest.raises(TypeError):
        ops.cache4_attention(q.double(), c[0], c[1])
    r, st = cache(2, 6, 4), i32(3, -1)
    par = torch.zeros(6, dtype=torch.int64)
    for args in ((r, par, st, 4), (r, par, st, 0), (r, par[:5], st, 3), (r, par.int(), st, 3), (r, par, st.long(), 3)):
        with pytest.raises(ValueError):
            ops.cache4_reorder(*args)
    with pytest.raises(ValueError):
        ops.cache4_reorder(r, par, st, 3, out=c)
    codes, meta = torch.zeros(3, 6, 4, 8, 32, dtype=torch.uint8), torch.zeros(3, 6, 4, 8, 2, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps"):
        ops.cache4_reorder(ops.Cache4(codes[:2], meta[:2]), par, st, 3, out=ops.Cache4(codes[1:], meta[1:]))


def test_library_refuses_before_it_launches():
    """host-side checks of the C entry points: a code and a message, nothing is launched (there is no device here)"""
    L = asr_amd.lib()
    p = lambda v=64: ctypes.c_void_p(v)  # noqa: E731   (never dereferenced)

    def put(x=64, dt=1, st=(0, 0, 0, 64), codes=64, meta=64, ps=0, sizes=(1, 1, 1, 1, 8)):
        return L.asr_cache4_put(None, p(x) if x else None, dt, *st, p(codes), p(meta), None, ps, None, *sizes)
    assert put(x=0) == -1 and b"cache4_put" in L.asr_last_error()
    assert put(dt=2) == -1 and put(ps=2) == -1 and put(sizes=(1, 1, 1, 1, 0)) == -1 and put(sizes=(1, 0, 1, 1, 8)) == -1
    assert put(x=72) == -2 and put(st=(0, 0, 0, 68)) == -2 and put(codes=72) == -2 and put(meta=66) == -2
    assert put(sizes=(1, 1, 1, 1, (1 << 24) + 1)) == -3 and put(sizes=(1 << 12, 1 << 12, 1 << 12, 1, 8)) == -3

    def get(out=64, dt=0, st=(0, 0, 0, 64), sizes=(1, 1, 1, 1, 8)):
        return L.asr_cache4_get(None, p(), p(), p(out) if out else None, dt, *st, None, 0, None, *sizes)
    assert get(out=0) == -1 and get(dt=2) == -1 and get(st=(0, 0, 0, 66)) == -2 and get(out=68) == -2 and get(sizes=(0, 1, 1, 1, 8)) == -1

    def reorder(oc=64, om=64, beam=2, T=8):
        return L.asr_cache4_reorder(None, p(), p(), p(oc), p(om), p(), p(), 1, 1, beam, 1, T)
    assert reorder(beam=9) == -3 and reorder(beam=0) == -3 and reorder(om=128) == -1 and reorder(T=0) == -1 and reorder(oc=72, om=128) == -2

    def attn(q=64, dt=1, kc=64, sizes=(1, 4, 4, 1, 8), ws=0, wsb=0):
        return L.asr_cache4_attention(None, p(q) if q else None, dt, 0, 0, 0, p(kc), p(), p(), p(), p(), None, *sizes, None, 0, p(ws) if ws else None, wsb)
    assert attn(q=0) == -1 and attn(dt=2) == -1 and attn(sizes=(1, 4, 3, 1, 8)) == -1 and attn(sizes=(1, 4, 4, 0, 8)) == -1 and attn(kc=72) == -2
    assert attn(sizes=(1, 4, 4, 1, (1 << 24) + 1)) == -3 and attn(sizes=(1 << 12, 1 << 10, 1, 64, 8)) == -3
    need = L.asr_cache4_attention_workspace_bytes(1, 4, 4, 1, 100000)
    assert need > 0 and need % 4 == 0
    assert attn(sizes=(1, 4, 4, 1, 100000)) == -1 and b"workspace" in L.asr_last_error()
    assert attn(sizes=(1, 4, 4, 1, 100000), ws=64, wsb=need - 4) == -1
    assert L.asr_cache4_attention_workspace_bytes(1, 4, 4, 1, 8) == 0 and L.asr_cache4_attention_workspace_bytes(1, 4, 3, 1, 8) == 0


def test_library_refuses_sizes_that_no_launch_holds():
    """a launch holds fewer than 2^32 threads, 2^24 blocks of 256; products of sizes that pass 64 bits are too many as well, not few"""
    L = asr_amd.lib()
    p, top = ctypes.c_void_p(64), (1 << 31) - 1

    def put(*sizes):
        return L.asr_cache4_put(None, p, 1, 0, 0, 0, 64, p, p, None, 0, None, *sizes)

    def get(*sizes):
        return L.asr_cache4_get(None, p, p, p, 1, 0, 0, 0, 64, None, 0, None, *sizes)

    for call in (put, get):
        assert call(1, 1 << 10, 1 << 10, 1 << 13, 1 << 13) == -3 and b"too many rows" in L.asr_last_error()      # 2^20 rows of 32 or 64 blocks
        assert call(1, 1 << 15, 1 << 15, 1, 1) == -3 and call(top, top, top, 1, 8) == -3 and call(1 << 30, 1 << 30, 16, 1, 8) == -3      # (2^64 rows)

    def reorder(n_kv, B, h, T):
        return L.asr_cache4_reorder(None, p, p, p, p, p, p, n_kv, B, 2, h, T)
    assert reorder(1, 1 << 12, 1 << 10, 1 << 9) == -3 and reorder(top, top, top, 8) == -3 and reorder(1 << 30, 1 << 30, 16, 8) == -3

    def attn(N, h, h_kv, Lq):
        return L.asr_cache4_attention(None, p, 1, 0, 0, 0, p, p, p, p, p, None, N, h, h_kv, Lq, 8, None, 0, None, 0)
    assert attn(1 << 30, 1 << 30, 1, 16) == -3 and attn(top, top, top, top) == -3 and attn(1 << 24, 1, 1, 1) == -3
    size = L.asr_cache4_attention_workspace_bytes
    assert size(1, 1 << 30, 1, 1, 1 << 24) == 0 and size(1 << 30, 1 << 30, 1 << 30, 16, 1 << 24) == 0 and size(1, 4, 4, 1, (1 << 24) + 1) == 0      # (no call that is taken)


def test_header_revision():
    assert asr_amd.lib().asr_version() >= 103
    assert "103 = asr_cache4_* added" in open(_lib.HEADER).read()
