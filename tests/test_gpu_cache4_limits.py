"""The 4-bit K / V cache at the ends of what asr_hip.h states for it: keys, values whose sums come near f32's largest,
rows near bf16's largest, parents outside their utterance.  Expected values are 64-bit arithmetic on the stored codes, or equality."""
import math

import pytest
import torch

from asr_amd import ops
from test_gpu_cache4 import i32, rand_cache, reference, same, values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32_MAX = torch.finfo(torch.float32).max
BF16_MAX = torch.finfo(torch.bfloat16).max


def check_rows(q, kc, vc, rows, causal=False):
    """rows of the whole call against the 64-bit reference and its tolerance (test_gpu_cache4.reference)"""
    T = kc.codes.shape[2]
    got, lse = ops.cache4_attention(q, kc, vc, causal=causal, need_lse=True)
    for n in rows:
        one = lambda c: ops.Cache4(c.codes[n:n + 1].contiguous(), c.meta[n:n + 1].contiguous())  # noqa: E731
        want, wl, tol, lt = reference(q[n:n + 1], one(kc), one(vc), [T], causal, q.dtype)
        d = (got[n:n + 1].double().cpu() - want).abs()
        assert bool((d <= tol).all()), "row %d: %s" % (n, "not finite" if not bool(d.isfinite().all()) else "worst %.3g of its tolerance" % float((d / tol).max()))
        assert bool(((lse[n:n + 1].double().cpu() - wl).abs() <= lt).all())


# one wave's second tile scores 2^30 times its first's: the first kernel, the same with split keys, the dense kernel
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("N,h,h_kv,Lq,T", [(2, 2, 2, 1, 1300), (1, 4, 1, 1, 1300), (1, 1, 1, 1, 5000), (100, 4, 4, 12, 600)])
def test_large_values_behind_rising_scores(N, h, h_kv, Lq, T, causal, dtype):
    """values around 2^100 - their sum over a row below 2^119 - where the scores rise by 30 half way along the row"""
    g = torch.Generator().manual_seed(T + h)
    c = rand_cache(g, 2, N, h_kv, T)
    q = torch.zeros(N, h, Lq, 64, device=DEV, dtype=dtype)
    q[..., 0] = 1.0
    c.codes[0, ..., 0] = (c.codes[0, ..., 0] & 0xF0) | 1                     # the first channel's code is 1, the mid 0: score = scale
    c.meta[0, ..., 1] = 0
    rise = torch.where(torch.arange(T) < T // 2, 0.0, 30.0) + torch.rand(N, h_kv, T, generator=g)
    c.meta[0, ..., 0] = rise.to(DEV)
    big = torch.rand(2, N, h_kv, T, generator=g) + 0.5
    c.meta[1, ..., 0] = (big[0] * 2.0 ** 98).to(DEV)
    c.meta[1, ..., 1] = (torch.randn(N, h_kv, T, generator=g) * 2.0 ** 101).to(DEV)
    total = (c.meta[1].double()[..., 1].abs() + 8 * c.meta[1].double()[..., 0]).sum(-1).max()
    assert float(total) < 2.0 ** 119
    check_rows(q, c[0], c[1], sorted({0, N - 1}), causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,Lq,T", [(2, 2, 300), (100, 12, 150)])
def test_large_keys(N, Lq, T, dtype):
    """keys up to 2^94 beside queries small enough for scores of order one"""
    g = torch.Generator().manual_seed(T)
    c = rand_cache(g, 2, N, 4, T)
    c.meta[0, ..., 0] = (torch.rand(N, 4, T, generator=g) * 2.0 ** 88).to(DEV)
    c.meta[0, ..., 1] = (torch.randn(N, 4, T, generator=g).clamp(-3, 3) * 2.0 ** 91).to(DEV)
    assert float((c.meta[0].double()[..., 1].abs() + 8 * c.meta[0].double()[..., 0]).max()) < 2.0 ** 94
    q = (torch.randn(N, 4, Lq, 64, generator=g) * 2.0 ** -93).to(dtype).to(DEV)
    check_rows(q, c[0], c[1], sorted({0, N - 1}))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_near_the_largest_value(dtype):
    """a row is finite (code, scale and middle) or NaN, never a middle of infinity: constants and narrow rows on both sides of bf16's largest"""
    fine = [torch.full((64,), BF16_MAX), torch.full((64,), -BF16_MAX), torch.linspace(0.0, BF16_MAX, 64), torch.linspace(-BF16_MAX, 0.0, 64),
            torch.linspace(3.0e38, 3.35e38, 64)]
    over = []
    if dtype == torch.float32:      # (bf16 has no finite value above its largest; its half step ends at 3.396e38)
        over = [torch.full((64,), F32_MAX), torch.full((64,), -F32_MAX), torch.linspace(3.397e38, 3.402e38, 64), -torch.linspace(3.397e38, 3.402e38, 64)]
    x = torch.stack(fine + over).to(dtype).to(DEV)[None, None]
    c = ops.Cache4.empty(None, 1, 1, x.shape[2], DEV)
    ops.cache4_put(c, x)
    n = len(fine)
    assert bool(c.meta[0, 0, :n].isfinite().all())
    assert bool(c.meta[0, 0, n:].isnan().all()) and int(c.codes[0, 0, n:].max() if over else 0) == 0
    got = ops.cache4_get(c, dtype=torch.float32)
    assert same(got, values(c)) and bool(got[0, 0, n:].isnan().all())
    assert torch.equal(got[0, 0, :2], torch.tensor([[BF16_MAX], [-BF16_MAX]], device=DEV).expand(2, 64))
    # within the middle's half step (2^-9 of it) and half a code's step (with the middle's own rounding in it) of the value, both bf16
    d = (got[0, 0, 2:n].double() - x[0, 0, 2:n].double()).abs()
    scale, mid = c.meta[0, 0, 2:n].double().unbind(-1)
    assert bool((d <= (scale / 2 + mid.abs() * 2.0 ** -8)[:, None]).all())


@pytest.mark.parametrize("in_place", [True, False])
def test_parents_outside_their_utterance(in_place):
    """cut to the nearest row of the utterance, however far outside: not modulo 2^32"""
    beam, B, T = 8, 3, 20
    g = torch.Generator().manual_seed(1)
    c = rand_cache(g, 2, B * beam, 2, T)
    parent, rows = [], []
    for b in range(B):
        first = b * beam
        parent += [first - 1, first + beam, first + 2 ** 32, first - 2 ** 32 + 3, first + 2 ** 31, first - 2 ** 40, -2 ** 63, 2 ** 63 - 1]
        rows += [first, first + beam - 1, first + beam - 1, first, first + beam - 1, first, first, first + beam - 1]
    before = ops.Cache4(c.codes.clone(), c.meta.clone())
    out = None if in_place else rand_cache(g, 2, B * beam, 2, T)
    ops.cache4_reorder(c, torch.tensor(parent, dtype=torch.int64, device=DEV), i32(T - 1, -1), beam, out=out)
    got = c if in_place else out
    assert torch.equal(got.codes, before.codes[:, rows]) and torch.equal(got.meta, before.meta[:, rows])


def test_finite_sums_stay_finite_with_many_slots():
    """20 000 slots whose values add up to just under 2^119, equal scores: the mean comes out"""
    T = 20000
    c = ops.Cache4.empty(2, 1, 1, T, DEV)
    v = 2.0 ** 104
    c.meta[1, ..., 1] = v
    got, _ = ops.cache4_attention(torch.zeros(1, 1, 1, 64, device=DEV), c[0], c[1])
    assert T * v < 2.0 ** 119 and math.isfinite(float(got[0, 0, 0]))
    assert bool(((got / v - 1).abs() <= 40 * 2.0 ** -24).all())


@pytest.mark.parametrize("beam", [2, 3, 4, 8])
@pytest.mark.parametrize("t", [0, 1, 2, 30, 31, 32, 63, 64])
def test_reorder_of_few_positions(beam, t):
    """fewer live lanes in a wave than parents to read: the last wave of the codes (2 (t + 1) pieces) and of the meta words (t + 1)"""
    g = torch.Generator().manual_seed(t)
    B, T = 2, 65
    c = rand_cache(g, 2, B * beam, 2, T)
    rows = [b * beam + (r + 1 + b) % beam for b in range(B) for r in range(beam)]
    before, parent = ops.Cache4(c.codes.clone(), c.meta.clone()), torch.tensor(rows, device=DEV)
    other = rand_cache(g, 2, B * beam, 2, T)
    was = ops.Cache4(other.codes.clone(), other.meta.clone())
    ops.cache4_reorder(c, parent, i32(t, -1), beam, out=other)
    ops.cache4_reorder(c, parent, i32(t, -1), beam)
    n = t + 1
    for got, old in ((other, was), (c, before)):
        for a, src, o in ((got.codes, before.codes, old.codes), (got.meta, before.meta, old.meta)):
            assert torch.equal(a[:, :, :, :n], src[:, rows, :, :n]) and torch.equal(a[:, :, :, n:], o[:, :, :, n:])
