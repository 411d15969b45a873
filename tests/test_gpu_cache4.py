"""The 4-bit K / V cache (csrc/cache4.hip) against its definition in 64 bits (asr_hip.h: asr_cache4_put).

Quantising and reading back are compared for equality: scale, mid and every code are defined exactly (the code is the nearest integer to
(x - mid) / scale, decided without rounding), and a value is one f32 rounding of mid + scale * code.
Attention's tolerance is computed beside the reference, from what the kernel may round (reference()): the digits of the query and of the
weights (half a unit each), f32 arithmetic (2^-24 an operation), the output's type (half a step)."""
import math

import pytest
import torch

from asr_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOG2E = 1.4426950408889634
FIFTEENTH = torch.tensor(1.0) / torch.tensor(15.0)                       # in f32, as the format has it
UNIT = {torch.bfloat16: 127 * 256, torch.float32: 127 * 65536}      # what the largest element becomes in digits of base 256


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def quantise(x):
    """[..., 64] -> codes int64 [..., 64], scale f64, mid f64 (f32-exact), in 64 bits"""
    x = x.double()
    lo, hi = x.amin(-1), x.amax(-1)
    span = (hi.float() - lo.float())
    scale = torch.where(span < 2.0 ** -100, torch.zeros_like(span), span * FIFTEENTH.to(span.device)).bfloat16().double()
    mid = (lo.float() + 8.0 * scale.float()).bfloat16().double()
    bad = ~(span < math.inf)
    q = (x - mid[..., None]) / scale[..., None]
    q = torch.where((scale[..., None] == 0) | bad[..., None], torch.zeros_like(q), q)
    f = torch.floor(q)
    # the rounding of the difference and of the quotient can only matter next to a border: there x is compared with the border itself, which
    # f64 holds exactly (mid has 8 bits, (f + 1/2) scale 13; x - mid may need more than 53)
    up = torch.sign(x - (mid[..., None] + (f + 0.5) * scale[..., None]))
    near = (q - f - 0.5).abs() < 1e-9
    k = torch.where(near, torch.where(up == 0, f + (f.remainder(2) == 1).double(), f + (up > 0).double()), torch.round(q))
    nan = torch.full_like(scale, math.nan)
    return k.clamp(-8, 7).long(), torch.where(bad, nan, scale), torch.where(bad, nan, mid)


def pack(codes, scale, mid):
    c = (codes & 15).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.stack([scale, mid], -1).bfloat16()


def unpack(codes):
    c = codes.to(torch.int64)
    return ((torch.stack([c & 15, c >> 4], -1).flatten(-2)) ^ 8) - 8


def values(cache):
    """f64 [..., 64] as the f32 rounding of mid + scale * code"""
    return (cache.meta[..., 1:].double() + cache.meta[..., :1].double() * unpack(cache.codes).double()).float()


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0)) and torch.equal(a.isnan(), b.isnan())


def check_put(cache, before, x, pos, n_new):
    """every slot of the cache: what put has to leave there"""
    n_kv, N, h, Tmax = cache.shape
    want_c, want_m = before.codes.clone().view(n_kv, N, h, Tmax, 32), before.meta.clone().view(n_kv, N, h, Tmax, 2)
    xc, xm = pack(*quantise(x))
    xc, xm = xc.view(n_kv, N, h, -1, 32), xm.view(n_kv, N, h, -1, 2)
    for n in range(N):
        for i in range(n_new[n]):
            if 0 <= pos[n] + i < Tmax:
                want_c[:, n, :, pos[n] + i] = xc[:, n, :, i]
                want_m[:, n, :, pos[n] + i] = xm[:, n, :, i]
    assert same(cache.meta.view_as(want_m), want_m)
    assert torch.equal(cache.codes.view_as(want_c), want_c)


def rand_cache(g, n_kv, N, h, T):
    c = ops.Cache4.empty(n_kv, N, h, T, DEV)
    c.codes.copy_(torch.randint(0, 256, c.codes.shape, generator=g, dtype=torch.uint8))
    m = torch.rand(c.meta.shape, generator=g) * 0.4 + 0.01
    m[..., 1] = torch.randn(m.shape[:-1], generator=g)
    c.meta.copy_(m)
    return c


def clone(c):
    return ops.Cache4(c.codes.clone(), c.meta.clone())


# ---- quantising and reading back -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_kv,N,h,L,T", [(1, 1, 1, 1, 1), (2, 3, 4, 1, 7), (1, 2, 3, 5, 9), (2, 5, 1, 31, 40), (1, 3, 2, 33, 33), (2, 2, 2, 127, 130), (1, 2, 1, 129, 300),
                                          (12, 32, 4, 1, 101)])
def test_put_and_get(n_kv, N, h, L, T, dtype):
    g = torch.Generator().manual_seed(L * 100 + N)
    x = (torch.randn(n_kv, N, h, L, 64, generator=g) * torch.rand(n_kv, N, h, L, 1, generator=g) * 4 + torch.randn(n_kv, N, h, L, 1, generator=g)).to(dtype).to(DEV)
    c = rand_cache(g, n_kv, N, h, T)
    before = clone(c)
    pos = [(7 * n + 3) % max(1, T - L + 1) for n in range(N)]
    n_new = [L - (n * 5) % (L + 1) for n in range(N)]                       # 0 .. L tokens
    ops.cache4_put(c, x, pos=i32(*pos), n_new=i32(*n_new))
    check_put(c, before, x, pos, n_new)
    for out in (torch.float32, torch.bfloat16):
        got = ops.cache4_get(c, L=L, pos=i32(*pos), n_tok=i32(*n_new), dtype=out)
        full = ops.cache4_get(c, dtype=out)
        assert torch.equal(full, values(c).to(out))
        for n in range(N):
            k = n_new[n]
            assert torch.equal(got[:, n, :, :k], full[:, n, :, pos[n]:pos[n] + k]) and int((got[:, n, :, k:] != 0).sum()) == 0


def test_put_common_position_and_slots_outside():
    """one position for all rows, in device memory; slots in front of and behind the cache are not written and read back as zeros"""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 3, 2, 6, 64, generator=g).to(DEV)
    for p in (-9, -3, 0, 4, 7, 8, 2 ** 31 - 3):
        c = rand_cache(g, 2, 3, 2, 8)
        before = clone(c)
        state = i32(p, -1)
        ops.cache4_put(c, x, pos=state[:1])
        check_put(c, before, x, [p] * 3, [6] * 3)
        got, full = ops.cache4_get(c, L=6, pos=state[:1], dtype=torch.float32), values(c)
        for i in range(6):
            want = full[:, :, :, p + i] if 0 <= p + i < 8 else torch.zeros_like(full[:, :, :, 0])
            assert torch.equal(got[:, :, :, i], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_borders_and_extremes(dtype):
    """rows on exact ties and next to them, constants, tiny and huge spans, a level far from the spread, NaN and infinities"""
    rows = []
    for sc in (1.0, 0.25, 2.0 ** -80, 2.0 ** 60, 1.5, 0.0078125 * 129):
        base = torch.arange(64).double() % 31 / 2.0 - 7.5                   # -7.5 .. 7.5 in halves of a step: every border of a unit scale
        rows += [base * sc, (base + 1.0) * sc, base * sc * (1 + 2.0 ** -20), base * sc * (1 - 2.0 ** -20), (base * sc).abs()]
    tie = torch.arange(64).double() % 15 - 7.0
    for e in (0.0, 1e-9, -1e-9, 2.0 ** -30):                                # a middle of half a step, and values that only f64 tells from a border
        rows.append(torch.where(torch.arange(64) % 3 == 0, torch.full((64,), e, dtype=torch.float64), tie + 0.5))
    rows += [torch.zeros(64), torch.full((64,), 3.14159), torch.full((64,), -1e-38), torch.full((64,), 1e-45), torch.linspace(0, 1e-40, 64), torch.linspace(1e30, 1.1e30, 64),
             torch.linspace(-1.6e38, 1.6e38, 64), torch.linspace(-3e38, 3e38, 64), torch.linspace(1000.0, 1000.5, 64), torch.linspace(-1e-30, 1.0, 64)]
    for bad in (math.nan, math.inf, -math.inf):
        for at in (0, 7, 8, 63):
            r = torch.linspace(-1, 1, 64)
            r[at] = bad
            rows.append(r)
    x = torch.stack([r.double() for r in rows]).to(dtype).to(DEV)[None, None]    # [1, 1, R, 64]: one head, R tokens
    R = x.shape[2]
    c = ops.Cache4.empty(None, 1, 1, R, DEV)
    before = clone(c)
    ops.cache4_put(c, x)
    check_put(c, before, x, [0], [R])
    got = ops.cache4_get(c, dtype=torch.float32)
    assert same(got, values(c))
    fine = torch.isfinite(x).all(-1) & torch.isfinite(x.float().amax(-1) - x.float().amin(-1))
    assert bool(got.isnan().all(-1)[~fine].all()) and not bool(got[fine].isnan().any())


def test_many_values_next_to_borders():
    """a million f32 values within a few ulp of a code's border: every decision is the exact quotient's"""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(2, 8, 4, 256, 64, generator=g)
    _, scale, mid = quantise(x)
    k = torch.randint(-7, 7, x.shape, generator=g).double() + 0.5
    near = (mid[..., None] + k * scale[..., None]).float()
    ulp = torch.randint(-2, 3, x.shape, generator=g).int()
    near = (near.view(torch.int32) + ulp).view(torch.float32)
    keep = torch.arange(64) < 2                                              # (the row's extremes stay: they fix scale and mid)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    x = torch.where(keep, torch.where(torch.arange(64) == 0, lo, hi), torch.minimum(torch.maximum(near, lo), hi)).to(DEV)
    c = ops.Cache4.empty(2, 8, 4, 256, DEV)
    before = clone(c)
    ops.cache4_put(c, x)
    check_put(c, before, x, [0] * 8, [256] * 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_put_strided(dtype):
    """token-major keys as a plain projection leaves them, a slice of a wider buffer, one row for all (stride 0)"""
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(3, 10, 3 * 4 * 64, generator=g).to(dtype).to(DEV)     # [N, L, q | k | v]
    x = wide[:, :, 256:512].view(3, 10, 4, 64).permute(0, 2, 1, 3)           # [N, h, L, 64]
    c = ops.Cache4.empty(None, 3, 4, 12, DEV)
    before = clone(c)
    ops.cache4_put(c, x, pos=i32(2))
    check_put(c, before, x, [2] * 3, [10] * 3)
    one = x[:1].expand(3, 4, 10, 64)
    before = clone(c)
    ops.cache4_put(c, one)
    check_put(c, before, one, [0] * 3, [10] * 3)
    with pytest.raises(RuntimeError, match="16 bytes"):
        ops.cache4_put(c, wide[:, :, 257:513].unflatten(2, (4, 64)).permute(0, 2, 1, 3))


def test_empty_calls():
    c = ops.Cache4.empty(2, 3, 4, 8, DEV)
    ops.cache4_put(c, torch.zeros(2, 3, 4, 0, 64, device=DEV))
    assert ops.cache4_get(c, L=0).shape == (2, 3, 4, 0, 64)
    ctx, lse = ops.cache4_attention(torch.zeros(3, 4, 0, 64, device=DEV), c[0], c[1], need_lse=True)
    assert ctx.shape == (3, 0, 256) and lse.shape == (3, 4, 0)
    bare = ops.Cache4.empty(2, 3, 4, 0, DEV)                                 # no slots
    ops.cache4_put(bare, torch.ones(2, 3, 4, 2, 64, device=DEV))
    assert int(ops.cache4_get(bare, L=2).abs().sum()) == 0
    ctx, lse = ops.cache4_attention(torch.ones(3, 4, 2, 64, device=DEV), bare[0], bare[1], need_lse=True)
    assert int(ctx.abs().sum()) == 0 and bool(torch.isinf(lse).all())
    none = ops.Cache4.empty(2, 0, 4, 8, DEV)
    assert ops.cache4_attention(torch.zeros(0, 4, 1, 64, device=DEV), none[0], none[1])[0].shape == (0, 1, 256)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(dtype):
    """a quarter of a million rows, spans over twelve octaves: scale and mid of every row (one f32 ulp in the span's multiple moves a bf16 scale in
    about one row of 2^16)"""
    g = torch.Generator().manual_seed(41)
    x = torch.randn(4, 16, 4, 1024, 64, generator=g) * torch.exp2(12 * torch.rand(4, 16, 4, 1024, 1, generator=g) - 6)
    x = (x + torch.randn(4, 16, 4, 1024, 1, generator=g)).to(dtype).to(DEV)
    c = ops.Cache4.empty(4, 16, 4, 1024, DEV)
    ops.cache4_put(c, x)
    codes, meta = pack(*quantise(x))
    assert torch.equal(c.meta, meta) and torch.equal(c.codes, codes)


# ---- attention -------------------------------------------------------------------------------------------------------------------------
def reference(q, kc, vc, k_len, causal, dtype):
    """-> ctx f64 [N, Lq, h*64], lse f64 [N, h, Lq], tolerances of both"""
    N, h, Lq, _ = q.shape
    h_kv, T = kc.codes.shape[1], kc.codes.shape[2]
    q = q.double().cpu()
    u, eps = UNIT[dtype], 2.0 ** -24
    ctx, tol = torch.zeros(N, Lq, h, 64, dtype=torch.float64), torch.full((N, Lq, h, 64), 1e-30, dtype=torch.float64)
    lse, ltol = torch.full((N, h, Lq), -math.inf, dtype=torch.float64), torch.zeros(N, h, Lq, dtype=torch.float64)
    for n in range(N):
        ln = max(0, min(T, int(k_len[n])))
        kk, vv = (unpack(c.codes[n, :, :ln]).double().cpu() for c in (kc, vc))
        km, vm = (c.meta[n, :, :ln].double().cpu() for c in (kc, vc))
        for head in range(h):
            g = head // (h // h_kv)
            ks, kmid, vs, vmid = km[g, :, 0], km[g, :, 1], vm[g, :, 0], vm[g, :, 1]
            for i in range(Lq):
                m = ln - Lq + i + 1 if causal else ln
                if m <= 0:
                    continue
                qq = q[n, head, i]
                a, b = (kk[g, :m] @ qq) * ks[:m], kmid[:m] * qq.sum()
                s = a + b
                top = s.max()
                w = torch.exp2(s - top)
                l = w.sum()
                p = w / l
                code, mid = vv[g, :m] * vs[:m, None], vmid[:m, None]
                o = (p[:, None] * (code + mid)).sum(0)
                ds = qq.abs().max() / (2 * u) * kk[g, :m].abs().sum(-1) * ks[:m] + eps * (6 * (a.abs() + b.abs()) + 8 * qq.abs().sum() * kmid[:m].abs() + 2 * (s - top).abs() + 64)
                dw = math.log(2.0) * ds.max()                                           # relative error of a weight, hence twice of a quotient of sums
                tiles = (m + 63) // 64
                part = torch.nn.functional.pad(p * vs[:m], (0, tiles * 64 - m)).view(tiles, 64).amax(-1)
                dig = (part.repeat_interleave(64)[:m, None] / (2 * u) * 1.01 * vv[g, :m].abs()).sum(0)      # half a unit of the tile's largest weight
                size = (p[:, None] * (code.abs() + mid.abs())).sum(0)
                out = torch.finfo(dtype).eps / 2
                t = 2.1 * dw * size + dig + (tiles + 24) * eps * size
                ctx[n, i, head], tol[n, i, head] = o, t + out * (o.abs() + t) + 1e-30
                lse[n, head, i] = top + torch.log2(l)
                ltol[n, head, i] = 1.1 * ds.max() + (tiles + 24) * eps * 1.5 + 2 * eps * lse[n, head, i].abs()
    return ctx.view(N, Lq, h * 64), lse, tol.view(N, Lq, h * 64), ltol


def check_attention(q, kc, vc, k_len, causal=False, lens=None):
    N, T = q.shape[0], kc.codes.shape[2]
    lens = [T] * N if lens is None else lens
    got, lse = ops.cache4_attention(q, kc, vc, k_len=k_len, causal=causal, need_lse=True)
    want, wl, tol, lt = reference(q, kc, vc, lens, causal, q.dtype)
    assert got.dtype == q.dtype and not bool(got.isnan().any())
    d = (got.double().cpu() - want).abs()
    assert bool((d <= tol).all()), "worst %.3g of its tolerance" % float((d / tol).max())
    empty = torch.isinf(wl)
    lse = lse.double().cpu()
    assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all())
    assert bool(((lse - wl).abs()[~empty] <= lt[~empty]).all())
    return got


def make(g, N, h, h_kv, Lq, T, dtype):
    q = (torch.randn(N, h, Lq, 64, generator=g) * LOG2E / 8).to(dtype).to(DEV)
    c = ops.Cache4.empty(2, N, h_kv, T, DEV)
    level = torch.randn(2, 1, h_kv, 1, 64, generator=g) * (1 + 3 * (torch.rand(64, generator=g) > 0.95))
    ops.cache4_put(c, (torch.randn(2, N, h_kv, T, 64, generator=g) + level).to(DEV))
    return q, c[0], c[1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,h,h_kv,Lq,T", [(1, 1, 1, 1, 1), (2, 4, 4, 1, 63), (3, 4, 4, 1, 64), (2, 4, 2, 1, 65), (3, 2, 1, 3, 130), (2, 4, 4, 5, 200), (2, 8, 2, 2, 257), (2, 3, 3, 7, 101),
                                           (1, 4, 1, 2, 100), (2, 6, 3, 3, 90), (1, 2, 2, 9, 70), (1, 8, 1, 4, 1030), (40, 4, 4, 1, 33)])
def test_attention(N, h, h_kv, Lq, T, dtype):
    g = torch.Generator().manual_seed(N * 1000 + T)
    q, kc, vc = make(g, N, h, h_kv, Lq, T, dtype)
    lens = [max(0, T - (n * 37) % (T + 1)) for n in range(N)]
    check_attention(q, kc, vc, i32(*lens), lens=lens)
    check_attention(q, kc, vc, None)
    check_attention(q, kc, vc, i32(*lens), causal=True, lens=lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_lengths(dtype):
    """every length around the tile's, none, one, and lengths outside [0, T]"""
    g = torch.Generator().manual_seed(3)
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 140, 141, 1000, -5]
    q, kc, vc = make(g, len(lens), 2, 2, 2, 140, dtype)
    for causal in (False, True):
        got = check_attention(q, kc, vc, i32(*lens), causal=causal, lens=lens)
        assert int((got[0] != 0).sum()) == 0 and int((got[-1] != 0).sum()) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,h,h_kv,Lq,T", [(1, 4, 4, 1, 5000), (2, 8, 2, 1, 3333), (1, 2, 2, 11, 2500), (1, 1, 1, 1, 20011)])
def test_attention_split(N, h, h_kv, Lq, T, dtype):
    """few rows of many keys: the keys are split over workgroups and joined; short rows leave splits without a tile"""
    g = torch.Generator().manual_seed(T)
    q, kc, vc = make(g, N, h, h_kv, Lq, T, dtype)
    for lens in ([T - 7 * n for n in range(N)], [1 + n for n in range(N)], [70] * N, [0] * N):
        check_attention(q, kc, vc, i32(*lens), lens=lens)
    check_attention(q, kc, vc, None, causal=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [40, 150, 4100])
def test_masked_slots_may_hold_anything(T, dtype):
    """NaN and infinities behind the last token, and - causal - in tokens that some queries do not see"""
    g = torch.Generator().manual_seed(T + 1)
    q, kc, vc = make(g, 2, 2, 2, 3, T, dtype)
    lens = [T - 20, 17]
    base = check_attention(q, kc, vc, i32(*lens), lens=lens)
    for c in (kc, vc):
        for n, ln in enumerate(lens):
            c.meta[n, :, ln:] = torch.tensor([math.nan, math.inf], dtype=torch.bfloat16, device=DEV)
            c.codes[n, :, ln:] = 0xA5
    assert torch.equal(base, ops.cache4_attention(q, kc, vc, k_len=i32(*lens))[0])
    want = ops.cache4_attention(q, kc, vc, k_len=i32(*lens), causal=True)[0]
    for c in (kc, vc):
        for n, ln in enumerate(lens):
            c.meta[n, :, ln - 1] = math.nan                                   # the last token: only the last query sees it
    got = ops.cache4_attention(q, kc, vc, k_len=i32(*lens), causal=True)[0]
    assert torch.equal(got[:, :2], want[:, :2]) and bool(got[:, 2].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_peaks_and_scales(dtype):
    """scores that rise by far more than the reference's slack from tile to tile (and fall again), a value row a thousand times the others, a
    zero query, zero values: the tolerance follows each"""
    g = torch.Generator().manual_seed(9)
    T = 400
    q, kc, vc = make(g, 1, 4, 4, 1, T, dtype)
    q[0, 1] = 0
    ramp = torch.linspace(-1, 1, T)
    x = torch.randn(2, 1, 4, T, 64, generator=g)
    x[0, 0, 0] += (ramp * 40)[:, None] * q[0, 0, 0].float().cpu().sign()       # head 0: rising scores
    x[0, 0, 2] -= (ramp * 40)[:, None] * q[0, 2, 0].float().cpu().sign()       # head 2: falling
    x[1, 0, :, 200] *= 1000
    x[1, 0, 3, :100] = 0
    c = ops.Cache4.empty(2, 1, 4, T, DEV)
    ops.cache4_put(c, x.to(DEV))
    check_attention(q, c[0], c[1], None)


def test_flat_tail_beside_a_peak():
    """one token of weight 1 and 20 000 of 1e-5 each: the tail is as heavy as the peak and must not fall below the digits"""
    T = 20001
    q = torch.zeros(1, 1, 1, 64, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    x = torch.zeros(2, 1, 1, T, 64)
    x[0, 0, 0, :, 0], x[0, 0, 0, 777, 0] = 0.0, 14.0
    x[0, 0, 0, :, 1] = torch.linspace(-1, 1, T)
    x[1, 0, 0, :, :] = torch.linspace(0.5, 1.5, 64)
    x[1, 0, 0, 777] = torch.linspace(-1.5, -0.5, 64)
    c = ops.Cache4.empty(2, 1, 1, T, DEV)
    ops.cache4_put(c, x.to(DEV))
    check_attention(q, c[0], c[1], None)


def test_attention_query_strides():
    """token-major queries (a plain projection's output) and a slice of a wider buffer"""
    g = torch.Generator().manual_seed(4)
    q, kc, vc = make(g, 3, 4, 4, 5, 77, torch.bfloat16)
    want = ops.cache4_attention(q, kc, vc)[0]
    wide = torch.zeros(3, 5, 3, 4, 64, dtype=torch.bfloat16, device=DEV)
    wide[:, :, 1] = q.transpose(1, 2)
    assert torch.equal(want, ops.cache4_attention(wide[:, :, 1].transpose(1, 2), kc, vc)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,h,h_kv,Lq,T", [(64, 2, 2, 33, 130), (140, 8, 1, 4, 65), (12, 8, 8, 33, 1300), (400, 4, 1, 3, 70), (2, 2, 1, 50, 20000),
                                           (600, 2, 2, 9, 40)])
def test_attention_many_queries(N, h, h_kv, Lq, T, dtype):
    """enough queries and rows for the dense kernel (16 queries a block, a lane a query: more than 8 a key head, and more than 1024 groups of four
    or 12 288 tiles of them; the longest with split keys): the first, the last and two rows between against the reference"""
    g = torch.Generator().manual_seed(N + T)
    q, kc, vc = make(g, N, h, h_kv, Lq, T, dtype)
    lens = [max(0, T - (n * 29) % (T + 1)) if n else T for n in range(N)]
    for causal in (False, True):
        got, lse = ops.cache4_attention(q, kc, vc, k_len=i32(*lens), causal=causal, need_lse=True)
        for n in sorted({0, 1, N // 2, N - 1}):
            one = lambda c: ops.Cache4(c.codes[n:n + 1].contiguous(), c.meta[n:n + 1].contiguous())  # noqa: E731
            want, wl, tol, lt = reference(q[n:n + 1], one(kc), one(vc), [lens[n]], causal, dtype)
            d = (got[n:n + 1].double().cpu() - want).abs()
            assert bool((d <= tol).all()), "row %d: worst %.3g of its tolerance" % (n, float((d / tol).max()))
            seen, l = ~torch.isinf(wl), lse[n:n + 1].double().cpu()
            assert torch.equal(torch.isinf(l), ~seen) and bool(((l - wl).abs()[seen] <= lt[seen]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_slots_many_queries(dtype):
    """the dense kernel: anything behind the last token; a NaN token that only the last queries see"""
    g = torch.Generator().manual_seed(77)
    N, T, Lq = 110, 300, 20
    q, kc, vc = make(g, N, 2, 2, Lq, T, dtype)
    lens = [T - 20 - n % 64 for n in range(N)]
    want = [ops.cache4_attention(q, kc, vc, k_len=i32(*lens), causal=causal)[0] for causal in (False, True)]
    for c in (kc, vc):
        for n, ln in enumerate(lens):
            c.meta[n, :, ln:] = torch.tensor([math.nan, math.inf], dtype=torch.bfloat16, device=DEV)
            c.codes[n, :, ln:] = 0x5A
    for causal in (False, True):
        assert torch.equal(ops.cache4_attention(q, kc, vc, k_len=i32(*lens), causal=causal)[0], want[causal])
    for c in (kc, vc):
        for n, ln in enumerate(lens):
            c.meta[n, :, ln - 3] = math.nan
    got = ops.cache4_attention(q, kc, vc, k_len=i32(*lens), causal=True)[0]
    assert torch.equal(got[:, :Lq - 3], want[1][:, :Lq - 3]) and bool(got[:, Lq - 3:].isnan().all())


def test_repeatable():
    g = torch.Generator().manual_seed(6)
    q, kc, vc = make(g, 2, 4, 2, 5, 6000, torch.bfloat16)
    a = ops.cache4_attention(q, kc, vc, need_lse=True)
    for _ in range(5):
        b = ops.cache4_attention(q, kc, vc, need_lse=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- re-gathering ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n_kv,B,beam,h,T,t", [(1, 1, 1, 1, 1, 0), (2, 3, 5, 4, 101, 50), (1, 2, 8, 2, 33, 32), (4, 1, 3, 1, 90, 0), (2, 2, 2, 3, 200, 199), (1, 2, 4, 1, 10, 30)])
def test_reorder(n_kv, B, beam, h, T, t):
    g = torch.Generator().manual_seed(T + beam)
    c = rand_cache(g, n_kv, B * beam, h, T)
    rows = [b * beam + int(torch.randint(0, beam, (1,), generator=g)) for b in range(B) for _ in range(beam)]
    parent = torch.tensor(rows, dtype=torch.int64, device=DEV)
    before, n = clone(c), min(t + 1, T)
    other = rand_cache(g, n_kv, B * beam, h, T)
    was = clone(other)
    ops.cache4_reorder(c, parent, i32(t, -1), beam, out=other)
    assert torch.equal(c.codes, before.codes) and torch.equal(c.meta, before.meta)
    for got, src, old in ((other.codes, before.codes, was.codes), (other.meta, before.meta, was.meta)):
        assert torch.equal(got[:, :, :, :n], src[:, parent, :, :n]) and torch.equal(got[:, :, :, n:], old[:, :, :, n:])
    ops.cache4_reorder(c, parent, i32(t, -1), beam)
    for got, src in ((c.codes, before.codes), (c.meta, before.meta)):
        assert torch.equal(got[:, :, :, :n], src[:, parent, :, :n]) and torch.equal(got[:, :, :, n:], src[:, :, :, n:])


# ---- together ----------------------------------------------------------------------------------------------------------------------------
def search_step(cache, kv, q, state, k_len, parent, beam):
    """a token of a beam search: append, attend, re-gather"""
    ops.cache4_put(cache, kv, pos=state[:1])
    ctx, _ = ops.cache4_attention(q, cache[0], cache[1], k_len=k_len)
    ops.cache4_reorder(cache, parent, state, beam)
    return ctx


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_attend_reorder(dtype):
    """twelve steps of a search on a cache kept by the operators against one kept in the test"""
    g = torch.Generator().manual_seed(21)
    B, beam, h, T = 3, 4, 2, 12
    N = B * beam
    c = ops.Cache4.empty(2, N, h, T, DEV)
    mine = clone(c)
    for t in range(T):
        kv = torch.randn(2, N, h, 1, 64, generator=g).to(dtype).to(DEV)
        q = (torch.randn(N, h, 1, 64, generator=g) * LOG2E / 8).to(dtype).to(DEV)
        parent = torch.tensor([b * beam + int(torch.randint(0, beam, (1,), generator=g)) for b in range(B) for _ in range(beam)], device=DEV)
        got = search_step(c, kv, q, i32(t, -1), i32(*[t + 1] * N), parent, beam)
        codes, meta = pack(*quantise(kv))
        mine.codes[:, :, :, t:t + 1], mine.meta[:, :, :, t:t + 1] = codes, meta
        want, _, tol, _ = reference(q, mine[0], mine[1], [t + 1] * N, False, dtype)
        assert bool(((got.double().cpu() - want).abs() <= tol).all())
        mine = ops.Cache4(mine.codes[:, parent].contiguous(), mine.meta[:, parent].contiguous())
        assert torch.equal(c.codes, mine.codes) and torch.equal(c.meta, mine.meta)


def test_captured_steps_replayed():
    """two graphs of a search step (one with split keys) replayed in turn, with eager work between, against eager calls on copies"""
    g = torch.Generator().manual_seed(31)
    setups = []
    for B, beam, h, T in ((2, 3, 4, 24), (1, 2, 1, 4000)):
        N = B * beam
        cache = rand_cache(g, 2, N, h, T)
        kv, q = torch.zeros(2, N, h, 1, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(N, h, 1, 64, device=DEV, dtype=torch.bfloat16)
        state, k_len, parent = i32(0, -1), torch.ones(N, dtype=torch.int32, device=DEV), torch.arange(N, device=DEV)
        search_step(clone(cache), kv, q, state, k_len, parent, beam)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ctx = search_step(cache, kv, q, state, k_len, parent, beam)
        setups.append((B, beam, h, T, N, cache, clone(cache), kv, q, state, k_len, parent, graph, ctx))
    for t in range(6):
        for B, beam, h, T, N, cache, mine, kv, q, state, k_len, parent, graph, ctx in setups:
            at = t if T < 100 else 600 * t
            kv.copy_(torch.randn(kv.shape, generator=g))
            q.copy_(torch.randn(q.shape, generator=g) * LOG2E / 8)
            state[0] = at
            k_len.fill_(at + 1)
            parent.copy_(torch.tensor([b * beam + int(torch.randint(0, beam, (1,), generator=g)) for b in range(B) for _ in range(beam)]))
            graph.replay()
            want = search_step(mine, kv, q, state, k_len, parent, beam)
            torch.cuda.synchronize()
            assert torch.equal(ctx, want) and torch.equal(cache.codes, mine.codes) and torch.equal(cache.meta, mine.meta)


def test_other_stream():
    g = torch.Generator().manual_seed(8)
    q, kc, vc = make(g, 2, 4, 4, 2, 3000, torch.bfloat16)
    want = ops.cache4_attention(q, kc, vc)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.cache4_attention(q, kc, vc)[0] for _ in range(4)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(want, t) for t in got)


def test_offsets_past_32_bits():
    """a cache of 2.9 GB of codes: the last row's last slots"""
    T = (1 << 24) - 5
    c = ops.Cache4.empty(None, 6, 1, T, DEV)
    g = torch.Generator().manual_seed(12)
    x = torch.randn(6, 1, 70, 64, generator=g).to(DEV)
    ops.cache4_put(c, x, pos=i32(T - 70))
    codes, meta = pack(*quantise(x))
    assert torch.equal(c.codes[:, :, T - 70:], codes) and torch.equal(c.meta[:, :, T - 70:], meta) and int(c.codes[:, :, :T - 70].max()) == 0
    assert torch.equal(ops.cache4_get(c, L=70, pos=i32(T - 70), dtype=torch.float32), values(ops.Cache4(c.codes[:, :, T - 70:].contiguous(), c.meta[:, :, T - 70:].contiguous())))
    # attention over the whole length: every slot in front has value 0 and score 0, the last 70 their own
    q = (torch.randn(6, 1, 1, 64, generator=g) * LOG2E / 8).to(DEV)
    got, lse = ops.cache4_attention(q, c, c, need_lse=True)
    v = values(ops.Cache4(c.codes[:, :, T - 70:].contiguous(), c.meta[:, :, T - 70:].contiguous())).double()
    w = torch.exp2((q.double() * v).sum(-1))                                  # [6, 1, 70]
    total = w.sum(-1) + (T - 70)
    assert bool(((lse[..., 0].double() - torch.log2(total)).abs() < 1e-4).all())
    want = (w[..., None] * v).sum(2) / total[..., None]
    assert bool(((got.view(6, 1, 64).double() - want).abs() <= 1e-3 * want.abs().max()).all())
