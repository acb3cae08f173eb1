"""A paged cache in 4 bits -- written, read back, attended to -- against its definition in 64 bits.

Bounds, from the arithmetic. Rounding to nearest is off by u = 2^-11 (fp16) or 2^-8 (bf16) of the value at most; outputs
round once. Written rows are integers and have to be equal; of turned rows a value is off by half a step. Attention:
weights round to fp16 and once more with the factor of a value's group, 2^-10 sum p |v| <= 2^-10 max |v| together, the
output once. Scores are sums in 32 bits of integers 0..15 times q, the tensor core's 4 additions a group each off by
2^-22 of its largest operand: delta = 2^-20 * 15 * step * sum |q| * scale at most, which moves a weight by
a share of 2 delta and the logarithm of a sum by delta."""
import math

import pytest
import torch

from compressai_b200 import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
BOTH = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------------------------- oracles
def factors64(r):
    """Ratios in [0, 1] rounded up to e4m3."""
    e = (torch.frexp(r.clamp_min(2.0 ** -40))[1] - 1).clamp_min(-6)
    grid = ((e.long() - 3 + 1023) << 52).view(torch.float64)
    return torch.ceil(r / grid) * grid


def pack64(x):
    """Rows [n, D] of 16-bit values: codes [n, D] 1..15, scale [n] fp32, factors [n, groups]. Ties away from zero."""
    n, d = x.shape
    x = x.double()
    top = x.abs().amax(-1)
    bad, none = ~torch.isfinite(top), top < 1e-30
    safe = torch.where(bad | none, torch.ones_like(top), top)
    x = torch.where((bad | none)[:, None], torch.zeros_like(x), x)
    codes = torch.zeros(n, d, dtype=torch.int64, device=x.device)
    factor = torch.zeros(n, -(-d // 64), dtype=torch.float64, device=x.device)
    for g in range(factor.shape[1]):
        v = x[:, 64 * g:64 * g + 64]
        u = factors64(v.abs().amax(-1) / safe)
        factor[:, g] = torch.where(bad, torch.ones_like(u), u)
        div = torch.where(u == 0, torch.ones_like(u), safe * u)
        t = 7 * v / div[:, None]
        codes[:, 64 * g:64 * g + 64] = (torch.sign(t) * torch.floor(t.abs() + 0.5)).long()
    scale = torch.where(bad, torch.full_like(top, math.nan), torch.where(none, torch.zeros_like(top), top / 7))
    return codes + 8, scale.float(), factor


def parts(pool, scales):
    """A pool's codes [pages, heads, page, D], scales [pages, heads, page], factors [pages, heads, page, groups]."""
    codes = torch.stack([pool & 15, pool >> 4], -1).flatten(-2).long()
    scale = scales[..., :4, :].flatten(-2).contiguous().view(torch.float32).flatten(-2)
    f = scales[..., 4:, :].contiguous().view(torch.float8_e4m3fn).double()   # [pages, heads, page / 16, groups, 16]
    return codes, scale, f.transpose(-1, -2).flatten(2, 3)


def values64(pool, scales):
    codes, scale, f = parts(pool, scales)
    step = (f * scale.double()[..., None]).repeat_interleave(64, -1)[..., : codes.shape[-1]]
    return (codes - 8).double() * step


def fill(pool, scales, x):
    """Every row of a pool [pages, heads, page, D] from x in 16 bits."""
    pages, heads, P, d = x.shape
    codes, scale, f = pack64(x.reshape(-1, d))
    c = codes.view(pages, heads, P, d).to(torch.uint8)
    pool.copy_(c[..., 1::2] << 4 | c[..., 0::2])
    scales[..., :4, :] = scale.view(torch.uint8).view(pages, heads, P // 16, 4, 16)
    f = f.float().to(torch.float8_e4m3fn).view(torch.uint8).view(pages, heads, P // 16, 16, -1)
    scales[..., 4:, :] = f.transpose(-1, -2)


def turn64(x, pos, f, interleaved=False, factor=1.0):
    x = x.double().clone()
    n = f.numel()
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        t = pos.double() * f[i].double()
        c, s = (factor * torch.cos(t))[:, None], (factor * torch.sin(t))[:, None]
        u, w = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = u * c - w * s, u * s + w * c
    return x


class Setup:
    """4-bit pools of random rows, pages in no order; what no sequence has written holds NaN scales and any bytes."""

    def __init__(self, news, lens, hq, hkv, d, dtype, page=16, seed=0, spread=0.5, spare=2):
        g = gen(seed)
        self.news, self.lens_list, self.dtype, self.page, self.d = news, lens, dtype, page, d
        T = sum(news)
        self.q = torch.randn(T, hq, d, generator=g, device=DEV).to(dtype)
        need = [-(-l // page) for l in lens]
        n = sum(need) + spare
        perm = torch.randperm(n, generator=g, device=DEV).to(torch.int32).tolist()
        self.table = torch.full((len(lens), max(need + [0]) + 1), -1, dtype=torch.int32, device=DEV)
        fresh = torch.ones(n, page, dtype=torch.bool, device=DEV)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = torch.tensor(perm[at:at + k], dtype=torch.int32, device=DEV)
            for j in range(k):
                fresh[perm[at + j], : min(page, lens[b] - j * page)] = False
            at += k
        self.pools, self.scales = [], []
        rec = fresh.view(n, 1, page // 16, 1, 16)
        for _ in range(2):
            pool, scales = A.empty_pool(n, hkv, page, d, torch.int4)
            gain = torch.exp(spread * torch.randn(d, generator=g, device=DEV))
            fill(pool, scales, (torch.randn(n, hkv, page, d, generator=g, device=DEV) * gain).to(dtype))
            pool.masked_fill_(fresh[:, None, :, None], 0)
            nan = torch.full((n, hkv, page // 16, 16), math.nan, device=DEV).view(torch.uint8).view(n, hkv, page // 16, 4, 16)
            ours = scales[..., :4, :].flatten(-2).contiguous().view(torch.float32)
            ours = ours.masked_fill(fresh.view(n, 1, page // 16, 16), math.nan)
            scales[..., :4, :] = ours.view(torch.uint8).view_as(nan)
            scales[..., 4:, :] = scales[..., 4:, :].masked_fill(rec, 0xFF)
            self.pools.append(pool)
            self.scales.append(scales)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.starts = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device=DEV)

    def run(self, **kw):
        return A.paged_attention(self.q, *self.pools, self.table, self.lens, kw.pop("starts", self.starts),
                                 k_scale=self.scales[0], v_scale=self.scales[1], **kw)

    def rows64(self, which, b, n):
        p = torch.arange(n, device=DEV)
        ids = self.table[b].long()[p // self.page]
        return values64(self.pools[which][ids.unique()], self.scales[which][ids.unique()])[
            torch.searchsorted(ids.unique(), ids), :, p % self.page]

    def check(self, out, lse=None, scale=None, causal=True, window=0):
        scale = self.d ** -0.5 if scale is None else scale
        at = 0
        for b, (n, l) in enumerate(zip(self.news, self.lens_list)):
            k, v = (self.rows64(c, b, l) for c in (0, 1))
            want, want_lse = attend64(self.q[at:at + n], k, v, torch.arange(l - n, l, device=DEV), scale, causal, window)
            got = out[at:at + n].double()
            assert torch.isfinite(got).all()
            top = v.abs().max().item() if l else 0.0
            step = k.abs().max().item() / 7 if l else 0.0
            delta = 2.0 ** -20 * 15 * step * abs(scale) * self.q[at:at + n].abs().double().sum(-1).max().item() if n else 0.0
            tol = (2.0 ** -10 + 2 * delta + 2e-5) * top + EPS[self.dtype] * want.abs()
            assert ((got - want).abs() <= tol).all(), (b, n, l, ((got - want).abs() - tol).max().item())
            if lse is not None:
                have = lse[at:at + n].double()
                assert torch.equal(torch.isinf(have), torch.isinf(want_lse))
                fine = ~torch.isinf(want_lse)
                assert ((have - want_lse).abs()[fine] <= delta + 1e-5 * (1 + want_lse.abs()[fine])).all()
            at += n


def attend64(q, k, v, pos, scale, causal, window):
    n, hq, d = q.shape
    l = torch.arange(k.shape[0], device=DEV)
    sees = torch.ones(n, k.shape[0], dtype=torch.bool, device=DEV)
    if causal:
        sees &= l[None] <= pos[:, None]
    if window:
        sees &= l[None] > pos[:, None] - window
    g = hq // k.shape[1]
    x = torch.einsum("nhd,lhd->hnl", q.double(), k.repeat_interleave(g, 1)) * scale
    x = x.masked_fill(~sees[None], -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    return torch.einsum("hnl,lhd->nhd", p, v.repeat_interleave(g, 1)), lse.t()


def one_sequence(T, heads, d, page):
    """Pools for one sequence of T tokens on pages in reverse order, and the call's table, lens and starts."""
    n = -(-T // page)
    pools = [A.empty_pool(n, heads, page, d, torch.int4) for _ in range(2)]
    table = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([T], dtype=torch.int32, device=DEV)
    return pools, table, lens, torch.tensor([0, T], dtype=torch.int32, device=DEV)


def stored(pool, scales, table, T, page):
    """Codes, scales and factors of positions 0 .. T - 1: [T, heads, ..]."""
    p = torch.arange(T, device=DEV)
    ids = table[0].long()[p // page]
    return [x[ids, :, p % page] for x in parts(pool, scales)]


# ------------------------------------------------------------------------------------- write, read
def awkward(x):
    """Some of the rows [T, heads, D] replaced by what quantising meets at its edges."""
    T, _, d = x.shape
    i = torch.arange(d, device=DEV)
    rows = [torch.zeros(d, device=DEV),
            torch.where(i == d - 1, 3.0e4, 0.001 * (i + 1.0)),                    # one channel far above the others
            (i % 15 - 7.0) / 14,                                                   # right between two codes: x / (1 / 14)
            torch.where(i == 0, 1.0, ((i % 14) * 2 + 1.0) / 32),
            torch.full((d,), 2.0 ** -24, device=DEV),
            torch.where(i < 32, 6.0e4, -6.0e4),
            torch.where(i == 5, math.inf, 1.0),
            torch.where(i == 7, math.nan, 1.0),
            torch.where(i == 0, 1.0, torch.where(i < 40, 0.4375, -0.3125))]
    for j, r in enumerate(rows):
        x[(3 * j + 1) % T] = r.to(x.dtype)
    return x


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("T,heads,d,page", [(29, 1, 32, 16), (31, 3, 64, 32), (40, 2, 96, 16), (27, 2, 160, 64), (33, 2, 256, 64),
                                            (5003, 8, 128, 16), (3001, 2, 224, 128)])
def test_written_rows_are_the_definitions(dtype, T, heads, d, page):
    """Not turned, the inputs are 16-bit values: every code, scale and factor is the exact one, ties included."""
    g = gen(T)
    k, v = (awkward((torch.randn(T, heads, d, generator=g, device=DEV)
                     * torch.exp(torch.randn(d, generator=g, device=DEV))).to(dtype)) for _ in range(2))
    pools, table, lens, starts = one_sequence(T, heads, d, page)
    assert A.cache_write(k, v, pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1]) is None
    back = A.cache_read(pools[0][0], pools[1][0], table, starts, T, k_scale=pools[0][1], v_scale=pools[1][1], dtype=dtype)
    for x, (pool, scales), y in zip((k, v), pools, back):
        codes, scale, factor = stored(pool, scales, table, T, page)
        c64, s64, f64 = (t.view(T, heads, *t.shape[1:]) for t in pack64(x.reshape(-1, d)))
        assert torch.equal(codes, c64) and torch.equal(factor, f64)
        assert torch.equal(scale.isnan(), s64.isnan())
        fine = ~s64.isnan()
        # amax / 7 rounded once to 32 bits
        assert ((scale - s64).abs()[fine] <= 2.0 ** -23 * s64[fine]).all()
        want = ((codes - 8).double() * (factor.repeat_interleave(64, -1)[..., :d] * scale.double()[..., None]))
        assert torch.equal(y.isnan().any(-1), ~fine) and torch.equal(y.isnan().all(-1), ~fine)
        w = want[fine]
        lost = 2.0 ** -25 if dtype == torch.float16 else 0.0   # half of fp16's smallest number
        assert ((y[fine].double() - w).abs() <= EPS[dtype] * (1 + 1e-3) * w.abs() + lost).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_every_size_of_number(dtype):
    """bf16 rows from 2^-140 to the largest numbers: a row below 1e-30 is zeros, the others keep their half step."""
    d, T = 64, 260
    e = torch.arange(T, device=DEV) - 140 if dtype == torch.bfloat16 else torch.arange(T, device=DEV) % 39 - 24
    x = torch.ldexp(1 + 0.9 * torch.rand(T, 1, d, generator=gen(1), device=DEV, dtype=torch.float64), e[:, None, None])
    x = x.clamp_max(torch.finfo(dtype).max).to(dtype)
    pools, table, lens, starts = one_sequence(T, 1, d, 16)
    A.cache_write(x, -x, pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1])
    for y, (pool, scales) in zip((x, -x), pools):
        codes, scale, factor = stored(pool, scales, table, T, 16)
        c64, s64, f64 = pack64(y.reshape(-1, d))
        assert torch.equal(codes[:, 0], c64) and torch.equal(factor[:, 0], f64)
        assert ((scale[:, 0] - s64).abs() <= 2.0 ** -23 * s64 + 2.0 ** -149).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,hq,heads,d,rot", [(1, 16, 2, 256, 64), (7, 4, 2, 96, 24), (3, 2, 1, 64, 10), (40, 3, 3, 32, 32),
                                              (3000, 8, 2, 128, 128), (2500, 4, 2, 96, 96), (2500, 4, 4, 256, 64),
                                              (2500, 6, 2, 160, 136), (2500, 3, 1, 64, 20)])
def test_turned_rows(dtype, interleaved, T, hq, heads, d, rot):
    """k is turned in 32 bits ahead of its rounding: every value within half a step, every step what the group needs."""
    g = gen(5)
    qkv = torch.randn(T, (hq + 2 * heads) * d, generator=g, device=DEV).to(dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, heads * d, heads * d], 1))
    f = A.rope_frequencies(rot)[0].to(DEV)
    old = 50
    n = -(-(T + old) // 16)
    pools = [A.empty_pool(n, heads, 16, d, torch.int4) for _ in range(2)]
    table = torch.randperm(n, generator=g, device=DEV).to(torch.int32)[None]
    lens, starts = torch.tensor([old + T], dtype=torch.int32, device=DEV), torch.tensor([0, T], dtype=torch.int32, device=DEV)
    got_q = A.cache_write(k, v, pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1], q=q,
                          inv_freq=f, interleaved=interleaved, factor=1.25)
    pos = torch.arange(old, old + T, device=DEV)
    want_q = turn64(q, pos, f, interleaved, 1.25)
    assert ((got_q.double() - want_q).abs() <= EPS[dtype] * want_q.abs() + 2e-6 * q.abs().max()).all()
    for x, (pool, scales) in zip((turn64(k, pos, f, interleaved, 1.25), v.double()), pools):
        codes, scale, factor = (y[old:] for y in stored(pool, scales, table, old + T, 16))
        assert codes.min() >= 1 and codes.max() <= 15
        amax = x.abs().amax(-1)
        near = 4e-6 * amax   # the turn in 32 bits: angle, cos, sin, two products and a sum
        assert ((scale.double() * 7 - amax).abs() <= near).all()
        step = (factor * scale.double()[..., None])
        for i in range(factor.shape[-1]):
            y, w, c = x[..., 64 * i:64 * i + 64], step[..., i], codes[..., 64 * i:64 * i + 64] - 8
            top = y.abs().amax(-1)
            assert (7 * w >= top - 2 * near).all() and (7 * w <= (top + 2 * near) * 9 / 8 + amax / 512).all()
            assert ((c.double() * w[..., None] - y).abs() <= w[..., None] * 0.5 + 2 * near[..., None]).all()


def test_rows_around_a_write_stay():
    """A token's rows alone change: not the other rows of its scale record, nor anything for a token without a page."""
    d, heads, page = 96, 2, 16
    pools = [A.empty_pool(3, heads, page, d, torch.int4) for _ in range(2)]
    for pool, scales in pools:
        pool.random_(0, 256, generator=gen(1))
        scales.random_(0, 256, generator=gen(2))
    before = [(p.clone(), s.clone()) for p, s in pools]
    table = torch.tensor([[2, -1], [7, 0], [-5, 1]], dtype=torch.int32, device=DEV)   # 7, -5, -1: no such pages
    lens = torch.tensor([6, 3, 40], dtype=torch.int32, device=DEV)                    # the third: past its table
    x = torch.randn(3, heads, d, generator=gen(3), device=DEV).half()
    A.cache_write(x, -x, pools[0][0], pools[1][0], table, lens, k_scale=pools[0][1], v_scale=pools[1][1])
    for (pool, scales), (p0, s0) in zip(pools, before):
        same = torch.ones(3, heads, page, dtype=torch.bool, device=DEV)
        same[2, :, 5] = False
        assert torch.equal(pool[same], p0[same])
        now, was = (torch.cat([s[..., :4, :].flatten(-2).unflatten(-1, (16, 4)), s[..., 4:, :].transpose(-1, -2)], -1).flatten(2, 3)
                    for s in (scales, s0))   # [pages, heads, page, 4 + groups]
        assert torch.equal(now[same], was[same]) and not torch.equal(now[~same], was[~same])
        c64, s64, f64 = pack64((x if pool is pools[0][0] else -x)[0])
        codes, scale, f = parts(pool, scales)
        assert torch.equal(codes[2, :, 5], c64) and torch.equal(f[2, :, 5], f64)


def test_read_of_missing_rows_and_past_the_last():
    pools, table, lens, starts = one_sequence(20, 1, 64, 16)
    x = torch.randn(20, 1, 64, generator=gen(0), device=DEV).to(torch.bfloat16)
    A.cache_write(x, x, pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1])
    table = torch.tensor([[1, -1], [9, 0]], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 18, 18 + 20], dtype=torch.int32, device=DEV)
    for t in (None, torch.float16):
        k, v = A.cache_read(pools[0][0], pools[1][0], table, starts, 45, k_scale=pools[0][1], v_scale=pools[1][1], dtype=t)
        assert k.dtype == (t or torch.bfloat16) and torch.equal(k, v)
        assert k[16:18].abs().max() == 0 and k[18:34].abs().max() == 0 and k[38:].abs().max() == 0
        assert k[:16].abs().min(-1).values.max() >= 0 and k[:16].abs().max() > 1 and k[34:38].abs().max() > 0.5


# ------------------------------------------------------------------------------------- attention
SHAPES = [(16, 2, 256), (32, 8, 128), (4, 4, 64), (6, 2, 96), (5, 1, 160), (3, 1, 32), (10, 2, 224)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_decode(dtype, hq, hkv, d, page):
    lens = [1, 2, 15, 16, 17, 33, 64, 65, 127, 300, 511, 700]
    s = Setup([1] * len(lens), lens, hq, hkv, d, dtype, page=page, seed=d + page)
    out, lse = s.run(return_lse=True, starts=None)
    s.check(out, lse)
    s.check(s.run(window=40, starts=None), window=40)
    s.check(s.run(causal=False, scale=0.3, max_new=1, max_len=700), scale=0.3, causal=False)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_few_new_tokens(dtype, hq, hkv, d):
    news, lens = [2, 5, 1, 3, 5, 4], [2, 77, 1, 260, 1030, 4]
    s = Setup(news, lens, hq, hkv, d, dtype, page=32, seed=d)
    for kw in (dict(), dict(window=33), dict(causal=False), dict(causal=False, window=7)):
        out, lse = s.run(return_lse=True, max_new=5, max_len=1030, **kw)
        s.check(out, lse, **kw)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 2, 256, 64), (8, 2, 128, 16), (4, 4, 64, 128), (6, 2, 96, 32), (5, 1, 160, 16), (2, 1, 32, 16)])
def test_chunks(dtype, hq, hkv, d, page):
    news, lens = [100, 257, 1, 64], [100, 700, 130, 1000]
    s = Setup(news, lens, hq, hkv, d, dtype, page=page, seed=d)
    for kw in (dict(), dict(window=100), dict(causal=False)):
        out, lse = s.run(return_lse=True, max_new=257, max_len=1000, **kw)
        s.check(out, lse, **kw)
    s.check(s.run())


@pytest.mark.parametrize("hq,hkv,d,ctx", [(16, 2, 256, 20011), (8, 8, 128, 9003), (4, 1, 64, 30001)])
def test_long_sequences_are_split_and_joined(hq, hkv, d, ctx):
    s = Setup([1, 1], [ctx, 77], hq, hkv, d, torch.float16, page=64, seed=3)
    out, lse = s.run(return_lse=True, starts=None, max_len=ctx)
    s.check(out, lse)
    again = s.run(starts=None, max_len=ctx)
    assert torch.equal(out, again)   # sums in a fixed order


@pytest.mark.parametrize("new", [1, 3, 200])
def test_rows_that_see_nothing_and_tokens_of_no_sequence(new):
    s = Setup([new, new], [new + 5, new + 40], 4, 2, 64, torch.bfloat16, page=16)
    s.lens.zero_()
    out, lse = s.run(return_lse=True, max_new=new)
    assert out.abs().max() == 0 and (lse == -math.inf).all()
    s = Setup([new, new], [new + 5, new + 40], 4, 2, 64, torch.bfloat16, page=16)
    pad = torch.randn(2 * new + 7, 4, 64, generator=gen(4), device=DEV).to(torch.bfloat16)
    pad[3:3 + 2 * new] = s.q
    out, lse = A.paged_attention(pad, *s.pools, s.table, s.lens, s.starts + 3, k_scale=s.scales[0], v_scale=s.scales[1],
                                 max_new=new, return_lse=True)
    s.check(out[3:3 + 2 * new], lse[3:3 + 2 * new])
    rest = torch.cat([out[:3], out[3 + 2 * new:]])
    assert rest.abs().max() == 0 and (torch.cat([lse[:3], lse[3 + 2 * new:]]) == -math.inf).all()


@pytest.mark.parametrize("new", [1, 60])
def test_pages_that_do_not_exist_hide_their_keys(new):
    s = Setup([new], [300], 4, 2, 128, torch.float16, page=16, seed=9)
    want = s.run(max_new=new)
    keep = s.table.clone()
    s.table[0, 3], s.table[0, 7] = -1, 10 ** 6
    got = s.run(max_new=new)
    k, v = (s.rows64(c, 0, 300) if False else None for c in (0, 1))
    s.table.copy_(keep)
    k, v = s.rows64(0, 0, 300), s.rows64(1, 0, 300)
    there = torch.ones(300, dtype=torch.bool, device=DEV)
    there[48:64] = there[112:128] = False
    pos = torch.arange(300 - new, 300, device=DEV)
    x = torch.einsum("nhd,lhd->hnl", s.q.double(), k.repeat_interleave(2, 1)) * 128 ** -0.5
    x = x.masked_fill(~(there[None] & (torch.arange(300, device=DEV)[None] <= pos[:, None]))[None], -math.inf)
    ref = torch.einsum("hnl,lhd->nhd", torch.softmax(x, -1), v.repeat_interleave(2, 1))
    assert torch.isfinite(got).all() and ((got.double() - ref).abs() <= (2.0 ** -10 + 1e-4) * v.abs().max() + 2.0 ** -11 * ref.abs()).all()
    assert not torch.equal(got, want)


def test_a_row_that_is_not_finite():
    """Its NaN reaches the rows that see it, and those alone."""
    d, T = 64, 200
    pools, table, lens, starts = one_sequence(T, 1, d, 16)
    x = torch.randn(T, 1, d, generator=gen(0), device=DEV).half()
    x[150, 0, 3] = math.inf
    A.cache_write(x, x, pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1])
    q = torch.randn(T, 1, d, generator=gen(1), device=DEV).half()
    for lo in (0, 140, 199):   # the kernel for many rows, for few, one
        at = torch.tensor([0, T - lo], dtype=torch.int32, device=DEV)
        out = A.paged_attention(q[lo:], pools[0][0], pools[1][0], table, lens, at, k_scale=pools[0][1], v_scale=pools[1][1])
        assert torch.equal(out.isnan().any(-1).any(-1), torch.arange(lo, T, device=DEV) >= 150)


@pytest.mark.parametrize("scale_of", [2.0 ** -100, 2.0 ** 60])
@pytest.mark.parametrize("new", [1, 100])
def test_sizes_of_q_and_v(scale_of, new):
    """bf16 queries and values of any size: the products' fp16 stays in range (scores kept to the usual size)."""
    s = Setup([new], [200], 4, 2, 128, torch.bfloat16, page=32, seed=2)
    s.q = (s.q.float() * scale_of).to(torch.bfloat16)
    v = torch.randn(s.pools[1].shape[0], 2, 32, 128, generator=gen(6), device=DEV)
    v *= torch.exp2(torch.randint(-20, 20, (v.shape[0], 1, 32, 1), generator=gen(7), device=DEV).float()) * scale_of
    v = v.to(torch.bfloat16)
    fill(s.pools[1], s.scales[1], v)
    k, v64 = s.rows64(0, 0, 200), s.rows64(1, 0, 200)
    scale = 128 ** -0.5 / scale_of
    got = s.run(scale=scale, max_new=new).double()
    want, _ = attend64(s.q, k, v64, torch.arange(200 - new, 200, device=DEV), scale, True, 0)
    p_abs, _ = attend64(s.q, k, v64.abs(), torch.arange(200 - new, 200, device=DEV), scale, True, 0)
    tol = 2.0 ** -9 * p_abs + 2.0 ** -22 * v64.abs().max() + EPS[torch.bfloat16] * want.abs()
    assert torch.isfinite(got).all() and ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (4, 1, 256), (16, 1, 64)])
def test_scales_of_hidden_keys(hq, hkv, d, new):
    """What a window or a later position hides has no say, whatever the size of its values beside those of the keys seen."""
    window, l = 30, 300
    s = Setup([new], [l], hq, hkv, d, torch.bfloat16, page=256, seed=4)
    for which, seen in ((0, 1.0), (1, 2.0 ** -90)):
        x = torch.randn(s.pools[which].shape[0], hkv, 256, d, generator=gen(which), device=DEV)
        pos = torch.full((x.shape[0], 256), -1, device=DEV)
        for j in range(2):
            pos[s.table[0, j].long()] = torch.arange(256 * j, 256 * j + 256, device=DEV)
        last = l - new - window + 1   # positions that no row sees
        x *= torch.where(pos < last, 2.0 ** (100 if which else 30), torch.where(pos < l, seen, 2.0 ** 90))[:, None, :, None]
        fill(s.pools[which], s.scales[which], x.to(torch.bfloat16))
    s.check(s.run(window=window, max_new=new), window=window)


def test_graph_streams_and_strides():
    s = Setup([1, 1, 1], [100, 300, 17], 8, 2, 128, torch.bfloat16, page=16, seed=1)
    want = s.run(starts=None, max_len=400)
    wide = torch.zeros(3, 3, 8, 128 + 8, dtype=torch.bfloat16, device=DEV)
    wide[:, 1, :, :128] = s.q
    args = dict(k_scale=s.scales[0], v_scale=s.scales[1], max_len=400)
    got = A.paged_attention(wide[:, 1, :, :128], *s.pools, s.table, s.lens, None, **args)
    assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = s.run(starts=None, max_len=400)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, want)
    k = torch.randn(3, 2, 128, generator=gen(8), device=DEV).to(torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.cache_write(k, -k, *s.pools, s.table, s.lens, k_scale=s.scales[0], v_scale=s.scales[1])
        out = s.run(starts=None, max_len=400)
    for lens in ([100, 300, 17], [31, 290, 1]):
        s.lens.copy_(torch.tensor(lens, dtype=torch.int32, device=DEV))
        s.lens_list = lens
        graph.replay()
        s.check(out)
    torch.cuda.synchronize()


def test_offsets_past_32_bits():
    """Rows and bytes of a pool counted past 2^31."""
    pages, heads, page, d = 40000, 8, 64, 256    # 2.6 GB of codes, 20 M rows
    pools = [A.empty_pool(pages, heads, page, d, torch.int4) for _ in range(2)]
    T = 130
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=DEV)
    lens, starts = torch.tensor([T], dtype=torch.int32, device=DEV), torch.tensor([0, T], dtype=torch.int32, device=DEV)
    x = torch.randn(2, T, heads, d, generator=gen(0), device=DEV).half()
    A.cache_write(x[0], x[1], pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1])
    k, v = A.cache_read(pools[0][0], pools[1][0], table, starts, T, k_scale=pools[0][1], v_scale=pools[1][1], dtype=torch.float16)
    for got, want in zip((k, v), x):
        c, s, f = pack64(want.reshape(-1, d))
        w = (c - 8).double() * (f * s.double()[:, None]).repeat_interleave(64, -1)
        assert ((got.reshape(-1, d).double() - w).abs() <= 2.0 ** -11 * (1 + 1e-3) * w.abs() + 2.0 ** -25).all()
    q = torch.randn(T, heads, d, generator=gen(1), device=DEV).half()
    for n in (1, T):
        got = A.paged_attention(q[T - n:], pools[0][0], pools[1][0], table, lens, torch.tensor([0, n], dtype=torch.int32, device=DEV),
                                k_scale=pools[0][1], v_scale=pools[1][1], max_new=n)
        want, _ = attend64(q[T - n:], k.double(), v.double(), torch.arange(T - n, T, device=DEV), d ** -0.5, True, 0)
        # over the values as read back: rounded to fp16 once more
        assert ((got.double() - want).abs() <= (2.0 ** -10 + 2.0 ** -10 * 4) * v.abs().max().double() + 2.0 ** -11 * want.abs()).all()


@pytest.mark.parametrize("new,old", [(1, 200), (90, 37)])
def test_a_step_as_it_is_used(new, old):
    """PagedKVCache in 4 bits: prompts, then a step, written and attended to, layer by layer."""
    c = A.PagedKVCache(2, 40, 2, 128, page_size=16, dtype=torch.int4)
    a, b = c.add(), c.add()
    g = gen(11)
    f = A.rope_frequencies(64)[0].to(DEV)
    hist = {}
    for counts in ([old, old // 2], [new, 1]):
        c.begin([a, b], counts)
        T = sum(counts)
        for layer in range(2):
            q, k, v = (torch.randn(T, h, 128, generator=g, device=DEV).to(torch.bfloat16) for h in (8, 2, 2))
            turned = c.write(layer, k, v, q=q, inv_freq=f)
            out = c.attend(layer, turned)
            at = 0
            for s, n in zip((a, b), counts):
                L = c.lengths[s]
                ids = torch.tensor(c.pages[s], device=DEV)
                kk, vv = (values64(c.pools[layer][i][ids], c.scales[layer][i][ids]).transpose(1, 2).flatten(0, 1)[:L] for i in (0, 1))
                hist.setdefault((layer, s), []).append(v[at:at + n])
                want_v = torch.cat(hist[layer, s]).double()
                step = want_v.abs().amax(-1, keepdim=True) / 7 * 9 / 8
                assert ((vv - want_v).abs() <= step * (0.5 + 1e-6)).all()
                want, _ = attend64(turned[at:at + n], kk, vv, torch.arange(L - n, L, device=DEV), 128 ** -0.5, True, 0)
                tol = (2.0 ** -10 + 2e-4) * vv.abs().max() + EPS[torch.bfloat16] * want.abs()
                assert ((out[at:at + n].double() - want).abs() <= tol).all()
                at += n
    A.check_status()
