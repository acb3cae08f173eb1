"""Rotary, the paged key/value cache and attention over it against their formulas in 64 bits.

Bounds, from the arithmetic: rounding to nearest in fp16 (11 significant bits) or bf16 (8) is off by
at most u = 2^-11 or 2^-8 of the value; outputs round once. Attention also rounds the softmax weights
to 16 bits, each by at most u, so a row is off by at most u * sum p |v| <= u * max |v| more."""
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


def randn(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(*shape, generator=gen(seed), device=DEV).to(dtype)


# ------------------------------------------------------------------------------------- oracles
def turn64(x, pos, f, interleaved=False, factor=1.0, sign=1.0):
    x = x.double().clone()
    n = f.numel()
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        t = pos.double() * f[i].double()
        c, s = (factor * torch.cos(t))[:, None], (sign * factor * torch.sin(t))[:, None]
        u, w = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = u * c - w * s, u * s + w * c
    return x


def cache64(pages, scale, table, b, n):
    """Positions 0 .. n-1 of sequence b in 64 bits: [n, kv_heads, D]."""
    P = pages.shape[2]
    p = torch.arange(n, device=DEV)
    ids = table[b].long()[p // P]
    x = pages[ids, :, p % P].double()
    return x if scale is None else x * scale[ids, :, p % P].double()[..., None]


def attend64(q, k, v, pos, scale, causal, window):
    """q [n, Hq, D] at positions pos over k, v [l, Hkv, D]: (out, lse) in 64 bits."""
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


class Setup:
    """Pools with NaN wherever no sequence has written, pages in no order, a table with -1 past the needed ones."""

    def __init__(self, news, lens, hq, hkv, d, dtype, int8=False, page=16, seed=0, garbage=float("nan"), spare=2):
        g = gen(seed)
        self.news, self.lens_list, self.dtype, self.page = news, lens, dtype, page
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
        self.scale = []
        self.pools = []
        for _ in range(2):
            x = torch.randn(n, hkv, page, d, generator=g, device=DEV).to(dtype)
            if int8:
                amax = x.abs().amax(-1, keepdim=True).float()
                self.pools.append(torch.round(x.float() * (127 / amax)).clamp(-127, 127).to(torch.int8))
                self.scale.append((amax[..., 0] / 127).masked_fill(fresh[:, None], garbage))
            else:
                self.pools.append(x.masked_fill(fresh[:, None, :, None], garbage))
                self.scale.append(None)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.starts = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device=DEV)

    def run(self, **kw):
        return A.paged_attention(self.q, *self.pools, self.table, self.lens, kw.pop("starts", self.starts),
                                 k_scale=self.scale[0], v_scale=self.scale[1], **kw)

    def check(self, out, lse=None, scale=None, causal=True, window=0):
        d = self.q.shape[2]
        scale = d ** -0.5 if scale is None else scale
        at = 0
        for b, (n, l) in enumerate(zip(self.news, self.lens_list)):
            k, v = (cache64(p, s, self.table, b, l) for p, s in zip(self.pools, self.scale))
            pos = torch.arange(l - n, l, device=DEV)
            want, want_lse = attend64(self.q[at:at + n], k, v, pos, scale, causal, window)
            got = out[at:at + n].double()
            assert torch.isfinite(got).all()
            top = v.abs().max().item() if l else 0.0
            # weights and output each rounded once to 16 bits, 32-bit scores and sums
            tol = (EPS[self.dtype] + 2e-5) * top + EPS[self.dtype] * want.abs()
            assert ((got - want).abs() <= tol).all(), (b, n, l, ((got - want).abs() - tol).max().item())
            if lse is not None:
                have = lse[at:at + n].double()
                assert torch.equal(torch.isinf(have), torch.isinf(want_lse))
                fine = ~torch.isinf(want_lse)
                assert ((have - want_lse).abs()[fine] <= 1e-4).all()
            at += n


# ------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,hq,hk,d,rot", [(1, 16, 2, 256, 64), (5, 3, 1, 64, 64), (1000, 4, 4, 96, 24), (3, 5, 0, 128, 2),
                                           (2, 1, 1, 16, 10), (300, 40, 8, 128, 128)])
def test_rotary(dtype, interleaved, T, hq, hk, d, rot):
    q, k = randn(T, hq, d, dtype=dtype, seed=1), randn(T, hk, d, dtype=dtype, seed=2) if hk else None
    f, _ = A.rope_frequencies(rot)
    f = f.to(DEV)
    pos = torch.randint(0, 200000, (T,), generator=gen(3), device=DEV)
    for inverse in (False, True):
        got = A.rotary(q, k, pos, f, interleaved=interleaved, factor=1.25, inverse=inverse)
        for x, y in zip((q, k), got):
            if x is None:
                assert y is None
                continue
            want = turn64(x, pos, f, interleaved, 1.25, -1.0 if inverse else 1.0)
            want[..., rot:] = x[..., rot:].double()
            tol = EPS[dtype] * want.abs() + 4e-6 * x.double().abs().max()
            assert ((y.double() - want).abs() <= tol).all()
    same = A.rotary(q, k, pos.int(), f, interleaved=interleaved, factor=1.25, inverse=True)
    assert torch.equal(same[0], got[0])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hk,d,rot", [(9, 2, 256, 64), (4, 7, 16, 10), (5, 5, 48, 8), (3, 1, 16, 8), (12, 0, 112, 112)])
def test_rotary_many_tokens_unaligned(interleaved, hq, hk, d, rot):
    """More tokens than blocks at once, rows that start anywhere, widths that are no whole number of loads."""
    T = 9001
    big = randn(T, (hq + hk) * d + 1, seed=30)
    q, k = big[:, 1:1 + hq * d].unflatten(1, (hq, d)), big[:, 1 + hq * d:].unflatten(1, (hk, d)) if hk else None
    f = A.rope_frequencies(rot)[0].to(DEV)
    pos = torch.arange(T, device=DEV) + 30000
    for views in ((q, k), (q.contiguous(), k.contiguous() if hk else None)):
        for x, y in zip(views, A.rotary(*views, pos, f, interleaved=interleaved)):
            if x is None:
                continue
            want = turn64(x, pos, f, interleaved, 1.0)
            want[..., rot:] = x[..., rot:].double()
            assert ((y.double() - want).abs() <= EPS[x.dtype] * want.abs() + 4e-6 * x.double().abs().max()).all()
            assert torch.equal(y[..., rot:], x[..., rot:])


def test_rotary_strided_and_unaligned():
    big = randn(9, 7 * 64 + 3, seed=4)
    f = A.rope_frequencies(64)[0].to(DEV)
    pos = torch.arange(9, device=DEV)
    for view in (big[:, 3:3 + 128].unflatten(1, (2, 64)), big[:, 8:8 + 384].unflatten(1, (3, 128))[..., :64],
                 randn(64, 9, 2, seed=5).permute(1, 2, 0)):
        got, _ = A.rotary(view, None, pos, f)
        assert torch.equal(got, A.rotary(view.contiguous(), None, pos, f)[0])


def test_rotary_inverse_is_the_gradient():
    """The inverse of a cotangent is the formula's gradient, and what differences of the forward pass say."""
    T, h, d, rot = 3, 2, 16, 12
    f = A.rope_frequencies(rot)[0].to(DEV)
    pos = torch.tensor([0, 7, 4097], device=DEV)
    x = randn(T, h, d, dtype=torch.float16, seed=6)
    w = randn(T, h, d, dtype=torch.float16, seed=7)
    for interleaved in (False, True):
        back = A.rotary(w, None, pos, f, interleaved=interleaved, factor=1.5, inverse=True)[0].double()
        y = x.double().requires_grad_()
        parts = turn64_grad(y, pos, f, interleaved, 1.5)
        (parts * w.double()).sum().backward()
        assert ((back - y.grad).abs() <= 2.0 ** -11 * y.grad.abs() + 1e-5).all()
        # differences: the map is linear, so a step along e_i moves <w, f(x)> by the i-th gradient times the step,
        # up to the fp16 rounding of the outputs it touches (at most 4 in magnitude, two of them)
        for i in (0, 5, 11, 15):
            e = torch.zeros_like(x)
            e[1, 1, i] = 1.0
            fwd = A.rotary(e, None, pos, f, interleaved=interleaved, factor=1.5)[0].double()
            assert abs((fwd * w.double()).sum().item() - back[1, 1, i].item()) <= 2 * 2.0 ** -11 * 2 * 4


def turn64_grad(x, pos, f, interleaved, factor):
    n = f.numel()
    t = pos.double()[:, None, None] * f.double()
    c, s = torch.cos(t) * factor, torch.sin(t) * factor
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    a, b = a * c - b * s, b * c + a * s
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


# ------------------------------------------------------------------------------------- cache
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("news,lens", [([1], [1]), ([1, 1, 1], [17, 1, 300]), ([33, 0, 5], [40, 9, 5]), ([700], [1234])])
@pytest.mark.parametrize("hq,hkv,d,rot,page", [(16, 2, 256, 64, 64), (3, 3, 96, 24, 16), (5, 1, 64, 64, 32)])
@pytest.mark.parametrize("int8", [False, True])
def test_cache_write_and_read(dtype, news, lens, hq, hkv, d, rot, page, int8):
    s = Setup(news, lens, hq, hkv, d, dtype, int8, page, seed=8, garbage=0.0)
    T = sum(news)
    qkv = randn(T, (hq + 2 * hkv) * d, dtype=dtype, seed=9)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    f = A.rope_frequencies(rot)[0].to(DEV)
    before = [p.clone() for p in s.pools]
    got_q = A.cache_write(k, v, *s.pools, s.table, s.lens, s.starts, k_scale=s.scale[0], v_scale=s.scale[1], q=q,
                          inv_freq=f, interleaved=True)
    pos = torch.cat([torch.arange(l - n, l, device=DEV) for n, l in zip(news, lens)])
    assert torch.equal(got_q, A.rotary(q, None, pos, f, interleaved=True)[0])
    want = [turn64(k, pos, f, True), v.double()]
    seq = torch.repeat_interleave(torch.arange(len(news), device=DEV), torch.tensor(news, device=DEV))
    ids, off = s.table[seq, pos // page].long(), pos % page
    for x, pool, scale, old in zip(want, s.pools, s.scale, before):
        have = pool[ids, :, off].double()
        if int8:
            step = x.abs().amax(-1) / 127
            have_step = scale[ids, :, off].double()
            assert ((have_step - step).abs() <= 1e-5 * step).all()
            # half a step of rounding, and the 32-bit error of the rotation and of the scale
            assert ((have * have_step[..., None] - x).abs() <= (0.5 + 2e-3) * step[..., None]).all()
        else:
            assert ((have - x).abs() <= EPS[dtype] * x.abs() + 4e-6 * x.abs().max()).all()
        other = pool.clone()       # nothing else was touched
        other[ids, :, off] = old[ids, :, off]
        assert torch.equal(other, old)
    ends = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    rk, rv = A.cache_read(*s.pools, s.table, ends, sum(lens), k_scale=s.scale[0], v_scale=s.scale[1], dtype=dtype)
    for got, pool, scale in zip((rk, rv), s.pools, s.scale):
        full = torch.cat([cache64(pool, scale, s.table, b, l) for b, l in enumerate(lens)])
        assert ((got.double() - full).abs() <= EPS[dtype] * full.abs()).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("news,lens", [([3], [5]), ([1500, 0, 2001], [1500, 9, 4000])])
@pytest.mark.parametrize("hq,hkv,d,rot", [(16, 2, 256, 64), (4, 3, 96, 28), (2, 2, 64, 64)])
def test_cache_write_half_layout(int8, news, lens, hq, hkv, d, rot):
    """The layout of `test_cache_write_and_read` is the neighbours'; here the halves', few tokens and many."""
    page, dtype = 32, torch.float16
    s = Setup(news, lens, hq, hkv, d, dtype, int8, page, seed=31, garbage=0.0)
    q, k, v = (randn(sum(news), h, d, dtype=dtype, seed=32 + i) for i, h in enumerate((hq, hkv, hkv)))
    f = A.rope_frequencies(rot)[0].to(DEV)
    got_q = A.cache_write(k, v, *s.pools, s.table, s.lens, s.starts, k_scale=s.scale[0], v_scale=s.scale[1], q=q, inv_freq=f)
    pos = torch.cat([torch.arange(l - n, l, device=DEV) for n, l in zip(news, lens)])
    want_q, want_k = (turn64(x, pos, f, False) for x in (q, k))
    assert ((got_q.double() - want_q).abs() <= EPS[dtype] * want_q.abs() + 4e-6 * q.double().abs().max()).all()
    seq = torch.repeat_interleave(torch.arange(len(news), device=DEV), torch.tensor(news, device=DEV))
    ids, off = s.table[seq, pos // page].long(), pos % page
    for x, pool, scale in zip((want_k, v.double()), s.pools, s.scale):
        have = pool[ids, :, off].double()
        if int8:
            step = x.abs().amax(-1) / 127
            have_step = scale[ids, :, off].double()
            assert ((have_step - step).abs() <= 1e-5 * step).all()
            assert ((have * have_step[..., None] - x).abs() <= (0.5 + 2e-3) * step[..., None]).all()
        else:
            assert ((have - x).abs() <= EPS[dtype] * x.abs() + 4e-6 * x.abs().max()).all()


def test_cache_write_int8_edges():
    """Zero rows, rows too small to scale, infinities and NaN; the largest values; no rotation."""
    d = 32
    k = randn(6, 1, d, dtype=torch.bfloat16, seed=10)
    k[0] = 0
    k[1] = 1e-35
    k[2, 0, 3] = float("inf")
    k[3, 0, 31] = float("nan")
    k[4, 0, 0] = 3e38
    pools = [torch.full((1, 1, 16, d), 77, dtype=torch.int8, device=DEV) for _ in range(2)]
    scale = [torch.full((1, 1, 16), 5.0, device=DEV) for _ in range(2)]
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    lens, starts = torch.tensor([6], dtype=torch.int32, device=DEV), torch.tensor([0, 6], dtype=torch.int32, device=DEV)
    assert A.cache_write(k, k, *pools, table, lens, starts, k_scale=scale[0], v_scale=scale[1]) is None
    for p, s in zip(pools, scale):
        s, p = s[0, 0], p[0, 0]
        assert (p[:4] == 0).all() and (s[:2] == 0).all() and torch.isnan(s[2:4]).all()
        assert p[4, 0] == 127 and p[5].abs().max() == 127 and (p[6:] == 77).all() and (s[6:] == 5).all()
    back = A.cache_read(*pools, table, starts, 6, k_scale=scale[0], v_scale=scale[1])[0]
    assert (back[:2] == 0).all() and torch.isnan(back[2:4]).all() and torch.isfinite(back[4:]).all()


def test_cache_tokens_without_a_page_are_not_stored():
    d, dt = 16, torch.float16
    pools = [torch.zeros(2, 1, 16, d, dtype=dt, device=DEV) for _ in range(2)]
    table = torch.tensor([[0, -1], [5, 1]], dtype=torch.int32, device=DEV)    # page 5 does not exist
    lens = torch.tensor([18, 40], dtype=torch.int32, device=DEV)             # 40 > 32: past the table
    starts = torch.tensor([0, 4, 14], dtype=torch.int32, device=DEV)
    k = randn(14, 1, d, dtype=dt, seed=11)
    A.cache_write(k, k, *pools, table, lens, starts)
    want = torch.zeros_like(pools[0])
    want[0, 0, 14:16] = k[:2, 0]
    want[1, 0, 14:16] = k[4:6, 0]                                            # positions 30, 31
    assert torch.equal(pools[0], want) and torch.equal(pools[1], want)
    ends = torch.tensor([0, 20, 40], dtype=torch.int32, device=DEV)
    got = A.cache_read(*pools, table, ends, 45)[0][:, 0]
    assert torch.equal(got[:16], pools[0][0, 0]) and (got[16:36] == 0).all()
    assert torch.equal(got[36:40], pools[0][1, 0, :4]) and (got[40:] == 0).all()


# ------------------------------------------------------------------------------------- attention
SHAPES = [(16, 2, 256), (8, 8, 64), (12, 4, 96), (5, 1, 128), (32, 2, 128), (20, 1, 16)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_attention_decode(dtype, int8, hq, hkv, d):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 700, 2049]
    s = Setup([1] * len(lens), lens, hq, hkv, d, dtype, int8, page=16, seed=12)
    out, lse = s.run(starts=None, return_lse=True)
    s.check(out, lse)
    assert torch.equal(out, s.run(max_new=1, max_len=2049))
    s.check(s.run(window=48, scale=0.3), window=48, scale=0.3)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 33), (False, 200)])
def test_attention_chunks(dtype, int8, hq, hkv, d, causal, window):
    news, lens = [5, 1, 130, 0, 64, 257, 2], [5, 40, 130, 33, 300, 700, 1025]
    s = Setup(news, lens, hq, hkv, d, dtype, int8, page=32, seed=13)
    out, lse = s.run(causal=causal, window=window, return_lse=True)
    s.check(out, lse, causal=causal, window=window)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("int8", [False, True])
def test_attention_page_sizes(page, int8):
    s = Setup([1, 40, 3], [333, 777, 129], 4, 2, 128, torch.bfloat16, int8, page, seed=14)
    s.check(s.run())
    d = Setup([1, 1], [333, 129], 4, 2, 128, torch.bfloat16, int8, page, seed=14)
    d.check(d.run(starts=None))


@pytest.mark.parametrize("page", [16, 64, 128, 256])
@pytest.mark.parametrize("d", [64, 160, 192, 256])
def test_attention_pages_end_inside_tiles(page, d):
    """Sequences that end everywhere in a tile and a page, every unwritten row of it NaN."""
    lens = [33, 64, 65, 95, 128, 129, 191, 193, 257, 300]
    s = Setup([min(n, 40) for n in lens], lens, 8, 2, d, torch.float16, False, page, seed=26)
    s.check(s.run())
    s.check(s.run(window=70), window=70)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (12, 3, 128), (4, 1, 256)])
@pytest.mark.parametrize("seqs", [3, 32, 33])
def test_attention_sequences_in_any_order(int8, hq, hkv, d, seqs):
    """Lengths that rise and fall, equal ones among them, new tokens from none to all, up to and past 32 sequences."""
    lens = [(37 * i * i + 11) % 530 + 1 for i in range(seqs)]
    lens[-1] = lens[0]
    news = [min(l, 0 if i % 7 == 3 else 40 + i) for i, l in enumerate(lens)]
    s = Setup(news, lens, hq, hkv, d, torch.float16, int8, page=32, seed=40)
    s.check(*s.run(return_lse=True))
    from compressai_b200 import _lib
    assert _lib.load().vq2_attention_status(0) == 0


@pytest.mark.parametrize("int8", [False, True])
def test_attention_rows_that_see_nothing(int8):
    """Empty sequences, more new tokens than the cache holds, and tokens of no sequence: zeros, lse -inf."""
    s = Setup([1, 1], [0, 20], 4, 2, 64, torch.float16, int8, seed=15)
    out, lse = s.run(starts=None, return_lse=True)
    assert (out[0] == 0).all() and torch.isinf(lse[0]).all() and (lse[0] < 0).all() and torch.isfinite(out[1]).all()
    s = Setup([7, 150], [20, 300], 4, 2, 64, torch.float16, int8, seed=15)
    s.lens = torch.tensor([3, 100], dtype=torch.int32, device=DEV)   # the first 4 and 50 rows are before position 0
    out, lse = s.run(return_lse=True)
    for lo, hi in ((0, 4), (7, 57)):
        assert (out[lo:hi] == 0).all() and torch.isinf(lse[lo:hi]).all()
    assert torch.isfinite(out).all() and torch.isfinite(lse[4:7]).all() and torch.isfinite(lse[57:]).all()
    q = randn(3, 4, 64, dtype=torch.float16)
    out = A.paged_attention(q[:0], *s.pools, s.table[:0], s.lens[:0], k_scale=s.scale[0], v_scale=s.scale[1])
    assert out.shape == (0, 4, 64)


def test_attention_extreme_scores():
    """Scores far apart and all alike; one key that outweighs the rest by e^200 appears late."""
    s = Setup([1, 130], [600, 600], 8, 2, 128, torch.bfloat16, page=64, seed=16)
    k = s.pools[0]
    for b in range(2):
        page, off = s.table[b, 500 // 64].long(), 500 % 64
        k[page, :, off] = 0
        k[page, :, off, 0] = 30.0
    s.q[..., 0] = 8.0
    s.check(s.run(scale=1.0), scale=1.0)
    s.q.zero_()
    s.check(s.run())


def test_attention_strided_queries_and_streams():
    s = Setup([1, 60], [200, 320], 8, 2, 64, torch.float16, seed=17)
    want = s.run()
    wide = randn(61, 3 * 8 * 64 + 1, dtype=torch.float16, seed=18)
    for view in (wide[:, 512:1024].unflatten(1, (8, 64)), wide[:, 1:513].unflatten(1, (8, 64)),
                 torch.empty(8, 61, 64, dtype=torch.float16, device=DEV).transpose(0, 1)):
        view.copy_(s.q)
        got = A.paged_attention(view, *s.pools, s.table, s.lens, s.starts)
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_attention_in_a_graph_follows_lengths():
    """A captured decode step reads lens and the table at replay."""
    s = Setup([1, 1], [900, 64], 16, 2, 256, torch.bfloat16, page=64, seed=19)
    s.run(starts=None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.run(starts=None)
    for lens in ([900, 64], [1, 33], [512, 7]):
        s.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        s.lens_list = lens
        graph.replay()
        s.check(out)


def test_attention_same_result_every_time():
    s = Setup([1, 1, 1], [5000, 64, 777], 16, 2, 256, torch.bfloat16, page=64, seed=20)
    c = Setup([40, 300], [3000, 300], 8, 2, 128, torch.float16, True, page=32, seed=21)
    first = s.run(starts=None), c.run()
    for _ in range(3):
        assert torch.equal(s.run(starts=None), first[0]) and torch.equal(c.run(), first[1])


def test_pool_rows_past_32_bits():
    """A pool of more than 2^32 bytes and 2^31 elements: the last pages are the ones in use."""
    pages, h, page, d = 70000, 2, 64, 256
    if torch.cuda.mem_get_info()[0] < 3 * pages * h * page * d * 2:
        pytest.skip("needs 14 GB of device memory")
    pools = [torch.empty(pages, h, page, d, dtype=torch.float16, device=DEV) for _ in range(2)]
    lens = torch.tensor([100], dtype=torch.int32, device=DEV)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=DEV)
    k, v = randn(100, h, d, dtype=torch.float16, seed=22), randn(100, h, d, dtype=torch.float16, seed=23)
    starts = torch.tensor([0, 100], dtype=torch.int32, device=DEV)
    A.cache_write(k, v, *pools, table, lens, starts)
    assert torch.equal(pools[0][pages - 1].transpose(0, 1), k[:64])
    rk, rv = A.cache_read(*pools, table, starts, 100)
    assert torch.equal(rk, k) and torch.equal(rv, v)
    for n in (1, 100):
        q = randn(n, 4, d, dtype=torch.float16, seed=24)
        want, _ = attend64(q, k.double(), v.double(), torch.arange(100 - n, 100, device=DEV), d ** -0.5, True, 0)
        got = A.paged_attention(q, *pools, table, lens, None if n == 1 else starts)
        assert ((got.double() - want).abs() <= 2.0 ** -10 * v.abs().max()).all()


# ------------------------------------------------------------------------------------- refusals
def test_refusals():
    s = Setup([1, 2], [20, 30], 4, 2, 64, torch.float16, seed=25)
    kp, vp = s.pools
    f = A.rope_frequencies(64)[0].to(DEV)
    pos = torch.arange(3, device=DEV)
    k = randn(3, 2, 64, dtype=torch.float16)

    def attn(**kw):
        a = dict(q=s.q, k_pages=kp, v_pages=vp, table=s.table, lens=s.lens, starts=s.starts) | kw
        return A.paged_attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), a.pop("table"), a.pop("lens"), a.pop("starts"), **a)

    bad = [lambda: attn(q=s.q.float()), lambda: attn(q=s.q.bfloat16()), lambda: attn(q=s.q[:, :3]), lambda: attn(q=s.q[0]),
           lambda: attn(q=s.q.cpu()), lambda: attn(lens=s.lens.long()), lambda: attn(lens=s.lens[:1]),
           lambda: attn(starts=None), lambda: attn(starts=s.starts[:-1]), lambda: attn(table=s.table.long()),
           lambda: attn(k_pages=kp[:, :, :12].contiguous(), v_pages=vp[:, :, :12].contiguous()),
           lambda: attn(k_pages=kp[..., :32], v_pages=vp[..., :32]), lambda: attn(v_pages=vp[:, :1].contiguous()),
           lambda: attn(k_pages=kp.to(torch.int8), v_pages=vp.to(torch.int8)), lambda: attn(window=-1),
           lambda: attn(k_scale=kp[..., 0].float().contiguous(), v_scale=vp[..., 0].float().contiguous()),
           lambda: attn(k_pages=kp.float(), v_pages=vp.float()), lambda: attn(max_len=-1),
           lambda: A.rotary(k, None, pos[:2], f), lambda: A.rotary(k, None, pos.float(), f),
           lambda: A.rotary(k, None, pos, f.half()), lambda: A.rotary(k[..., :32], None, pos, f),
           lambda: A.rotary(k.float(), None, pos, f), lambda: A.rotary(k, k[:2], pos, f),
           lambda: A.rotary(k[..., :24].contiguous(), None, pos, f[:4]),
           lambda: A.cache_write(k, k[:, :1], kp, vp, s.table, s.lens, s.starts),
           lambda: A.cache_write(k, k, kp, vp, s.table, s.lens), lambda: A.cache_write(k.bfloat16(), k.bfloat16(), kp, vp, s.table, s.lens, s.starts),
           lambda: A.cache_write(k[..., :32], k[..., :32], kp, vp, s.table, s.lens, s.starts),
           lambda: A.cache_read(kp, vp, s.table, s.starts, 3, dtype=torch.bfloat16),
           lambda: A.cache_read(kp, vp, s.table, s.starts.long(), 3), lambda: A.cache_read(kp.cpu(), vp.cpu(), s.table, s.starts, 3)]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {n} was accepted")
