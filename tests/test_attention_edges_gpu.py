"""Rotary, the paged cache and attention at the edges of what a caller may pass: bounds that are too
small, tables that share rows, scales of 0 and below, tokens of no sequence, values far apart in size.

Bounds as in test_attention_gpu.py: outputs round once to 16 bits (u), the softmax weights once more."""
import math

import pytest
import torch

from compressai_b200 import attention as A
from test_attention_gpu import DEV, EPS, Setup, attend64, cache64, randn

pytestmark = pytest.mark.gpu


def rows64(s, b, keys, causal=True, window=0):
    """Sequence b's new tokens over its first `keys` keys, in 64 bits: (out, lse, values)."""
    n, l = s.news[b], s.lens_list[b]
    k, v = (cache64(p, x, s.table, b, keys) for p, x in zip(s.pools, s.scale))
    at = sum(s.news[:b])
    out, lse = attend64(s.q[at:at + n], k, v, torch.arange(l - n, l, device=DEV), s.q.shape[2] ** -0.5, causal, window)
    return out, lse, v


@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 64), (8, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("window", [0, 30])
def test_lengths_past_max_len_over_int8(hq, hkv, d, window):
    """A length beyond the bound that the launch was made with (a replayed graph's, say): the keys that the fp16 copy
    of the cache holds, 128 here, and nothing beyond it; the other sequences as ever."""
    s = Setup([20, 20, 20], [100, 200, 90], hq, hkv, d, torch.float16, int8=True, page=16, seed=50)
    out, lse = s.run(max_new=20, max_len=100, window=window, return_lse=True)
    for b, keys in enumerate((100, 128, 90)):
        want, want_lse, v = rows64(s, b, keys, window=window)
        got, have = out[20 * b:20 * b + 20].double(), lse[20 * b:20 * b + 20].double()
        assert ((got - want).abs() <= (EPS[s.dtype] + 2e-5) * v.abs().max() + EPS[s.dtype] * want.abs()).all()
        seen = ~torch.isinf(want_lse)
        assert torch.equal(torch.isinf(have), ~seen) and ((have - want_lse).abs()[seen] <= 1e-4).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new", [1, 60])
def test_tables_whose_rows_overlap(int8, new):
    """Sequences on the same pages (one row expanded, with a second row elsewhere in memory behind it), rows that
    start one page later each, one column of a wider table: as with a copy of the table."""
    s = Setup([200], [200], 4, 2, 64, torch.float16, int8, page=16, seed=51, spare=6)
    pool = s.pools[0].shape[0]
    flat = torch.cat([s.table[0, :13], torch.arange(30, device=DEV, dtype=torch.int32) % pool])   # what follows names pages too
    lens = torch.tensor([200, 77, 160], dtype=torch.int32, device=DEV)
    q = randn(3 * new, 4, 64, dtype=torch.float16, seed=52)
    starts = None if new == 1 else torch.tensor([0, new, 2 * new, 3 * new], dtype=torch.int32, device=DEV)
    ends = torch.tensor([0, 90, 100, 180], dtype=torch.int32, device=DEV)
    kw = dict(k_scale=s.scale[0], v_scale=s.scale[1])
    zeroed = [p.masked_fill(p != p, 0) for p in s.pools]   # rows past 200 are in some of these sequences
    if int8:
        kw = {n: x.masked_fill(x != x, 0) for n, x in kw.items()}
    for table in (flat[:13].expand(3, 13), flat.as_strided((3, 13), (1, 1)), flat.as_strided((3, 13), (7, 1))):
        want, got = (A.paged_attention(q, *zeroed, t, lens, starts, **kw) for t in (table.contiguous(), table))
        assert torch.equal(want, got) and torch.isfinite(got).all()
        want, got = (A.cache_read(*zeroed, t, ends, 180, dtype=torch.float16, **kw) for t in (table.contiguous(), table))
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    k, v = randn(3, 2, 64, dtype=torch.float16, seed=53), randn(3, 2, 64, dtype=torch.float16, seed=54)
    written = []
    for table in (flat[:13].expand(3, 13).contiguous(), flat[:13].expand(3, 13)):
        pools, sc = [p.clone() for p in zeroed], [None if x is None else x.clone() for x in (kw["k_scale"], kw["v_scale"])]
        A.cache_write(k, v, *pools, table, lens, k_scale=sc[0], v_scale=sc[1])   # positions 199, 76, 159 of the same pages
        written.append(pools + [x for x in sc if x is not None])
    assert all(torch.equal(a, b) for a, b in zip(*written))
    short = torch.tensor([9, 16, 3], dtype=torch.int32, device=DEV)
    table = flat[:39].view(3, 13)[:, 4:5]
    want, got = (A.paged_attention(q[:3], *zeroed, t, short, **kw) for t in (table.contiguous(), table))
    assert torch.equal(want, got)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.2, 1e-44])
def test_scales_of_zero_and_below(int8, dtype, d, scale):
    """Uniform weights, and scores turned round, for few rows and many, hidden keys among the tiles' keys."""
    few = Setup([1, 3], [1, 333], 4, 2, d, dtype, int8, page=16, seed=55)
    many = Setup([70, 130], [200, 130], 8, 2, d, dtype, int8, page=16, seed=56)
    for s in (few, many):
        out, lse = s.run(scale=scale, return_lse=True)
        s.check(out, lse, scale=scale)
        s.check(s.run(scale=scale, window=40), scale=scale, window=40)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hq,hkv,d,new", [(4, 2, 64, 3), (4, 2, 48, 40), (8, 2, 128, 40), (4, 1, 256, 40)])
def test_tokens_of_no_sequence(int8, hq, hkv, d, new):
    """A step padded in front and behind: zeros and -inf there, the sequences' rows right."""
    s = Setup([new, new - 2], [300, new], hq, hkv, d, torch.bfloat16, int8, page=16, seed=57)
    n, before, after = 2 * new - 2, 5, 900
    q = torch.cat([randn(before, hq, d, seed=58), s.q, randn(after, hq, d, seed=59)])
    torch.full((before + n + after, hq, d), float("nan"), dtype=torch.bfloat16, device=DEV)   # what the allocator hands out next
    kw = dict(k_scale=s.scale[0], v_scale=s.scale[1], max_new=new, return_lse=True)
    out, lse = A.paged_attention(q, *s.pools, s.table, s.lens, s.starts + before, **kw)
    s.check(out[before:before + n], lse[before:before + n])
    for part, l in ((out[:before], lse[:before]), (out[before + n:], lse[before + n:])):
        assert (part == 0).all() and (l == -float("inf")).all()
    for nothing in (torch.zeros(3, dtype=torch.int32, device=DEV), torch.full((3,), len(q) + 7, dtype=torch.int32, device=DEV)):
        out, lse = A.paged_attention(q, *s.pools, s.table, s.lens, nothing, **kw)   # two sequences without a token here
        assert (out == 0).all() and (lse == -float("inf")).all()
    out, lse = A.paged_attention(q, *s.pools, s.table[:0], s.lens[:0], s.starts[:1], **kw)   # no sequences
    assert (out == 0).all() and (lse == -float("inf")).all()
    turned = A.cache_write(q[:, :hkv], q[:, :hkv], *s.pools, s.table[:0], s.lens[:0], s.starts[:1], q=q,
                           **{n: kw[n] for n in ("k_scale", "v_scale")})
    assert torch.equal(turned, q)
    back = A.cache_read(*s.pools, s.table[:0], s.starts[:1], 9, **{n: kw[n] for n in ("k_scale", "v_scale")})
    assert all((x == 0).all() and x.shape == (9, hkv, d) for x in back)


def test_a_table_without_columns():
    """Sequences that have no page yet: nothing to see, nothing stored."""
    s = Setup([1, 1], [0, 0], 4, 2, 64, torch.float16, seed=60)
    table = s.table[:, :0].contiguous()
    before = [p.clone() for p in s.pools]
    out, lse = A.paged_attention(s.q, *s.pools, table, s.lens, return_lse=True)
    assert (out == 0).all() and (lse == -float("inf")).all()
    A.cache_write(s.q[:, :2], s.q[:, :2], *s.pools, table, s.lens + 1)
    assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(before, s.pools))


def test_check_status():
    s = Setup([1, 70], [20, 300], 8, 2, 128, torch.bfloat16, seed=61)
    s.run()
    A.check_status()
    A.check_status("cuda:0")


def check_rows(s, out, scale, causal=True, window=0):
    """Every row within its own bound: u * sum p |v| for the weights' rounding and 32-bit work, u |out| for its own."""
    at = 0
    for b, (n, l) in enumerate(zip(s.news, s.lens_list)):
        k, v = (cache64(p, x, s.table, b, l) for p, x in zip(s.pools, s.scale))
        q, pos = s.q[at:at + n], torch.arange(l - n, l, device=DEV)
        want, sizes = (attend64(q, k, y, pos, scale, causal, window)[0] for y in (v, v.abs()))
        off = (out[at:at + n].double() - want).abs()
        assert (off <= (EPS[s.dtype] + 2e-5) * sizes + EPS[s.dtype] * want.abs()).all(), (b, (off / sizes).max().item())
        at += n


@pytest.mark.parametrize("by", [1e4, 1e8, 1e30])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (4, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("new", [4, 70])
def test_int8_values_of_hidden_keys_cost_nothing(by, hq, hkv, d, new):
    """A token with a far larger V row, later than some rows or out of their window: the rows that do not see it are as
    exact as ever."""
    s = Setup([new, 1], [300, 200], hq, hkv, d, torch.float16, int8=True, page=16, seed=62)
    for b, key in ((0, 298), (1, 161)):
        s.scale[1][s.table[b, key // 16].long(), :, key % 16] *= by
    out = s.run(window=30)   # sequence 0: hidden from all rows but the last two; sequence 1: 9 keys before its window
    rows = torch.arange(new - 2)
    s.q, s.news, s.lens_list = torch.cat([s.q[rows], s.q[new:]]), [new - 2, 1], [298, 200]
    check_rows(s, torch.cat([out[rows], out[new:]]), d ** -0.5, window=30)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_small_weights_beside_a_large_one(int8, dtype):
    """One key outweighs each of 200,000 others by 2^26: together they are 0.3 % of the sum, and all of the output."""
    new, h, d, page, keys = 4096, 10, 64, 256, 200_000
    kind = torch.int8 if int8 else dtype
    k = torch.zeros(2, h, page, d, dtype=kind, device=DEV)
    v = torch.full_like(k, 64 if int8 else 1)
    k[0, :, 0, 0] = 104 if int8 else 26
    v[0, :, 0] = 0
    scale = [torch.full((2, h, page), by, device=DEV) for by in (0.25, 2.0 ** -6)] if int8 else [None, None]
    table = torch.ones(1, -(-keys // page), dtype=torch.int32, device=DEV)
    table[0, 0] = 0
    lens = torch.tensor([keys], dtype=torch.int32, device=DEV)
    for n in (new, 1):
        q = torch.zeros(n, h, d, dtype=dtype, device=DEV)
        q[..., 0] = 1
        starts = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        out, lse = A.paged_attention(q, k, v, table, lens, starts, k_scale=scale[0], v_scale=scale[1], scale=math.log(2.0),
                                     causal=False, return_lse=True)
        rest = (keys - 1) * 2.0 ** -26
        want = rest / (1 + rest)
        # weights and output rounded once each, relative to themselves; 1e-3 and 1e-4 for the 32-bit sums of 200,000 terms
        assert ((out.double() - want).abs() <= (2 * EPS[dtype] + 1e-3) * want).all()
        assert ((lse.double() - (26 * math.log(2) + math.log1p(rest))).abs() <= 1e-4).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new", [2, 70])
def test_nothing_cached_at_all(int8, new):
    """New tokens whose sequences have no key and no page, the bound on lengths 0: zeros."""
    s = Setup([new, 1], [0, 0], 4, 2, 64, torch.float16, int8, seed=63)
    for table, kw in ((s.table, dict(max_len=0)), (s.table[:, :0].contiguous(), {})):
        out, lse = A.paged_attention(s.q, *s.pools, table, s.lens, s.starts, k_scale=s.scale[0], v_scale=s.scale[1],
                                     return_lse=True, **kw)
        assert (out == 0).all() and (lse == -float("inf")).all()


def test_the_longest_sequence():
    """2^31 - 256 positions on two pages: the last page, on which all the weight lies, is read."""
    cols, d = (2 ** 31 - 256) // 256, 16
    k = torch.zeros(2, 1, 256, d, dtype=torch.float16, device=DEV)
    v = torch.ones_like(k)
    k[1, :, :, 0], v[1] = 10, 3
    table = torch.zeros(1, cols, dtype=torch.int32, device=DEV)
    table[0, -1] = 1
    q = torch.full((1, 1, d), 4.0, dtype=torch.float16, device=DEV)
    lens = torch.tensor([2 ** 31 - 256], dtype=torch.int32, device=DEV)
    out, lse = A.paged_attention(q, k, v, table, lens, scale=1.0, return_lse=True)
    # e^40 * 256 against 2^31: the rest is 4e-11 of it
    assert (out == 3).all() and abs(lse.item() - 40 - math.log(256)) <= 1e-4
    with pytest.raises(ValueError):
        A.cache_read(k, v, table.new_zeros(1, cols + 1), torch.zeros(2, dtype=torch.int32, device=DEV), 1)


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("size", [1e34, 1e31, 1e-31, 1e-38])
def test_int8_with_queries_of_any_size(size, d, new):
    """bf16 queries from the smallest normal numbers to the largest, the scale set against them."""
    s = Setup([new], [300], 4, 1, d, torch.bfloat16, int8=True, page=16, seed=64)
    s.q = (s.q.float().clamp(-4, 4) * size).bfloat16()
    scale = d ** -0.5 / size
    check_rows(s, s.run(scale=scale), scale)


def test_a_cache_stays_on_its_device():
    """Named without an index, the device is the one that was current when the pools were made."""
    c = A.PagedKVCache(1, 2, 1, 16, page_size=16)
    assert c.device == c.pools[0][0].device == torch.device("cuda", torch.cuda.current_device())
    c.begin([c.add()], [3])
    assert c.batch["table"].device == c.device


@pytest.mark.parametrize("dtype,int8,new", [(torch.float16, False, 4), (torch.bfloat16, False, 2), (torch.float16, True, 12),
                                            (torch.bfloat16, True, 5)])
@pytest.mark.parametrize("hq,hkv,d", [(16, 4, 256), (8, 8, 64), (8, 2, 96), (12, 3, 128)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 21), (False, 0), (False, 40)])
def test_few_new_tokens_of_several_positions(dtype, int8, new, hq, hkv, d, causal, window):
    """Drafts: rows of several tokens in one block of the kernel for few rows (16 rows, over int8 48), ragged."""
    news = [new, 1, 0, max(1, new - 1), new]
    s = Setup(news, [new, 40, 9, 333, 1500], hq, hkv, d, dtype, int8, page=16, seed=65)
    out, lse = s.run(causal=causal, window=window, max_new=new, max_len=1500, return_lse=True)
    s.check(out, lse, causal=causal, window=window)


@pytest.mark.parametrize("window", [0, 50])
def test_int8_with_a_table_too_wide_to_widen(window):
    """Room for more keys than the fp16 copy of an int8 cache may hold (2^30 values): many rows go to the kernel for
    few, as many blocks of them as it takes."""
    s = Setup([150, 1, 40], [700, 333, 40], 8, 2, 256, torch.bfloat16, int8=True, page=256, seed=66)
    wide = torch.full((3, 2800), -1, dtype=torch.int32, device=DEV)   # 3 * 2 * 2800 * 256 * 256 > 2^30
    wide[:, :s.table.shape[1]] = s.table
    s.table = wide
    out, lse = s.run(window=window, return_lse=True)
    s.check(out, lse, window=window)
