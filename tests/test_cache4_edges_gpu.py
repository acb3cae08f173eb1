"""A 4-bit cache at its edges: scales and sizes, tables, lengths and strides that a program may hand over."""
import math

import pytest
import torch

from compressai_b200 import attention as A
from test_cache4_gpu import DEV, EPS, Setup, attend64, awkward, fill, gen, one_sequence, pack64, parts, stored, values64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.2, 1e-44])
def test_scales_of_zero_and_below(dtype, d, scale):
    """Uniform weights, and scores turned round, for few rows and many, hidden keys among the tiles' keys."""
    few = Setup([1, 3], [1, 333], 4, 2, d, dtype, page=16, seed=55)
    many = Setup([70, 130], [200, 130], 8, 2, d, dtype, page=16, seed=56)
    for s in (few, many):
        out, lse = s.run(scale=scale, return_lse=True)
        s.check(out, lse, scale=scale)
        s.check(s.run(scale=scale, window=40), scale=scale, window=40)


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("size", [1e34, 1e31, 1e-31, 1e-38])
def test_queries_of_any_size(size, d, new):
    """bf16 queries from the smallest normal numbers to the largest, the scale set against them."""
    s = Setup([new], [300], 4, 1, d, torch.bfloat16, page=16, seed=64)
    s.q = (s.q.float().clamp(-4, 4) * size).bfloat16()
    s.check(s.run(scale=d ** -0.5 / size), scale=d ** -0.5 / size)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_small_weights_beside_a_large_one(dtype):
    """One key outweighs each of 200,000 others by 2^26: together they are 0.3 % of the sum, and all of the output."""
    new, h, d, page, keys = 4096, 10, 64, 256, 200_000
    x = torch.zeros(2, h, page, d, device=DEV)
    x[0, :, 0, 0] = 26
    v = torch.full((2, h, page, d), 7 / 64, device=DEV)   # a scale of 2^-6
    v[0, :, 0] = 0
    pools = [A.empty_pool(2, h, page, d, torch.int4) for _ in range(2)]
    for (pool, scales), y in zip(pools, (x, v)):
        fill(pool, scales, y.to(torch.bfloat16))
    k64 = values64(*pools[0])
    table = torch.ones(1, -(-keys // page), dtype=torch.int32, device=DEV)
    table[0, 0] = 0
    lens = torch.tensor([keys], dtype=torch.int32, device=DEV)
    top = k64[0, 0, 0, 0].item()
    rest = (keys - 1) * 2.0 ** -top
    want = 7 / 64 * rest / (1 + rest)
    for n in (new, 1):
        q = torch.zeros(n, h, d, dtype=dtype, device=DEV)
        q[..., 0] = 1
        starts = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        out, lse = A.paged_attention(q, pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1],
                                     scale=math.log(2.0), causal=False, return_lse=True)
        # weights (twice) and output rounded relative to themselves; 1e-3 and 1e-4 for the 32-bit sums of 200,000 terms
        assert ((out.double() - want).abs() <= (2 * EPS[dtype] + 1e-3) * want).all()
        assert ((lse.double() - (top * math.log(2) + math.log1p(rest))).abs() <= 1e-4).all()


@pytest.mark.parametrize("by", [2.0 ** 13, 2.0 ** 27, 2.0 ** 100])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (4, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("new", [4, 70])
def test_values_of_hidden_keys_cost_nothing(by, hq, hkv, d, new):
    """A token with a far larger V row, later than some rows or out of their window: the rows that do not see it are as
    exact as ever."""
    s = Setup([new, 1], [300, 200], hq, hkv, d, torch.float16, page=16, seed=62)
    for b, key in ((0, 298), (1, 161)):
        page = s.table[b, key // 16].long()
        x = s.scales[1][page, :, 0, :4].reshape(hkv, 64).clone().view(torch.float32)   # the page's 16 scales
        x[:, key % 16] *= by
        s.scales[1][page, :, 0, :4] = x.view(torch.uint8).view(hkv, 4, 16)
    out = s.run(window=30)   # sequence 0: hidden from all rows but the last two; sequence 1: 9 keys before its window
    rows = torch.arange(new - 2)
    for b, (at, n, l) in enumerate(((0, new - 2, 298), (new, 1, 200))):
        k, v = s.rows64(0, b, l), s.rows64(1, b, l)
        if b == 1:
            v[161] = 0   # not seen
        want, _ = attend64(s.q[at:at + n], k, v, torch.arange(l - n, l, device=DEV), d ** -0.5, True, 30)
        tol = (2.0 ** -10 + 3e-4) * v.abs().max() + EPS[torch.float16] * want.abs()
        assert ((out[at:at + n].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("new", [2, 70])
def test_nothing_cached_at_all(new):
    """New tokens whose sequences have no key and no page, the bound on lengths 0: zeros."""
    s = Setup([new, 1], [0, 0], 4, 2, 64, torch.float16, seed=63)
    for table, kw in ((s.table, dict(max_len=0)), (s.table[:, :0].contiguous(), {})):
        out, lse = A.paged_attention(s.q, *s.pools, table, s.lens, s.starts, k_scale=s.scales[0], v_scale=s.scales[1],
                                     return_lse=True, **kw)
        assert (out == 0).all() and (lse == -float("inf")).all()


def test_no_sequence_and_no_token():
    s = Setup([1], [5], 4, 2, 64, torch.float16)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    kw = dict(k_scale=s.scales[0], v_scale=s.scales[1])
    out = A.paged_attention(s.q[:0], *s.pools, s.table[:0], none, **kw)
    assert out.shape == (0, 4, 64)
    starts = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = A.paged_attention(s.q, *s.pools, s.table[:0], none, starts, **kw)
    assert (out == 0).all()
    assert A.cache_write(s.q[:0, :2], s.q[:0, :2], *s.pools, s.table[:0], none, **kw) is None
    k, v = A.cache_read(*s.pools, s.table[:0], starts, 3, **kw)
    assert (k == 0).all() and (v == 0).all()


def test_the_longest_sequence():
    """2^31 - 256 positions on two pages: the last page, on which all the weight lies, is read."""
    cols, d = (2 ** 31 - 256) // 256, 32
    x, y = torch.zeros(2, 1, 256, d, device=DEV), torch.ones(2, 1, 256, d, device=DEV)
    x[1, :, :, 0], y[1] = 10, 3
    pools = [A.empty_pool(2, 1, 256, d, torch.int4) for _ in range(2)]
    for (pool, scales), z in zip(pools, (x, y)):
        fill(pool, scales, z.half())
    table = torch.zeros(1, cols, dtype=torch.int32, device=DEV)
    table[0, -1] = 1
    q = torch.full((1, 1, d), 4.0, dtype=torch.float16, device=DEV)
    lens = torch.tensor([2 ** 31 - 256], dtype=torch.int32, device=DEV)
    out, lse = A.paged_attention(q, pools[0][0], pools[1][0], table, lens, k_scale=pools[0][1], v_scale=pools[1][1], scale=1.0,
                                 return_lse=True)
    # e^40 * 256 against 2^31: the rest is 4e-11 of it; 10 and 3 are off by 2^-23
    assert (out == 3).all() and abs(lse.item() - 40 - math.log(256)) <= 1e-4


@pytest.mark.parametrize("new", [1, 60])
def test_tables_whose_rows_overlap(new):
    """Sequences on the same pages, rows that start one page later each, one column of a wider table: as with a copy."""
    s = Setup([200], [200], 4, 2, 64, torch.float16, page=16, seed=51, spare=6)
    for pool, scales in zip(s.pools, s.scales):
        fill(pool, scales, torch.randn(pool.shape[0], 2, 16, 64, generator=gen(1), device=DEV).half())
    n = s.pools[0].shape[0]
    flat = torch.cat([s.table[0, :13], torch.arange(30, device=DEV, dtype=torch.int32) % n])
    lens = torch.tensor([200, 77, 160], dtype=torch.int32, device=DEV)
    q = torch.randn(3 * new, 4, 64, generator=gen(52), device=DEV).half()
    starts = None if new == 1 else torch.tensor([0, new, 2 * new, 3 * new], dtype=torch.int32, device=DEV)
    ends = torch.tensor([0, 90, 100, 180], dtype=torch.int32, device=DEV)
    kw = dict(k_scale=s.scales[0], v_scale=s.scales[1])
    for table in (flat[:13].expand(3, 13), flat.as_strided((3, 13), (1, 1)), flat.as_strided((3, 13), (7, 1))):
        want, got = (A.paged_attention(q, *s.pools, t, lens, starts, **kw) for t in (table.contiguous(), table))
        assert torch.equal(want, got) and torch.isfinite(got).all()
        want, got = (A.cache_read(*s.pools, t, ends, 180, **kw) for t in (table.contiguous(), table))
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("window", [0, 50])
def test_a_table_too_wide_to_widen(window):
    """Room for more keys than the fp16 copy may hold (2^30 values): many rows go to the kernel for few, in many blocks of rows."""
    s = Setup([150, 1, 40], [700, 333, 40], 8, 2, 256, torch.bfloat16, page=256, seed=66)
    wide = torch.full((3, 2800), -1, dtype=torch.int32, device=DEV)   # 3 * 2 * 2800 * 256 * 256 > 2^30
    wide[:, :s.table.shape[1]] = s.table
    s.table = wide
    out, lse = s.run(window=window, return_lse=True)
    s.check(out, lse, window=window)


@pytest.mark.parametrize("new", [1, 5])
def test_lengths_past_max_len(new):
    """A length beyond the bound that the launch was made with (a replayed graph's): still all of its keys."""
    s = Setup([new] * 3, [100, 5000, 90], 4, 2, 128, torch.float16, page=16, seed=50)
    out, lse = s.run(max_new=new, max_len=100, return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("seqs", [130, 700])
def test_many_sequences(seqs):
    """More than the block's threads: each counts several, ragged, some of them empty and some without new tokens."""
    lens = [(37 * i * i) % 400 for i in range(seqs)]
    news = [min(l, (i % 3)) for i, l in enumerate(lens)]
    s = Setup(news, lens, 4, 2, 64, torch.float16, page=16, seed=7)
    out, lse = s.run(max_new=2, max_len=400, return_lse=True)
    s.check(out, lse)


def test_starts_that_are_no_starts_stay_in_range():
    """Descending, negative and far ones: nothing is read or written out of range, and the next call is right."""
    s = Setup([3, 3], [40, 900], 4, 2, 64, torch.float16, page=16, seed=8)
    for bad in ([5, 2, -7], [-100, 3, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 4]):
        starts = torch.tensor(bad, dtype=torch.int32, device=DEV)
        for kw in ({}, dict(max_new=3, max_len=900)):
            s.run(starts=starts, **kw)
        A.cache_write(s.q[:, :2], s.q[:, :2], *[p.clone() for p in s.pools], s.table, s.lens, starts,
                      k_scale=s.scales[0].clone(), v_scale=s.scales[1].clone())
        A.cache_read(*s.pools, s.table, starts, 50, k_scale=s.scales[0], v_scale=s.scales[1])
    s.check(s.run())


@pytest.mark.parametrize("shift,wide", [(0, 0), (8, 0), (8, 8), (1, 3), (16, 16)])
@pytest.mark.parametrize("T", [1, 40])
def test_strides_and_alignment_of_what_is_written(shift, wide, T):
    d, heads = 96, 3
    base = torch.randn(2, T, heads, d + wide + shift, generator=gen(3), device=DEV).to(torch.bfloat16)
    k, v = base[0, ..., shift:shift + d], base[1, ..., shift:shift + d]
    pools, table, lens, starts = one_sequence(T, heads, d, 32)
    kw = dict(k_scale=pools[0][1], v_scale=pools[1][1])
    A.cache_write(k, v, pools[0][0], pools[1][0], table, lens, starts, **kw)
    for x, (pool, scales) in zip((k, v), pools):
        codes, scale, factor = stored(pool, scales, table, T, 32)
        c, s, f = (t.view(T, heads, *t.shape[1:]) for t in pack64(x.reshape(-1, d)))
        assert torch.equal(codes, c) and torch.equal(factor, f)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [3, 3000])
def test_queries_beside_keys_that_are_not_turned(dtype, T):
    """With q and without frequencies q comes back as it is, and the rows are those of a write without q."""
    d = 128
    q, k, v = (awkward(torch.randn(T, h, d, generator=gen(h), device=DEV).to(dtype)) for h in (4, 2, 2))
    got = []
    for with_q in (None, q):
        pools, table, lens, starts = one_sequence(T, 2, d, 16)
        for pool, scales in pools:
            pool.zero_()
            scales.zero_()
        back = A.cache_write(k, v, pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1], q=with_q)
        assert with_q is None or torch.equal(back.view(torch.int16), q.view(torch.int16))
        got.append([x for p in pools for x in p])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_refusals():
    s = Setup([1, 1], [20, 30], 4, 2, 64, torch.float16)
    kw = dict(k_scale=s.scales[0], v_scale=s.scales[1])
    k = torch.zeros(2, 2, 64, dtype=torch.float16, device=DEV)
    bad = [dict(k_scale=None, v_scale=None), dict(kw, k_scale=s.scales[0].float()), dict(kw, v_scale=s.scales[1][..., :4, :]),
           dict(kw, k_scale=s.scales[0].transpose(-1, -2)), dict(kw, k_scale=torch.zeros(s.pools[0].shape[:3], device=DEV)),
           dict(kw, k_scale=s.scales[0].cpu())]
    for b in bad:
        with pytest.raises(ValueError):
            A.paged_attention(s.q, *s.pools, s.table, s.lens, **b)
        with pytest.raises(ValueError):
            A.cache_write(k, k, *s.pools, s.table, s.lens, **b)
        with pytest.raises(ValueError):
            A.cache_read(*s.pools, s.table, s.starts, 2, **b)
    for q in (s.q[..., :32], s.q.float(), torch.zeros(2, 3, 64, dtype=torch.float16, device=DEV)):
        with pytest.raises(ValueError):
            A.paged_attention(q, *s.pools, s.table, s.lens, **kw)
    odd = torch.zeros(3, 2, 16, 24, dtype=torch.uint8, device=DEV)   # heads of 48
    scales = torch.zeros(3, 2, 1, 5, 16, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError, match="32"):
        A.cache_read(odd, odd, s.table, s.starts, 2, k_scale=scales, v_scale=scales)
    with pytest.raises(ValueError):
        A.paged_attention(s.q, s.pools[0], s.pools[1].to(torch.int8), s.table, s.lens, **kw)


def test_the_stack_decodes_on_it():
    """Greedy decode of the small stack twice: the same ids, every page back."""
    from compressai_b200 import stack
    from test_stack_paged_gpu import small_model
    model = small_model(5)
    cache = stack.use_paged_attention(model, pages=8, page_size=16, dtype=torch.int4)
    t1, ids1 = stack.decode(model, batch=3, prompt_len=20, steps=3, warmup=1, seed=9, cache=cache)
    t2, ids2 = stack.decode(model, batch=3, prompt_len=20, steps=3, warmup=1, seed=9, cache=cache)
    assert t1 > 0 and torch.equal(ids1, ids2) and len(cache.free) == 8 and not cache.pages


def test_two_graphs_and_an_eager_call_between():
    """Each captured call has workspaces of its own."""
    a, b = (Setup([1] * n, [900] * n, 8, 1, 128, torch.float16, page=64, seed=n) for n in (2, 5))
    graphs, outs = [], []
    for s in (a, b):
        s.run(starts=None, max_len=900)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run(starts=None, max_len=900))
        graphs.append(g)
    for _ in range(3):
        graphs[0].replay()
        eager = b.run(starts=None, max_len=900)
        graphs[1].replay()
    torch.cuda.synchronize()
    a.check(outs[0])
    b.check(outs[1])
    assert torch.equal(eager, outs[1])
    A.check_status()


@pytest.mark.parametrize("off", [0, 16])
def test_a_workspace_on_any_16_bytes(off):
    """The C entry point asks for 16-byte alignment of its workspace, no more."""
    import ctypes

    from compressai_b200 import _lib
    s = Setup([120], [300], 4, 2, 128, torch.float16, page=16, seed=3)
    lib = _lib.load()
    kind, T = _lib.VQ2_I4, 120
    bytes_ = lib.vq2_paged_attention_workspace(T, 4, 2, 128, kind, 1, T, 300, 0)
    ws = torch.empty(bytes_ + 64, dtype=torch.uint8, device=DEV)
    out = torch.empty(T, 4, 128, dtype=torch.float16, device=DEV)
    p = ctypes.c_void_p
    n = s.pools[0].shape[0]
    _lib.check(lib.vq2_paged_attention(
        p(s.q.data_ptr()), 512, 128, _lib.VQ2_F16, T, 4, p(s.pools[0].data_ptr()), p(s.pools[1].data_ptr()), kind,
        p(s.scales[0].data_ptr()), p(s.scales[1].data_ptr()), n, 2, 16, 128, p(s.table.data_ptr()), s.table.stride(0), s.table.shape[1],
        p(s.lens.data_ptr()), p(s.starts.data_ptr()), 1, T, 300, 128 ** -0.5, 1, 0, p(out.data_ptr()), None, p(ws.data_ptr() + off),
        bytes_, p(torch.cuda.current_stream().cuda_stream)), "vq2_paged_attention")
    s.check(out)
