"""A 4-bit cache's numbers to the last bit where the definition gives them, and attention over it where it adds up many keys, or
weights and values of very different sizes, against 64 bits."""
import math

import pytest
import torch

from compressai_b200 import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def pools_of(codes, scale, factor):
    """A pool and its scales from codes [pages, heads, page, D] (-7..7), scales [pages, heads, page] (fp32), factors [.., groups]."""
    pages, heads, page, d = codes.shape
    c = (codes + 8).to(torch.uint8)
    pool = c[..., 1::2] << 4 | c[..., 0::2]
    scales = torch.empty(pages, heads, page // 16, 4 + factor.shape[-1], 16, dtype=torch.uint8, device=DEV)
    scales[..., :4, :] = scale.float().view(torch.uint8).view(pages, heads, page // 16, 4, 16)
    f = factor.float().to(torch.float8_e4m3fn).view(torch.uint8).view(pages, heads, page // 16, 16, -1)
    scales[..., 4:, :] = f.transpose(-1, -2)
    return pool.contiguous(), scales


@pytest.mark.parametrize("L,seqs,new,d", [(131072, 224, 1, 64), (131072, 224, 2, 128), (40000, 450, 1, 256), (131072, 2, 100, 64)])
def test_sums_over_many_keys(L, seqs, new, d):
    """Queries of zeros: all keys weigh the same, the output is the values' mean, small beside them. All sequences are on the same
    pages, as many pairs as blocks, so that a warp adds up a quarter of a sequence. A weight, 2^7 times the row's scale over
    a power of two, has 11 bits: exact in fp16. What is left is the output's rounding (2^-11 of it and 2^-25) and the sums: L / 16 matrix
    instructions at most, each off by 2^-22 of the largest number in it, a partial sum. Sums of any of the keys stay below 6
    standard deviations of a sum of all of them; 1.2 for values that are added beside 16 times as large ones."""
    heads, page = 2, 256
    g = gen(d)
    pages = -(-L // page)
    shape = (pages, heads, page)
    codes = [torch.randint(-7, 8, (*shape, d), generator=g, device=DEV, dtype=torch.int8) for _ in range(2)]
    scale = [1 + torch.randint(0, 1024, shape, generator=g, device=DEV) / 1024 for _ in range(2)]
    ones = torch.ones(*shape, -(-d // 64), device=DEV)
    (kp, ks), (vp, vs) = (pools_of(c, s, ones) for c, s in zip(codes, scale))
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)[None].expand(seqs, -1)
    lens = torch.full((seqs,), L, dtype=torch.int32, device=DEV)
    starts = torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device=DEV)
    q = torch.zeros(seqs * new, heads, d, dtype=torch.float16, device=DEV)
    got = A.paged_attention(q, kp, vp, table, lens, starts, k_scale=ks, v_scale=vs, causal=False, max_new=new, max_len=L)
    there = (torch.arange(page, device=DEV)[None] + page * torch.argsort(table[0])[:, None]) < L
    v = codes[1].double() * (scale[1].double() * there[:, None])[..., None]
    want = v.sum((0, 2)) / L
    sums = L / 16 * 2.0 ** -22 * 1.2 * 6 * v.square().mean().sqrt().item() * math.sqrt(L) / L
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -25 + sums
    assert sums < 0.05 * want.abs().max()   # the bound says something
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max().item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 3, 100])
@pytest.mark.parametrize("d,factors", [(128, [0, 8]), (128, [9, 0]), (256, [0, 4, 6, 9]), (96, [2, 7])])
@pytest.mark.parametrize("less,at", [(11, 0), (17, 0), (19, 2740)])
def test_groups_far_below_their_rows_largest(dtype, new, d, factors, less, at):
    """Values whose group has a factor of 2^-factors[g], and eight keys without a value, 32 apart, that outweigh each other one by
    2^less: what is left of a group is its own, and as exact as the others. Enough sequences (on the same pages) that each has blocks
    of its own, whose warps see such a key each. All values are positive, so that a sum of weights times values is the output:
    a weight, 2^7 times 2^-less times the row's scale over a power of two, is a normal fp16 number and rounds by 2^-11 of itself;
    the output by its type's half step (and half of fp16's smallest number, 2^-25); scores are sums of 15 numbers times 1 at most, off by 2^-20 of 15
    steps (0.25 here, times q of 4 log 2: less than 2^-16 a score, twice that of a weight), the tensor core's 3000 / 16 additions by 2^-22 each, all else in 32 bits: 2e-4 together."""
    L, heads, hq, page = 3000, 2, 4, 32
    g = gen(d + less)
    pages = -(-L // page)
    shape = (pages, heads, page)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    k, v = torch.zeros(*shape, d, dtype=torch.int8, device=DEV), torch.randint(1, 8, (*shape, d), generator=g, device=DEV, dtype=torch.int8)
    k[..., 1:] = torch.randint(-7, 8, (*shape, d - 1), generator=g, device=DEV, dtype=torch.int8)
    heavy = (at // page + torch.arange(8, device=DEV), slice(None), at % page)   # a row of eight pages
    k[*heavy, 0] = 4      # times 0.25 and q: a score of less * log 2
    v_scale = torch.tensor([16 * 1.3, 16 * 1.9], device=DEV)[None, :, None].repeat(pages, 1, page)   # roundings that do not average out
    v_scale[heavy] = 0
    f = torch.tensor([2.0 ** -e for e in factors], device=DEV).expand(*shape, -1)
    kp, ks = pools_of(k, torch.full(shape, 0.25, device=DEV), torch.ones(*shape, len(factors), device=DEV))
    vp, vs = pools_of(v, v_scale, f)
    seqs = 2 if new == 100 else 225
    q = torch.zeros(seqs * new, hq, d, dtype=dtype, device=DEV)
    q[..., 0] = less
    lens, starts = torch.full((seqs,), L, dtype=torch.int32, device=DEV), torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device=DEV)
    got = A.paged_attention(q, kp, vp, table.expand(seqs, -1), lens, starts, k_scale=ks, v_scale=vs, scale=math.log(2.0), causal=False, max_new=new)
    v64 = v.double() * v_scale.double()[..., None] * f.double().repeat_interleave(64, -1)[..., :d]
    w = torch.full((pages, page), 2.0 ** -less, dtype=torch.float64, device=DEV)
    w.view(-1)[L:] = 0
    w[heavy[0], heavy[2]] = 1
    want = torch.einsum("np,nhpd->hd", w, v64) / w.sum()
    want = want.repeat_interleave(hq // heads, 0)
    eps = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    tol = (eps + 2.0 ** -11 + 2e-4) * want + 2.0 ** -25
    assert ((got.double() - want).abs() <= tol).all(), (((got.double() - want).abs() / want).amax((0, 1)), less)


def write_rows(x, page, **kw):
    """Rows x [T, 1, D] written as K and V of one sequence: the pools with their scales, and what cache_read needs."""
    T, _, d = x.shape
    n = -(-T // page)
    pools = [A.empty_pool(n, 1, page, d, torch.int4) for _ in range(2)]
    table = torch.arange(n, dtype=torch.int32, device=DEV)[None]
    lens, starts = torch.tensor([T], dtype=torch.int32, device=DEV), torch.tensor([0, T], dtype=torch.int32, device=DEV)
    A.cache_write(x, x, pools[0][0], pools[1][0], table, lens, starts, k_scale=pools[0][1], v_scale=pools[1][1], **kw)
    return pools, table, starts


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("turned,every", [(False, 1), (True, 1), (True, 300)])
def test_scales_are_a_seventh_rounded_once(dtype, turned, every):
    """Of every 16-bit number from 1e-30 on, by each kernel that writes (few tokens and many are turned by two). V's rows are never turned."""
    top = torch.arange(0x7f80 if dtype == torch.bfloat16 else 0x7c00, device=DEV).to(torch.int16).view(dtype)
    top = top[top.float() >= 1e-30][::every]
    x = torch.zeros(top.numel(), 1, 32, dtype=dtype, device=DEV)
    x[torch.arange(top.numel(), device=DEV), 0, torch.arange(top.numel(), device=DEV) % 32] = -top
    pools, _, _ = write_rows(x, 64, **(dict(inv_freq=A.rope_frequencies(32)[0].to(DEV)) if turned else {}))
    for _, scales in pools[turned:]:
        got = scales[..., :4, :].flatten(-2).contiguous().view(torch.float32).flatten()[: top.numel()]
        assert torch.equal(got, (top.double() / 7).float())   # no quotient by 7 is near enough to a tie of 32 bits for the rounding to 64 to matter


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,d", [(1, 32), (3, 96), (2, 256)])
def test_read_back_rows_and_missing_ones(dtype, heads, d):
    """Rows that the table names are theirs; a page that does not exist and tokens of no sequence give zeros without a sign."""
    g, page = gen(d), 16
    codes = [torch.randint(-7, 8, (4, heads, page, d), generator=g, device=DEV, dtype=torch.int8) for _ in range(2)]
    scale = [torch.rand(4, heads, page, generator=g, device=DEV) for _ in range(2)]
    factor = [2.0 ** -torch.randint(0, 9, (4, heads, page, -(-d // 64)), generator=g, device=DEV).float() for _ in range(2)]
    (kp, ks), (vp, vs) = (pools_of(c, s, f) for c, s, f in zip(codes, scale, factor))
    table = torch.tensor([[3, -1, 0], [4, 2, 1]], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 37, 37 + 25], dtype=torch.int32, device=DEV)
    back = A.cache_read(kp, vp, table, starts, 70, k_scale=ks, v_scale=vs, dtype=dtype)
    eps = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    for got, c, s, f in zip(back, codes, scale, factor):
        x = (c.double() * s.double()[..., None] * f.double().repeat_interleave(64, -1)[..., :d]).transpose(1, 2)   # [page, row, head, D]
        want = torch.zeros(70, heads, d, dtype=torch.float64, device=DEV)
        want[:16], want[32:37], want[53:62] = x[3], x[0, :5], x[2, :9]
        assert ((got.double() - want).abs() <= eps * (1 + 2.0 ** -10) * want.abs() + 2.0 ** -25).all()
        there = torch.zeros(70, dtype=torch.bool, device=DEV)
        there[:16] = there[32:37] = there[53:62] = True
        assert (got[~there].view(torch.int16) == 0).all()
