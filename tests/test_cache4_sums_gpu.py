"""Attention over a 4-bit cache where it adds up many keys, or weights and values of very different sizes, against 64 bits."""
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
