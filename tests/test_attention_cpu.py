"""Rotary frequencies against the published formulas, and the C-ABI's refusals (no device needed)."""
import ctypes
import math

import pytest
import torch

from compressai_b200 import _lib
from compressai_b200 import attention as A


def test_rope_frequencies_plain_and_linear():
    f, factor = A.rope_frequencies(64, 1e6)
    assert factor == 1.0 and f.dtype == torch.float32
    for i in (0, 1, 31):
        assert f[i].item() == pytest.approx(1e6 ** (-2 * i / 64), rel=1e-6)
    g, factor = A.rope_frequencies(64, 1e6, {"type": "linear", "factor": 4.0})
    assert factor == 1.0 and torch.allclose(g * 4, f, rtol=1e-6)


def test_rope_frequencies_yarn():
    rot, theta, by, original = 128, 10000.0, 8.0, 4096
    f, _ = A.rope_frequencies(rot, theta)
    g, factor = A.rope_frequencies(rot, theta, {"type": "yarn", "factor": by, "original": original})
    assert factor == pytest.approx(0.1 * math.log(by) + 1)
    ratio = (f / g).double()
    turns = original * f.double() / (2 * math.pi)
    # a pair more than one index inside either bound is kept, or stretched whole
    assert torch.allclose(ratio[turns > 32 * 1.2], torch.ones((), dtype=torch.float64), rtol=1e-5)
    assert torch.allclose(ratio[turns < 1 / 1.2], torch.full((), by, dtype=torch.float64), rtol=1e-5)
    assert (ratio[1:] >= ratio[:-1] - 1e-6).all()


def test_rope_frequencies_llama3():
    f, _ = A.rope_frequencies(128, 500000.0)
    g, factor = A.rope_frequencies(128, 500000.0, {"type": "llama3", "factor": 8.0, "original": 8192})
    assert factor == 1.0
    for i in range(64):
        wave = 2 * math.pi / f[i].double().item()
        if wave < 8192 / 4:
            want = f[i].item()
        elif wave > 8192:
            want = f[i].item() / 8
        else:
            s = (8192 / wave - 1) / 3
            want = (1 - s) * f[i].item() / 8 + s * f[i].item()
        assert g[i].item() == pytest.approx(want, rel=1e-5)


def test_rope_frequencies_refusals():
    for args in ((3,), (0,), (64, 1e4, {"type": "dynamic", "factor": 2.0}), (64, 1e4, {"type": "linear", "factor": 0.5})):
        with pytest.raises(ValueError):
            A.rope_frequencies(*args)


def test_abi_refusals_without_device():
    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never dereferenced: validation fails first
    odd = ctypes.c_void_p(264)

    def attn(q=p, dtype=1, T=4, hq=4, kp=p, kv_dtype=1, ks=None, pages=8, h=2, page=16, d=64, cols=4, lens=p, starts=p,
             seqs=2, window=0, out=p, stride=256):
        return lib.vq2_paged_attention(q, stride, 64, dtype, T, hq, kp, p, kv_dtype, ks, ks, pages, h, page, d, p, cols, cols,
                                       lens, starts, seqs, 4, 64, 0.125, 1, window, out, None, None, 0, None)
    assert attn(q=None) == _lib.VQ2_ERR_ARG and attn(lens=None) == _lib.VQ2_ERR_ARG and attn(out=None) == _lib.VQ2_ERR_ARG
    assert attn(dtype=2) == _lib.VQ2_ERR_DTYPE and attn(kv_dtype=0) == _lib.VQ2_ERR_DTYPE and attn(kv_dtype=9) == _lib.VQ2_ERR_DTYPE
    assert attn(kv_dtype=3) == _lib.VQ2_ERR_ARG and attn(ks=p) == _lib.VQ2_ERR_ARG   # scales: int8 pools, and only they
    assert attn(d=60) == _lib.VQ2_ERR_SHAPE and attn(d=272) == _lib.VQ2_ERR_SHAPE and attn(page=24) == _lib.VQ2_ERR_SHAPE
    assert attn(hq=3) == _lib.VQ2_ERR_SHAPE and attn(starts=None) == _lib.VQ2_ERR_SHAPE and attn(window=-1) == _lib.VQ2_ERR_SHAPE
    assert attn(pages=1 << 40) == _lib.VQ2_ERR_SHAPE
    assert attn(q=odd) == _lib.VQ2_ERR_ALIGN and attn(kp=odd) == _lib.VQ2_ERR_ALIGN and attn(stride=252) == _lib.VQ2_ERR_ALIGN
    assert attn(T=0, starts=p) == _lib.VQ2_OK

    def rot(q=p, k=None, kh=0, pos=p, f=p, r=64, d=64, dtype=0, T=3, out=p):
        return lib.vq2_rotary(q, 64, 64, 1, k, 64, 64, kh, dtype, T, d, pos, 0, f, r, 0, 1.0, 0, out, None, None)
    assert rot(q=None) == _lib.VQ2_ERR_ARG and rot(kh=1) == _lib.VQ2_ERR_ARG and rot(f=None) == _lib.VQ2_ERR_ARG
    assert rot(r=63) == _lib.VQ2_ERR_SHAPE and rot(r=66) == _lib.VQ2_ERR_SHAPE and rot(d=72) == _lib.VQ2_ERR_SHAPE
    assert rot(dtype=3) == _lib.VQ2_ERR_DTYPE and rot(out=odd) == _lib.VQ2_ERR_ALIGN and rot(T=0) == _lib.VQ2_OK
