"""Rotary, the paged cache and attention at the edges of what a caller may pass: bounds that are too
small, tables that share rows, scales of 0 and below, tokens of no sequence, values far apart in size.

Bounds as in test_attention_gpu.py: outputs round once to 16 bits (u), the softmax weights once more."""
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
