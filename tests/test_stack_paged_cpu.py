"""What the paged attention layer refuses before it launches anything (no device needed)."""
from types import SimpleNamespace

import pytest
import torch
import torch.nn as nn

from compressai_b200.attention import PagedKVCache, rope_frequencies
from compressai_b200.stack import PagedAttention, use_paged_attention


class Reached(Exception):
    pass


class Attn(nn.Module):
    """Stands in for the transformers layer: every forward that passes the checks ends at its first projection."""

    def q_proj(self, x):
        raise Reached


def layer(seqs, counts):
    cache = PagedKVCache(1, 8, 1, 16, page_size=16, device="cpu")
    ids = [cache.add() for _ in range(seqs)]
    if counts is not None:
        cache.begin(ids, counts)
    return PagedAttention(Attn(), cache, 0, None), cache, ids


def test_every_forward_needs_a_begin():
    m, cache, ids = layer(2, None)
    x = torch.zeros(2, 5, 8)
    with pytest.raises(RuntimeError, match="begin"):
        m(hidden_states=x)
    cache.begin(ids, [5, 5])
    with pytest.raises(Reached):
        m(hidden_states=x)
    with pytest.raises(RuntimeError, match="begin"):   # would overwrite the rows just written, at the same positions
        m(hidden_states=x)
    cache.begin(ids, [1, 1])
    with pytest.raises(Reached):
        m(hidden_states=x[:, :1])


@pytest.mark.parametrize("counts", [[5, 4], [10], [6, 4], [1, 1]])
def test_tokens_are_the_batch_s(counts):
    m, _, _ = layer(len(counts), counts)
    with pytest.raises(ValueError, match="counted"):
        m(hidden_states=torch.zeros(2, 5, 8))


def masks(q, k, hidden):
    """A causal mask of the last q of k positions, `hidden` keys of the first sequence padding, in every form."""
    m = torch.ones(2, 1, q, k, dtype=torch.bool).tril(k - q)
    m[0, :, :, hidden] = False
    flat = torch.ones(2, k, dtype=torch.long)
    flat[0, hidden] = 0
    return m, torch.zeros(m.shape).masked_fill(~m, float("-inf")), torch.zeros(m.shape).masked_fill(~m, -3e38), flat, flat.bool()


@pytest.mark.parametrize("q,k", [(5, 5), (1, 1), (1, 9), (3, 9)])
def test_padding_masks_are_refused_and_causal_ones_taken(q, k):
    for hidden, error in (([], Reached), ([0], ValueError), ([k - 1], ValueError)):
        for mask in masks(q, k, hidden):
            m, _, _ = layer(2, [q, q])
            with pytest.raises(error):
                m(hidden_states=torch.zeros(2, q, 8), attention_mask=mask)


class Model(nn.Module):
    """As much of a stack as use_paged_attention looks at."""

    def __init__(self, **rope):
        super().__init__()
        self.weight = nn.Parameter(torch.zeros(1))
        self.config = SimpleNamespace(num_key_value_heads=1, head_dim=64,
                                      rope_parameters={"rope_theta": 10000.0, "partial_rotary_factor": 0.25, **rope})
        self.model = nn.Module()
        self.model.layers = nn.ModuleList([nn.Module(), nn.Module()])
        self.model.layers[1].self_attn = Attn()


def test_a_second_cache_takes_the_place_of_the_first():
    m = Model()
    attn = m.model.layers[1].self_attn
    use_paged_attention(m, pages=4)
    cache = use_paged_attention(m, pages=6, page_size=16, dtype=torch.int8)
    layer = m.model.layers[1].self_attn
    assert layer.attn is attn and layer.cache is cache and len(cache.free) == 6 and not hasattr(m.model.layers[0], "self_attn")


def test_stretched_rotary_is_given():
    m = Model(rope_type="yarn", factor=8.0)
    with pytest.raises(ValueError, match="inv_freq"):
        use_paged_attention(m, pages=4)
    assert isinstance(m.model.layers[1].self_attn, Attn)
    f, factor = rope_frequencies(16, 10000.0, {"type": "yarn", "factor": 8.0, "original": 4096})
    use_paged_attention(m, pages=4, inv_freq=f, factor=factor)
    layer = m.model.layers[1].self_attn
    assert torch.equal(layer.inv_freq, f) and layer.factor == factor != 1.0
    use_paged_attention(Model(), pages=4)
