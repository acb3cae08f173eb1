"""The decode stack with its full-attention layers on this library's rotary, paged cache and attention,
against the same model with the transformers cache: teacher-forced logits, greedy decode, pages given back."""
import pytest
import torch

from compressai_b200 import stack

pytestmark = pytest.mark.gpu
DEV = "cuda"


def small_model(seed=4):
    from transformers import Qwen3_5MoeTextConfig
    cfg = Qwen3_5MoeTextConfig(hidden_size=512, num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=2,
                               head_dim=128, linear_key_head_dim=64, linear_value_head_dim=64, linear_num_key_heads=4,
                               linear_num_value_heads=8, moe_intermediate_size=256, shared_expert_intermediate_size=256,
                               num_experts=32, num_experts_per_tok=4, vocab_size=1024)
    return stack.build_vq2_moe_model(cfg, DEV, seed=seed)


@torch.no_grad()
def attention_outputs(model, ids, cache):
    """The full-attention layer's input and output, over a prefill and 5 one-token steps of the same ids."""
    seen = []
    layer = model.model.layers[3]
    hook = layer.self_attn.register_forward_hook(
        lambda m, args, kw, out: seen.append((kw["hidden_states"].float(), out[0].float())), with_kwargs=True)
    seqs = [cache.add() for _ in range(ids.shape[0])] if cache else None
    past = None
    for lo, hi in [(0, 11)] + [(t, t + 1) for t in range(11, 16)]:
        if cache:
            cache.begin(seqs, [hi - lo] * len(seqs))
        past = model(input_ids=ids[:, lo:hi], past_key_values=past, use_cache=True).past_key_values
    hook.remove()
    for s in seqs or ():
        cache.release(s)
    return seen


@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 2e-2), (torch.int8, 4e-2)])
def test_paged_layer_matches_the_transformers_layer(dtype, tol):
    """The layers before the full-attention one are the same modules, so its inputs agree bit for bit and its
    outputs to what bf16 (2^-8 a rounding; q, k after rotary, weights, output, gate: five in a row) and int8
    (half a step of 1/127 of the row's largest value, on k and v) leave."""
    ids = torch.randint(0, 1024, (3, 16), device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    want = attention_outputs(small_model(), ids, None)
    model = small_model()
    cache = stack.use_paged_attention(model, pages=12, page_size=16, dtype=dtype)
    got = attention_outputs(model, ids, cache)
    assert len(cache.free) == 12
    for (xi, xo), (yi, yo) in zip(want, got):
        assert torch.equal(xi, yi)
        assert ((xo - yo).norm() / xo.norm()).item() < tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_paged_greedy_decode(dtype):
    model = small_model(5)
    cache = stack.use_paged_attention(model, pages=8, page_size=16, dtype=dtype)
    t1, ids1 = stack.decode(model, batch=3, prompt_len=20, steps=3, warmup=1, seed=9, cache=cache)
    t2, ids2 = stack.decode(model, batch=3, prompt_len=20, steps=3, warmup=1, seed=9, cache=cache)
    assert t1 > 0 and torch.equal(ids1, ids2) and len(cache.free) == 8 and not cache.pages
    with pytest.raises(MemoryError):
        stack.decode(model, batch=9, prompt_len=20, steps=1, warmup=0, cache=cache)
    assert len(cache.free) == 8


@torch.no_grad()
def test_model_refuses_padding_and_a_forward_without_begin():
    model = small_model(6)
    cache = stack.use_paged_attention(model, pages=8, page_size=16)
    ids = torch.randint(0, 1024, (2, 6), device=DEV)
    with pytest.raises(RuntimeError, match="begin"):
        model(input_ids=ids)
    seqs = [cache.add(), cache.add()]
    mask = torch.ones(2, 6, dtype=torch.long, device=DEV)
    mask[0, :2] = 0
    cache.begin(seqs, [6, 6])
    with pytest.raises(ValueError, match="mask"):
        model(input_ids=ids, attention_mask=mask)
    want = model(input_ids=ids, attention_mask=torch.ones_like(mask)).logits
    with pytest.raises(RuntimeError, match="begin"):
        model(input_ids=ids)
    again = [cache.add(), cache.add()]
    cache.begin(again, [6, 6])
    assert torch.equal(model(input_ids=ids).logits, want)


@torch.no_grad()
def test_stretched_rotary_reaches_the_layer():
    """Frequencies and factor given are those that the keys are stored with."""
    model = small_model(7)
    f, factor = stack.attention.rope_frequencies(32, 10000.0, {"type": "yarn", "factor": 8.0, "original": 64})
    cache = stack.use_paged_attention(model, pages=4, page_size=16, inv_freq=f, factor=factor)
    seen = []
    layer = model.model.layers[3].self_attn
    hook = layer.attn.k_norm.register_forward_hook(lambda m, args, out: seen.append(out.clone()))
    seq = cache.add()
    cache.begin([seq], [16])
    model(input_ids=torch.randint(0, 1024, (1, 16), device=DEV))
    hook.remove()
    want, _ = stack.attention.rotary(seen[0], None, torch.arange(16, device=DEV), f.to(DEV), factor=factor)
    assert torch.equal(cache.pools[0][0][cache.pages[seq][0]].transpose(0, 1), want)
