"""The decode stack on a 4-bit cache: what its layers write and read, call by call, against 64 bits."""
import pytest
import torch

from compressai_b200 import stack
from test_cache4_gpu import EPS, attend64, parts, turn64, values64
from test_stack_paged_gpu import small_model

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("prompt", [20, 150])
def test_every_call_of_a_decode(prompt):
    """A prompt (150: by the kernel for many rows), then steps of one token. Keys, turned at their positions, and values are within half a
    step of what the layer gave (the turn in 32 bits is off by 4e-6 of the row's largest value); the attention's bounds are those of
    test_cache4_gpu."""
    model = small_model(5)
    cache = stack.use_paged_attention(model, pages=32, page_size=16, dtype=torch.int4)
    write, attend, news = cache.write, cache.attend, []

    def rows(layer, which, seq):
        ids, n = torch.tensor(cache.pages[seq], device=DEV), cache.lengths[seq]
        pool, scales = cache.pools[layer][which][ids], cache.scales[layer][which][ids]
        _, scale, factor = parts(pool, scales)
        step = (scale.double()[..., None] * factor).repeat_interleave(64, -1)[..., : 2 * pool.shape[-1]]
        return [x.transpose(1, 2).flatten(0, 1)[:n] for x in (values64(pool, scales), step)]

    def checked_write(layer, k, v, *, q, inv_freq, factor):
        out = write(layer, k, v, q=q, inv_freq=inv_freq, factor=factor)
        at = 0
        for seq, n in zip(cache.batch["seqs"], cache.batch["counts"]):
            pos = torch.arange(cache.lengths[seq] - n, cache.lengths[seq], device=DEV)
            want_q = turn64(q[at:at + n], pos, inv_freq, factor=factor)
            assert ((out[at:at + n].double() - want_q).abs() <= EPS[torch.bfloat16] * want_q.abs() + 4e-6 * q.abs().max()).all()
            for which, x in enumerate((turn64(k[at:at + n], pos, inv_freq, factor=factor), v[at:at + n].double())):
                got, step = (y[-n:] for y in rows(layer, which, seq))
                near = 4e-6 * x.abs().amax(-1, keepdim=True)
                assert ((got - x).abs() <= step * 0.5 + 2 * near).all()
                assert (step <= (9 / 8 / 7 * (1 + 1e-5)) * x.abs().amax(-1, keepdim=True)).all()
            at += n
        return out

    def checked_attend(layer, q, *, scale):
        out = attend(layer, q, scale=scale)
        at = 0
        for seq, n in zip(cache.batch["seqs"], cache.batch["counts"]):
            L = cache.lengths[seq]
            (k, kstep), (v, _) = rows(layer, 0, seq), rows(layer, 1, seq)
            want, _ = attend64(q[at:at + n], k, v, torch.arange(L - n, L, device=DEV), scale, True, 0)
            delta = 2.0 ** -20 * 15 * kstep.max() * scale * q[at:at + n].abs().double().sum(-1).max()
            tol = (2.0 ** -10 + 2 * delta + 2e-5) * v.abs().max() + EPS[torch.bfloat16] * want.abs()
            assert ((out[at:at + n].double() - want).abs() <= tol).all()
            news.append((layer, n))
            at += n
        return out
    cache.write, cache.attend = checked_write, checked_attend
    _, ids = stack.decode(model, batch=2, prompt_len=prompt, steps=2, warmup=1, seed=9, cache=cache)
    assert [n for _, n in news] == [prompt] * 2 + [1] * 6 and ids.shape == (2, 1)
