"""What stands between a decoder layer's q/k/v projections and its output projection: rotary
positions, a paged key/value cache (16-bit, or 8-bit with a scale per token and head) and attention
of new tokens over it -- one token per sequence while decoding, chunks or whole prompts before that.

Tensors. A cache layer is two pools ``[pages, kv_heads, page_size, head_size]`` (int8 ones with two
fp32 scale tensors ``[pages, kv_heads, page_size]``); ``table`` int32 ``[seqs, cols]`` names the pages
of each sequence, ``lens`` int32 ``[seqs]`` counts its tokens, the new ones included, and ``starts``
int32 ``[seqs + 1]`` says where its new tokens begin in q, k and v (None: one new token each). They
stay on the device; a call reads them when its kernels run, so a CUDA graph replays with whatever
they hold then. ``PagedKVCache`` keeps them for a program that has no allocator of its own.

The reference leaves these blocks to the transformers modules (vq2/load_and_test_full_35b.py:124-223),
whose cache is concatenated anew every step.
"""
import math

import torch

from . import _lib

_KV_CODE = {torch.float16: _lib.VQ2_F16, torch.bfloat16: _lib.VQ2_BF16, torch.int8: _lib.VQ2_I8}
_Q_CODE = {torch.float16: _lib.VQ2_F16, torch.bfloat16: _lib.VQ2_BF16}


def rope_frequencies(rot, theta=10000.0, scaling=None):
    """(inv_freq fp32 [rot / 2] on the CPU, factor): the angle per position of each pair, theta^(-2i/rot),
    and what cos and sin are multiplied by. ``scaling`` stretches the context: None, or a dict with ``type``

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"yarn"`` (Peng et al. 2023): pairs that turn fewer than ``beta_slow`` (1) times in ``original`` positions
      are divided by ``factor``, those that turn more than ``beta_fast`` (32) times are kept, a linear ramp over
      the pair index between; cos and sin times 0.1 ln(factor) + 1 (or ``attention_factor``);
    * ``"llama3"``: wavelengths above ``original / low`` (1) divided by ``factor``, below ``original / high`` (4)
      kept, interpolated in original / wavelength between.
    """
    if rot < 2 or rot % 2:
        raise ValueError(f"the rotary width must be even and at least 2; got {rot}")
    f = float(theta) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    factor = 1.0
    if scaling is not None:
        kind, by = scaling["type"], float(scaling["factor"])
        if by < 1:
            raise ValueError("a scaling factor stretches: it is at least 1")
        if kind == "linear":
            f = f / by
        elif kind == "yarn":
            original = scaling["original"]

            def pair_of(turns):  # the (real-valued) pair that turns so often in the original context
                return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo = max(math.floor(pair_of(scaling.get("beta_fast", 32))), 0)
            hi = min(math.ceil(pair_of(scaling.get("beta_slow", 1))), rot - 1)
            keep = 1 - ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            f = f / by * (1 - keep) + f * keep
            factor = scaling.get("attention_factor", 0.1 * math.log(by) + 1.0)
        elif kind == "llama3":
            low, high = scaling.get("low", 1.0), scaling.get("high", 4.0)
            turns = scaling["original"] * f / (2 * math.pi)
            keep = ((turns - low) / (high - low)).clamp(0, 1)
            f = f / by * (1 - keep) + f * keep
        else:
            raise ValueError(f"unknown rotary scaling {kind!r}")
    return f.float(), float(factor)


def _call(name, device, *args):
    """The entry point on the current stream of ``device`` (its last argument)."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        status = getattr(_lib._lib or _lib.load(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = getattr(_lib.load(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, name)


def _rows(x, name, like=None):
    """[T, H, D] fp16 / bf16 CUDA tensor with a contiguous last dimension."""
    if not x.is_cuda:
        _lib.require_cuda(x)
    if x.dim() != 3 or x.dtype not in _Q_CODE:
        raise ValueError(f"{name} must be [tokens, heads, head_size] in fp16 or bf16; got {tuple(x.shape)} {x.dtype}")
    if like is not None and (x.dtype != like.dtype or x.shape[0] != like.shape[0] or x.shape[2] != like.shape[2]
                             or x.device != like.device):
        raise ValueError(f"{name} {tuple(x.shape)} {x.dtype} does not go with {tuple(like.shape)} {like.dtype}")
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _int32(x, name, shape, device):
    if x.dtype != torch.int32 or x.shape != shape or x.device != device or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} on {device}; got "
                         f"{x.dtype} {tuple(x.shape)} on {x.device}")
    return x.data_ptr()


def _pools(k_pages, v_pages, k_scale, v_scale, table, dtype, heads, head_size, device):
    """The cache's arguments as the entry points take them: (pools and scales, pages .. table cols)."""
    code = _KV_CODE.get(k_pages.dtype)
    if code is None or v_pages.dtype != k_pages.dtype:
        raise ValueError(f"pools hold fp16, bf16 or int8, both the same; got {k_pages.dtype} and {v_pages.dtype}")
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("pools must be contiguous [pages, kv_heads, page_size, head_size], k and v alike")
    if k_pages.device != device or v_pages.device != device:
        raise ValueError(f"pools on {k_pages.device} and {v_pages.device}, tokens on {device}")
    pages, h, page, d = k_pages.shape
    ks = vs = None
    if code == _lib.VQ2_I8:
        for s in (k_scale, v_scale):
            if (s is None or s.dtype != torch.float32 or s.shape != (pages, h, page) or not s.is_contiguous()
                    or s.device != device):
                raise ValueError("int8 pools need contiguous fp32 k_scale and v_scale [pages, kv_heads, page_size]")
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    elif k_scale is not None or v_scale is not None:
        raise ValueError("scales go with int8 pools only")
    elif dtype is not None and k_pages.dtype != dtype:
        raise ValueError(f"pools hold {k_pages.dtype}, the tokens are {dtype}")
    if (heads is not None and h != heads) or (head_size is not None and d != head_size):
        raise ValueError(f"pools have {h} heads of {d}; the tokens {heads} of {head_size}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.device != device or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError("table must be int32 [seqs, cols] with contiguous rows, on the tokens' device")
    cols = table.shape[1]
    return ((k_pages.data_ptr(), v_pages.data_ptr(), code, ks, vs),
            (pages, h, page, d, table.data_ptr(), max(table.stride(0), cols), cols))


def _freq(inv_freq, head_size, device):
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or inv_freq.device != device:
        raise ValueError("inv_freq must be a contiguous fp32 vector on the tokens' device")
    rot = 2 * inv_freq.shape[0]
    if not 2 <= rot <= head_size:
        raise ValueError(f"inv_freq turns {rot} values of a head of {head_size}")
    return inv_freq.data_ptr(), rot


def rotary(q, k, positions, inv_freq, *, interleaved=False, factor=1.0, inverse=False):
    """q [T, Hq, D] and k [T, Hk, D] (or None) turned by ``positions`` (int32 or int64 [T]): new contiguous tensors
    (q', k'). Pair i of the first 2 * len(inv_freq) values of a head -- (x[i], x[i + len]), or (x[2i], x[2i+1]) when
    ``interleaved`` -- turns by positions * inv_freq[i] and is multiplied by ``factor``; the rest is copied. The angle
    is exact to 32 bits at any position below 2^31. ``inverse`` turns back: the gradient of the forward pass."""
    q = _rows(q, "q")
    T, hq, d = q.shape
    dev = q.device
    if positions.shape != (T,) or positions.dtype not in (torch.int32, torch.int64) or positions.device != dev:
        raise ValueError(f"positions must be int32 or int64 [{T}] on {dev}")
    f, rot = _freq(inv_freq, d, dev)
    q_out = torch.empty(T, hq, d, dtype=q.dtype, device=dev)
    k_out, k_args = None, (None, 0, 0, 0)
    if k is not None:
        k = _rows(k, "k", q)
        k_out = torch.empty(T, k.shape[1], d, dtype=q.dtype, device=dev)
        k_args = (k.data_ptr(), k.stride(0), k.stride(1), k.shape[1])
    if not T:
        return q_out, k_out
    positions = positions.contiguous()
    _call("vq2_rotary", dev, q.data_ptr(), q.stride(0), q.stride(1), hq, *k_args, _Q_CODE[q.dtype], T, d,
          positions.data_ptr(), positions.dtype == torch.int64, f, rot, interleaved, factor, inverse, q_out.data_ptr(),
          None if k is None else k_out.data_ptr())
    return q_out, k_out


def cache_write(k, v, k_pages, v_pages, table, lens, starts=None, *, k_scale=None, v_scale=None, q=None, inv_freq=None,
                interleaved=False, factor=1.0):
    """Write the new tokens' k and v [T, kv_heads, D] into the pools, in one launch. With ``inv_freq`` k is turned at
    its position first, and ``q`` [T, Hq, D] with it: the turned q is returned (None without q). int8 pools: every
    (token, head) row is quantised with its own scale, amax / 127, from the turned values in 32 bits; a row with an
    infinity or a NaN reads back as NaN. Tokens whose position has no page in ``table`` are not stored."""
    k = _rows(k, "k")
    v = _rows(v, "v", k)
    T, h, d = k.shape
    dev = k.device
    pools, shape = _pools(k_pages, v_pages, k_scale, v_scale, table, k.dtype, h, d, dev)
    if v.shape[1] != h:
        raise ValueError("k and v must have the same heads")
    seqs = table.shape[0]
    lens_p = _int32(lens, "lens", (seqs,), dev)
    if starts is None and T != seqs:
        raise ValueError(f"without starts every sequence has one new token; got {T} tokens for {seqs} sequences")
    starts_p = None if starts is None else _int32(starts, "starts", (seqs + 1,), dev)
    f, rot = (None, 0) if inv_freq is None else _freq(inv_freq, d, dev)
    q_out, q_args = None, (None, 0, 0, 0, None)
    if q is not None:
        q = _rows(q, "q", k)
        q_out = torch.empty(T, q.shape[1], d, dtype=q.dtype, device=dev)
        q_args = (q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], q_out.data_ptr())
    if not T:
        return q_out
    _call("vq2_cache_write", dev, *q_args, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
          _Q_CODE[k.dtype], T, f, rot, interleaved, factor, *pools, *shape, lens_p, starts_p, seqs)
    return q_out


def cache_read(k_pages, v_pages, table, starts, total, *, k_scale=None, v_scale=None, dtype=None):
    """Whole sequences back out of the pools: (k, v) [total, kv_heads, D], sequence b's first starts[b+1] - starts[b]
    positions from row starts[b] on. ``dtype``: of the result for int8 pools (default bf16)."""
    if not k_pages.is_cuda:
        _lib.require_cuda(k_pages)
    dev = k_pages.device
    if dtype is None:
        dtype = torch.bfloat16 if k_pages.dtype == torch.int8 else k_pages.dtype
    if dtype not in _Q_CODE:
        raise ValueError(f"a cache is read back as fp16 or bf16; got {dtype}")
    pools, shape = _pools(k_pages, v_pages, k_scale, v_scale, table, dtype, None, None, dev)
    seqs = table.shape[0]
    starts_p = _int32(starts, "starts", (seqs + 1,), dev)
    k, v = (torch.empty(total, shape[1], shape[3], dtype=dtype, device=dev) for _ in range(2))
    if not total:
        return k, v
    _call("vq2_cache_read", dev, *pools, *shape, starts_p, seqs, k.data_ptr(), v.data_ptr(), _Q_CODE[dtype], total)
    return k, v


def paged_attention(q, k_pages, v_pages, table, lens, starts=None, *, k_scale=None, v_scale=None, scale=None, causal=True,
                    window=0, max_new=None, max_len=None, return_lse=False):
    """Attention of the new tokens q [T, Hq, D] over their sequences' cached keys and values (their own among them):
    [T, Hq, D]. A token at position p sees the keys l < lens, l <= p when ``causal``, l > p - window when ``window``
    is not 0; one that sees none gives zeros. Query head h reads key/value head h // (Hq / kv_heads). ``scale``
    defaults to D^-0.5. ``max_new`` and ``max_len`` bound every sequence's new tokens and length; the defaults (all of
    T, all that ``table`` has room for) are right and size the launch for more than may be needed. ``return_lse``:
    also fp32 [T, Hq], the natural logarithm of each row's sum of exponentials (-inf where no key is seen)."""
    q = _rows(q, "q")
    T, hq, d = q.shape
    dev = q.device
    pools, shape = _pools(k_pages, v_pages, k_scale, v_scale, table, q.dtype, None, d, dev)
    h = shape[1]
    if hq % h or not hq:
        raise ValueError(f"{hq} query heads do not share {h} key/value heads")
    seqs = table.shape[0]
    lens_p = _int32(lens, "lens", (seqs,), dev)
    room = shape[6] * shape[2]
    max_len = room if max_len is None else min(int(max_len), room)
    if starts is None:
        if T != seqs:
            raise ValueError(f"without starts every sequence has one new token; got {T} tokens for {seqs} sequences")
        max_new, starts_p = 1, None
    else:
        starts_p = _int32(starts, "starts", (seqs + 1,), dev)
        max_new = T if max_new is None else min(int(max_new), T)
    if window < 0 or max_len < 0 or max_new < 0:
        raise ValueError("window, max_new and max_len count tokens: none is negative")
    if q.data_ptr() % 16 or q.stride(0) % 8 or q.stride(1) % 8:  # the kernels read 16 bytes at a time
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty(T, hq, d, dtype=q.dtype, device=dev)
    lse = torch.empty(T, hq, dtype=torch.float32, device=dev) if return_lse else None
    if not T:
        return (out, lse) if return_lse else out
    lib = _lib._lib or _lib.load()
    nbytes = lib.vq2_paged_attention_workspace(T, hq, h, d, pools[2], seqs, max_new, max_len, window)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _call("vq2_paged_attention", dev, q.data_ptr(), q.stride(0), q.stride(1), _Q_CODE[q.dtype], T, hq, *pools, *shape,
          lens_p, starts_p, seqs, max_new, max_len, d ** -0.5 if scale is None else scale, causal, window,
          out.data_ptr(), lse.data_ptr() if return_lse else None, ws.data_ptr() if nbytes else None, nbytes)
    return (out, lse) if return_lse else out
