"""What stands between a decoder layer's q/k/v projections and its output projection: rotary
positions, a paged key/value cache (16-bit, or 8-bit with a scale per token and head) and attention
of new tokens over it -- one token per sequence while decoding, chunks or whole prompts before that.

Tensors. A cache layer is two pools ``[pages, kv_heads, page_size, head_size]`` (int8 ones with two
fp32 scale tensors ``[pages, kv_heads, page_size]``); ``table`` int32 ``[seqs, cols]`` names the pages
of each sequence, ``lens`` int32 ``[seqs]`` counts its tokens, the new ones included, and ``starts``
int32 ``[seqs + 1]`` says where its new tokens begin in q, k and v (None: one new token each). They
stay on the device; a call reads them when its kernels run, so a CUDA graph replays with whatever
they hold then. ``PagedKVCache`` keeps them for a program that has no allocator of its own.

Nothing here is recorded by autograd: rotary's gradient is its ``inverse``, the rest is for inference.

The reference leaves these blocks to the transformers modules (vq2/load_and_test_full_35b.py:124-223),
whose cache is concatenated anew every step.
"""
import ctypes
import math
import os

import torch

from . import _lib

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


_host = None


def _load():
    """The host module (built beside the library), with the library's entry points bound."""
    global _host
    if _host is None:
        import importlib.util
        lib = _lib.load()
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_attention_host.so")
        if not os.path.exists(path):
            raise _lib.VQ2Error(f"compressai_b200 attention host module not built: {path} is missing "
                                "(run `python -m compressai_b200.build`); there is no fallback")
        spec = importlib.util.spec_from_file_location("_attention_host", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        names = ("vq2_rotary", "vq2_cache_write", "vq2_cache_read", "vq2_paged_attention", "vq2_paged_attention_workspace")
        mod.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names}, _lib.check,
                 torch.OutOfMemoryError)
        _host = mod
    return _host


def rotary(q, k, positions, inv_freq, *, interleaved=False, factor=1.0, inverse=False):
    """q [T, Hq, D] and k [T, Hk, D] (or None) turned by ``positions`` (int32 or int64 [T]): new contiguous tensors
    (q', k'). Pair i of the first 2 * len(inv_freq) values of a head -- (x[i], x[i + len]), or (x[2i], x[2i+1]) when
    ``interleaved`` -- turns by positions * inv_freq[i] and is multiplied by ``factor``; the rest is copied. The angle
    is exact to 32 bits at any position below 2^31. ``inverse`` turns back: the gradient of the forward pass."""
    return (_host or _load()).rotary(q, k, positions, inv_freq, interleaved, factor, inverse)


def cache_write(k, v, k_pages, v_pages, table, lens, starts=None, *, k_scale=None, v_scale=None, q=None, inv_freq=None,
                interleaved=False, factor=1.0):
    """Write the new tokens' k and v [T, kv_heads, D] into the pools, in one launch. With ``inv_freq`` k is turned at
    its position first, and ``q`` [T, Hq, D] with it: the turned q is returned (None without q; a token of no sequence
    turns as at position 0). int8 pools: every (token, head) row is quantised with its own scale, amax / 127, from the
    turned values in 32 bits; a row with an infinity or a NaN reads back as NaN. Tokens whose position has no page in
    ``table`` are not stored."""
    return (_host or _load()).cache_write(k, v, k_pages, v_pages, table, k_scale, v_scale, lens, starts, q, inv_freq,
                                          interleaved, factor)


def cache_read(k_pages, v_pages, table, starts, total, *, k_scale=None, v_scale=None, dtype=None):
    """Whole sequences back out of the pools: (k, v) [total, kv_heads, D], sequence b's first starts[b+1] - starts[b]
    positions from row starts[b] on. ``dtype``: of the result for int8 pools (default bf16)."""
    return (_host or _load()).cache_read(k_pages, v_pages, table, k_scale, v_scale, starts, total, dtype)


def paged_attention(q, k_pages, v_pages, table, lens, starts=None, *, k_scale=None, v_scale=None, scale=None, causal=True,
                    window=0, max_new=None, max_len=None, return_lse=False):
    """Attention of the new tokens q [T, Hq, D] over their sequences' cached keys and values (their own among them):
    [T, Hq, D]. A token at position p sees the keys l < lens, l <= p when ``causal``, l > p - window when ``window``
    is not 0; one that sees none gives zeros, and so do tokens of no sequence, before ``starts[0]`` and from
    ``starts[-1]`` on (a step padded to a fixed size). Query head h reads key/value head h // (Hq / kv_heads). ``scale``
    defaults to D^-0.5. ``max_new`` and ``max_len`` bound every sequence's new tokens and length; the defaults (all of
    T, all that ``table`` has room for) are right and size the launch for more than may be needed; of a sequence past
    them, keys from ``max_len`` on may be left out and rows from ``max_new`` on hold anything. ``return_lse``:
    also fp32 [T, Hq], the natural logarithm of each row's sum of exponentials (-inf where no key is seen).

    A value that is not finite in a cached V row makes NaN, besides in the rows that see its token, in rows of the same
    launch tile that do not (their weight of 0 is multiplied with it, as a masked dense product would). What lies past
    a sequence's end or in pages that no sequence has may hold anything.

    A call returns before its kernels have run; ``check_status`` says whether any of them gave up (NaN in its rows)."""
    return (_host or _load()).paged_attention(q, k_pages, v_pages, table, k_scale, v_scale, lens, starts, scale, causal, window,
                                              max_new, max_len, return_lse)


def check_status(device=None):
    """Wait for the device and raise VQ2Error if a ``paged_attention`` on it, on any stream, gave up a wait since this
    was last called: the kernels wait for their own copies about 2 s at most, then leave NaN in the rows they were at.
    For where a program synchronises anyway."""
    with torch.cuda.device(device):
        _lib.check(_lib.load().vq2_attention_status(1), "vq2_paged_attention")


class PagedKVCache:
    """The cache of a model's attention layers: pools for ``layers`` layers that share one page table, and who
    has which page. A program ``add``s sequences, says with ``begin`` how many tokens each one adds, and then
    calls ``write`` and ``attend`` once a layer; ``release`` gives a sequence's pages back.

    ``dtype`` is that of q, k and v, or torch.int8, which quantises what is written. The tables are kept on
    the host and go to the device in one copy a step, as new tensors: a captured step would replay with the ones it
    was captured with (keep tables of your own for that)."""

    def __init__(self, layers, pages, kv_heads, head_size, *, page_size=64, max_len=32768, dtype=torch.bfloat16,
                 device="cuda"):
        if pages < 1 or layers < 1 or max_len < 1:
            raise ValueError("layers, pages and max_len are at least 1")
        self.page_size, self.max_len = page_size, max_len
        shape = (pages, kv_heads, page_size, head_size)
        self.pools = [tuple(torch.empty(shape, dtype=dtype, device=device) for _ in range(2)) for _ in range(layers)]
        self.device = self.pools[0][0].device   # with its index: the current device may change
        self.scales = [tuple(torch.empty(shape[:3], device=device) for _ in range(2)) if dtype == torch.int8 else (None, None)
                       for _ in range(layers)]
        self.free = list(range(pages - 1, -1, -1))
        self.pages, self.lengths = {}, {}
        self._next, self.batch = 0, None

    def add(self):
        """A new, empty sequence's id."""
        self._next += 1
        self.pages[self._next], self.lengths[self._next] = [], 0
        return self._next

    def release(self, seq):
        self.free += reversed(self.pages.pop(seq))
        del self.lengths[seq]

    def begin(self, seqs, counts):
        """The next calls' tokens are ``counts[i]`` new ones of sequence ``seqs[i]``, in this order. Pages are taken
        for all of them or, with a MemoryError, for none. The tokens count from here on: where a step fails before
        every layer has written them, ``cancel`` takes them back."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("seqs are different sequences, counts their numbers of new tokens")
        P = self.page_size
        lens = [self.lengths[s] + c for s, c in zip(seqs, counts)]
        if max(lens, default=0) > self.max_len:
            raise ValueError(f"a sequence of {max(lens)} tokens: this cache's are at most {self.max_len}")
        need = [-(-n // P) - len(self.pages[s]) for s, n in zip(seqs, lens)]
        if sum(need) > len(self.free):
            raise MemoryError(f"{sum(need)} pages are needed, {len(self.free)} are free")
        for s, n, k in zip(seqs, lens, need):
            self.pages[s] += [self.free.pop() for _ in range(k)]
            self.lengths[s] = n
        self.batch = dict(seqs=list(seqs), counts=list(counts))
        try:
            self.batch.update(self._tables(lens, counts, seqs))
        except BaseException:
            self.cancel()
            raise

    def _tables(self, lens, counts, seqs):
        B, cols = len(seqs), max([len(self.pages[s]) for s in seqs] + [1])
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        flat = lens + starts + [p for s in seqs for p in self.pages[s] + [-1] * (cols - len(self.pages[s]))]
        host = torch.tensor(flat, dtype=torch.int32)
        if self.device.type == "cuda":
            host = host.pin_memory()
        t = host.to(self.device, non_blocking=True)
        one = all(c == 1 for c in counts)
        return dict(lens=t[:B], starts=None if one else t[B:2 * B + 1], table=t[2 * B + 1:].view(B, cols),
                    max_new=max(counts, default=0), max_len=max(lens, default=0))

    def cancel(self):
        """Take back the last ``begin``: its tokens, and the pages that they alone needed (for sequences not released since)."""
        if self.batch is None:
            raise RuntimeError("no batch to take back")
        for s, c in reversed(list(zip(self.batch["seqs"], self.batch["counts"]))):
            if s in self.pages:
                self.lengths[s] -= c
                keep = -(-self.lengths[s] // self.page_size)
                self.free += reversed(self.pages[s][keep:])
                del self.pages[s][keep:]
        self.batch = None

    def _batch(self, tokens):
        if self.batch is None:
            raise RuntimeError("no batch: begin says which sequences the tokens belong to")
        if tokens != sum(self.batch["counts"]):
            raise ValueError(f"the batch has {sum(self.batch['counts'])} new tokens; got {tokens}")
        return self.batch

    def write(self, layer, k, v, *, q=None, inv_freq=None, interleaved=False, factor=1.0):
        """``cache_write`` of the batch's tokens into a layer."""
        b = self._batch(k.shape[0])
        return cache_write(k, v, *self.pools[layer], b["table"], b["lens"], b["starts"], k_scale=self.scales[layer][0],
                           v_scale=self.scales[layer][1], q=q, inv_freq=inv_freq, interleaved=interleaved, factor=factor)

    def attend(self, layer, q, *, scale=None, causal=True, window=0):
        """``paged_attention`` of the batch's tokens over a layer."""
        b = self._batch(q.shape[0])
        return paged_attention(q, *self.pools[layer], b["table"], b["lens"], b["starts"], k_scale=self.scales[layer][0],
                               v_scale=self.scales[layer][1], scale=scale, causal=causal, window=window,
                               max_new=b["max_new"], max_len=b["max_len"])
