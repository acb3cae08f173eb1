"""What stands between a decoder layer's q/k/v projections and its output projection: rotary
positions, a paged key/value cache (16-bit, 8-bit with a scale per token and head, or 4-bit) and attention
of new tokens over it -- one token per sequence while decoding, chunks or whole prompts before that.

Tensors. A cache layer is two pools ``[pages, kv_heads, page_size, head_size]`` (int8 ones with two
fp32 scale tensors ``[pages, kv_heads, page_size]``; 4-bit ones, of head sizes that are multiples of 32, as
uint8 ``[.., head_size / 2]`` with two uint8 scale tensors ``[pages, kv_heads, page_size / 16, 4 + groups, 16]``,
``groups`` of 64 values a head: ``empty_pool`` makes either); ``table`` int32 ``[seqs, cols]`` names the pages
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
        names = ("vq2_rotary", "vq2_cache_write", "vq2_cache_read", "vq2_paged_attention", "vq2_paged_attention_workspace",
                 "vq2_copy_pages")
        mod.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names}, _lib.check,
                 torch.OutOfMemoryError)
        _host = mod
    return _host


def empty_pool(pages, kv_heads, page_size, head_size, dtype=torch.bfloat16, device="cuda"):
    """(pool, scales) of one layer's K or V, their contents not set; scales are None for fp16 and bf16. ``dtype``
    torch.int8 or torch.int4 makes a quantised one (4 bits: two values a byte, uint8)."""
    shape = (pages, kv_heads, page_size, head_size)
    if dtype == torch.int4:
        if head_size % 32 or page_size % 16:
            raise ValueError(f"a 4-bit cache has heads of a multiple of 32 values and pages of one of 16 rows; got {head_size}, {page_size}")
        return (torch.empty(*shape[:3], head_size // 2, dtype=torch.uint8, device=device),
                torch.empty(pages, kv_heads, page_size // 16, 4 + -(-head_size // 64), 16, dtype=torch.uint8, device=device))
    scale = torch.empty(shape[:3], device=device) if dtype == torch.int8 else None
    return torch.empty(shape, dtype=dtype, device=device), scale


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
    turned values in 32 bits; a row with an infinity or a NaN reads back as NaN. 4-bit pools (uint8): a row's scale is
    amax / 7; each 64 of its values share a factor, their amax over the row's, rounded up to 8 bits (e4m3), and
    become integers from -7 to 7, to the nearest, ties away from zero: off by half of factor * scale at most. Tokens
    whose position has no page in ``table`` are not stored."""
    return (_host or _load()).cache_write(k, v, k_pages, v_pages, table, k_scale, v_scale, lens, starts, q, inv_freq,
                                          interleaved, factor)


def cache_read(k_pages, v_pages, table, starts, total, *, k_scale=None, v_scale=None, dtype=None):
    """Whole sequences back out of the pools: (k, v) [total, kv_heads, D], sequence b's first starts[b+1] - starts[b]
    positions from row starts[b] on. ``dtype``: of the result for int8 and 4-bit pools (default bf16)."""
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


def copy_pages(pools, src, dst):
    """In every one of ``pools`` (contiguous tensors [pages, ..], of any type, a page a multiple of 16 bytes: K and V of
    all layers with their scales, say) page ``dst[i]`` becomes what page ``src[i]`` is, in a launch for 128 pools. ``src`` and ``dst``:
    int32 on the pools' device, read when the kernel runs (ids outside the pools copy nothing), or lists, which are
    checked: pages in ``dst`` are different ones and none is in ``src``. Where a tensor breaks that, such a page
    holds bytes of any of its sources."""
    if not isinstance(src, torch.Tensor) or not isinstance(dst, torch.Tensor):
        src, dst = ([int(p) for p in x] for x in (src, dst))
        if not pools:
            return
        pages = pools[0].shape[0]
        if len(src) != len(dst) or len(set(dst)) != len(dst) or set(dst) & set(src):
            raise ValueError("src and dst name as many pages each, those in dst different ones, none of them in src")
        if any(not 0 <= p < pages for p in src + dst):
            raise ValueError(f"the pools have pages 0 to {pages - 1}")
        src, dst = _ints([src, dst], pools[0].device)
    (_host or _load()).copy_pages(pools, src, dst)


def _ints(lists, device):
    """Lists of integers as int32 tensors on a device, in one copy that does not wait."""
    host = torch.tensor([v for x in lists for v in x], dtype=torch.int32)
    if device.type == "cuda":
        host = host.pin_memory()
    return host.to(device, non_blocking=True).split([len(x) for x in lists])


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

    ``fork`` makes a sequence that goes on from another one's tokens, on the same pages: whole pages stay shared, a
    partly filled one is copied (in all layers at once) when one of those that share it writes on. ``truncate`` takes a
    sequence's last tokens back, ``compact`` moves the pages in use to the front of the pools, and ``resize``
    gives the pools another size. These belong between steps: they end the batch that ``begin`` has set.

    ``dtype`` is that of q, k and v, or torch.int8 or torch.int4, which quantise what is written. The tables are kept on
    the host and go to the device in one copy a step, as new tensors: a captured step would replay with the ones it
    was captured with (keep tables of your own for that). Page copies run on the current stream, as the step's calls do."""

    def __init__(self, layers, pages, kv_heads, head_size, *, page_size=64, max_len=32768, dtype=torch.bfloat16,
                 device="cuda"):
        if pages < 1 or layers < 1 or max_len < 1:
            raise ValueError("layers, pages and max_len are at least 1")
        self.page_size, self.max_len = page_size, max_len
        made = [[empty_pool(pages, kv_heads, page_size, head_size, dtype, device) for _ in range(2)] for _ in range(layers)]
        self.pools = [(k[0], v[0]) for k, v in made]
        self.scales = [(k[1], v[1]) for k, v in made]
        self.device = self.pools[0][0].device   # with its index: the current device may change
        self.free = list(range(pages - 1, -1, -1))
        self.users = [0] * pages                # sequences on each page
        self.pages, self.lengths = {}, {}
        self._next, self.batch = 0, None

    def add(self):
        """A new, empty sequence's id."""
        self._next += 1
        self.pages[self._next], self.lengths[self._next] = [], 0
        return self._next

    def fork(self, seq):
        """A new sequence's id, with the tokens of ``seq`` and on its pages."""
        pages, length = self.pages[seq], self.lengths[seq]
        self.batch = None
        new = self.add()
        self.pages[new], self.lengths[new] = list(pages), length
        for p in pages:
            self.users[p] += 1
        return new

    def release(self, seq):
        self._give_back(self.pages.pop(seq))
        del self.lengths[seq]

    def truncate(self, seq, length):
        """Keep the first ``length`` tokens of a sequence; the pages of the others go back (drafts that were not taken)."""
        if not 0 <= length <= self.lengths[seq]:
            raise ValueError(f"the sequence has {self.lengths[seq]} tokens; {length} cannot be kept")
        self.batch = None
        keep = -(-length // self.page_size)
        self._give_back(self.pages[seq][keep:])
        del self.pages[seq][keep:]
        self.lengths[seq] = length

    def compact(self):
        """Move the pages in use to ids 0 .. n - 1, as few of them as that takes, in one ``copy_pages``; returns n."""
        n = sum(1 for u in self.users if u)
        to = iter([p for p in range(n) if not self.users[p]])
        moves = {p: next(to) for p in range(n, len(self.users)) if self.users[p]}
        self.batch = None
        if moves:
            self._copy(*_ints([list(moves), list(moves.values())], self.device))
        for pages in self.pages.values():
            pages[:] = [moves.get(p, p) for p in pages]
        for old, new in moves.items():
            self.users[new], self.users[old] = self.users[old], 0
        self.free = list(range(len(self.users) - 1, n - 1, -1))
        return n

    def resize(self, pages):
        """Pools of ``pages`` pages, the ones in use compacted into them; memory is taken and given back a pool at a time.
        Where it runs out on the way, more pages than before are not had, fewer are; the pools are of one size then too (and
        where there is not even memory to move them into that size, views of larger ones)."""
        n = sum(1 for u in self.users if u)
        if pages < max(n, 1):
            raise ValueError(f"{n} pages are in use: {pages} do not hold them")
        self.compact()
        size = min(pages, len(self.users))

        def moved(x, rows):
            y = x.new_empty(rows, *x.shape[1:])
            y[:n].copy_(x[:n])
            return y

        def resized(rows, move):   # by index: a loop over the pairs would hold the old pools until its next turn
            for kept in (self.pools, self.scales):
                for i in range(len(kept)):
                    if kept[i][0] is not None:
                        kept[i] = (move(kept[i][0], rows), kept[i][1])
                        kept[i] = (kept[i][0], move(kept[i][1], rows))

        def left(x, rows):
            if x.shape[0] == rows:
                return x
            try:
                return moved(x, rows)
            except RuntimeError:
                return x[:rows]
        try:
            resized(pages, moved)
            size = pages
        except BaseException:
            resized(size, left)
            raise
        finally:
            self.users = self.users[:n] + [0] * (size - n)
            self.free = list(range(size - 1, n - 1, -1))

    def _give_back(self, pages):
        for p in reversed(pages):
            self.users[p] -= 1
            if not self.users[p]:
                self.free.append(p)

    def _take(self):
        p = self.free.pop()
        self.users[p] = 1
        return p

    def _copy(self, src, dst):
        copy_pages([x for both in (self.pools, self.scales) for pair in both for x in pair if x is not None], src, dst)

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
        # partly filled pages that other sequences are on too: all but the last of these write on in a copy
        own, left = [], {}
        for s, c in zip(seqs, counts):
            if c and self.lengths[s] % P:
                p = self.pages[s][-1]
                left[p] = left.get(p, self.users[p]) - 1
                if left[p]:
                    own.append(s)
        if sum(need) + len(own) > len(self.free):
            raise MemoryError(f"{sum(need) + len(own)} pages are needed, {len(self.free)} are free")
        moves = []
        for s in own:
            old, new = self.pages[s][-1], self._take()
            self.pages[s][-1] = new
            self.users[old] -= 1
            moves.append((s, old, new))
        for s, n, k in zip(seqs, lens, need):
            self.pages[s] += [self._take() for _ in range(k)]
            self.lengths[s] = n
        self.batch = dict(seqs=list(seqs), counts=list(counts), moves=moves)
        try:
            self.batch.update(self._tables(lens, counts, seqs, moves))
            if moves:
                self._copy(self.batch["src"], self.batch["dst"])
        except BaseException:
            self.cancel()
            raise

    def _tables(self, lens, counts, seqs, moves):
        B, cols = len(seqs), max([len(self.pages[s]) for s in seqs] + [1])
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        lens_t, starts_t, src, dst, table = _ints([lens, starts, [m[1] for m in moves], [m[2] for m in moves], [
            p for s in seqs for p in self.pages[s] + [-1] * (cols - len(self.pages[s]))]], self.device)
        one = all(c == 1 for c in counts)
        return dict(lens=lens_t, starts=None if one else starts_t, table=table.view(B, cols), src=src, dst=dst,
                    max_new=max(counts, default=0), max_len=max(lens, default=0))

    def cancel(self):
        """Take back the last ``begin``: its tokens, and the pages that they alone needed (for sequences not released since)."""
        if self.batch is None:
            raise RuntimeError("no batch to take back")
        for s, c in reversed(list(zip(self.batch["seqs"], self.batch["counts"]))):
            if s in self.pages:
                self.lengths[s] -= c
                keep = -(-self.lengths[s] // self.page_size)
                self._give_back(self.pages[s][keep:])
                del self.pages[s][keep:]
        for s, old, new in reversed(self.batch["moves"]):
            if s in self.pages and self.users[old]:   # else its copy is the only one by now
                self.pages[s][-1] = old
                self.users[old] += 1
                self._give_back([new])
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
