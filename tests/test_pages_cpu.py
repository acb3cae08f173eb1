"""PagedKVCache's bookkeeping of shared pages on the host, and the refusals of 4-bit pools and page copies (no device needed)."""
import ctypes
import weakref

import pytest
import torch

from compressai_b200 import _lib
from compressai_b200 import attention as A


def cache(pages=8, **kw):
    c = A.PagedKVCache(2, pages, 1, 32, page_size=16, device="cpu", **kw)
    c.copied = []
    c._copy = lambda src, dst: c.copied.append((src.tolist(), dst.tolist()))
    return c


def state(c):
    return list(c.free), list(c.users), {s: list(p) for s, p in c.pages.items()}, dict(c.lengths)


def test_a_fork_shares_until_one_writes_on():
    c = cache()
    a = c.add()
    c.begin([a], [20])
    b = c.fork(a)
    assert c.batch is None and c.pages[b] == [0, 1] and c.users[:3] == [2, 2, 0] and c.lengths[b] == 20 and len(c.free) == 6
    c.begin([b], [1])          # in a copy; a keeps its page
    assert c.pages[b] == [0, 2] and c.pages[a] == [0, 1] and c.users[:3] == [2, 1, 1] and c.copied == [([1], [2])]
    assert c.batch["table"].tolist() == [[0, 2]] and c.batch["lens"].tolist() == [21]
    c.begin([a], [1])          # nobody else on its last page
    assert len(c.copied) == 1 and c.pages[a] == [0, 1]
    c.release(a)
    assert c.users[:3] == [1, 0, 1] and c.free[-1] == 1


def test_of_all_that_share_one_writes_in_place():
    c = cache()
    a = c.add()
    c.begin([a], [3])
    b, d = c.fork(a), c.fork(a)
    c.begin([a, b, d], [1, 0, 2])       # b writes nothing and keeps the page: both others copy it
    assert c.copied == [([0, 0], [1, 2])] and c.pages[b] == [0] and c.users[:3] == [1, 1, 1]
    e = c.fork(b)
    c.begin([b, e], [1, 1])
    assert c.copied[1:] == [([0], [3])] and c.pages[e] == [0] and c.pages[b] == [3]


def test_a_full_last_page_is_not_copied():
    c = cache()
    a = c.add()
    c.begin([a], [32])
    b = c.fork(a)
    c.begin([a, b], [1, 1])
    assert not c.copied and c.pages[a] == [0, 1, 2] and c.pages[b] == [0, 1, 3]
    assert c.batch["moves"] == []


def test_refused_for_pages_changes_nothing():
    c = cache(pages=3)
    a = c.add()
    c.begin([a], [33])
    b = c.fork(a)
    before = state(c)
    with pytest.raises(MemoryError, match="1 pages are needed"):
        c.begin([b], [1])
    with pytest.raises(MemoryError, match="2 pages"):
        c.begin([a, b], [15, 16])
    assert state(c) == before and not c.copied


def test_a_copy_that_fails_is_taken_back():
    c = cache()
    a = c.add()
    c.begin([a], [20])
    b = c.fork(a)
    before = state(c)

    def full(src, dst):
        raise torch.OutOfMemoryError("full")
    c._copy = full
    with pytest.raises(torch.OutOfMemoryError):
        c.begin([b, a], [30, 1])
    assert state(c)[1:] == before[1:] and sorted(c.free) == sorted(before[0]) and c.batch is None


def test_cancel_gives_copies_back_or_keeps_the_only_one():
    c = cache()
    a = c.add()
    c.begin([a], [20])
    b = c.fork(a)
    before = state(c)
    c.begin([b, a], [1, 1])
    c.cancel()
    assert state(c)[1:] == before[1:]
    c.begin([b], [1])
    c.release(a)               # b's copy is all that is left of the page
    c.cancel()
    assert c.lengths[b] == 20 and c.pages[b] == [0, 2] and c.users[:3] == [1, 0, 1]
    c.release(b)
    assert sorted(c.free) == list(range(8))


def test_truncate():
    c = cache()
    a = c.add()
    c.begin([a], [50])
    c.truncate(a, 17)
    assert c.batch is None and c.pages[a] == [0, 1] and c.lengths[a] == 17 and c.free[-2:] == [3, 2]
    for n in (18, -1):
        with pytest.raises(ValueError):
            c.truncate(a, n)
    c.truncate(a, 16)
    assert c.pages[a] == [0]
    b = c.fork(a)
    c.truncate(b, 3)
    c.begin([b], [1])          # into a page that a still reads
    assert c.copied == [([0], [1])] and c.pages[a] == [0]
    c.truncate(a, 0)
    assert c.pages[a] == [] and c.users[0] == 0


def test_compact_moves_the_fewest():
    c = cache()
    a, b, d = c.add(), c.add(), c.add()
    for s, n in ((a, 20), (b, 40), (d, 33)):
        c.begin([s], [n])
    e = c.fork(d)
    c.release(a)
    assert c.pages[d] == [5, 6, 7] and c.compact() == 6
    assert c.copied == [([6, 7], [0, 1])] and c.pages[d] == c.pages[e] == [5, 0, 1] and c.pages[b] == [2, 3, 4]
    assert c.free == [7, 6] and c.users == [2, 2, 1, 1, 1, 2, 0, 0] and c.batch is None
    assert c.compact() == 6 and len(c.copied) == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.int4])
def test_resize(dtype):
    c = cache(dtype=dtype)
    a = c.add()
    c.begin([a], [40])
    for pool in c.pools[1]:
        pool[:3] = 5
    for n in (2, 0):
        with pytest.raises(ValueError):
            c.resize(n)
    for n in (3, 11):
        c.resize(n)
        shapes = {x.shape[0] for both in (c.pools, c.scales) for pair in both for x in pair if x is not None}
        assert shapes == {n} and len(c.free) == n - 3 and len(c.users) == n and (c.pools[1][1][:3] == 5).all()
    c.begin([a], [100])
    assert c.pages[a][:3] == [0, 1, 2] and len(c.pages[a]) == 9


@pytest.mark.parametrize("to", [4, 20])
def test_resize_that_runs_out_of_memory_leaves_pools_of_one_size(to, monkeypatch):
    c = cache()
    a = c.add()
    c.begin([a], [40])
    real, calls = torch.Tensor.new_empty, []

    def new_empty(self, *shape):
        calls.append(shape)
        if len(calls) == 3:
            raise torch.OutOfMemoryError("full")
        return real(self, *shape)
    monkeypatch.setattr(torch.Tensor, "new_empty", new_empty)
    with pytest.raises(torch.OutOfMemoryError):
        c.resize(to)
    size = min(to, 8)
    assert {x.shape[0] for pair in c.pools for x in pair} == {size} and len(c.users) == size and sorted(c.free) == list(range(3, size))


def test_a_step_ends_where_pages_move():
    """The batch's tables would name other pages, or tokens that are gone."""
    x = torch.zeros(1, 1, 32, dtype=torch.bfloat16)
    for end in (lambda c, a: c.fork(a), lambda c, a: c.truncate(a, 1), lambda c, a: c.compact(), lambda c, a: c.resize(5)):
        c = cache()
        a = c.add()
        c.begin([a], [1])
        end(c, a)
        with pytest.raises(RuntimeError, match="begin"):
            c.write(0, x, x)
        with pytest.raises(RuntimeError, match="no batch"):
            c.cancel()


def test_unknown_sequences_change_nothing():
    c = cache()
    a = c.add()
    c.begin([a], [20])
    before, batch = state(c), c.batch
    for call in (lambda: c.fork(99), lambda: c.truncate(99, 0), lambda: c.release(99)):
        with pytest.raises(KeyError):
            call()
    assert state(c) == before and c.batch is batch


# ------------------------------------------------------------------------------------- shapes, refusals
def test_pools_of_4_bits():
    pool, scales = A.empty_pool(3, 2, 32, 96, torch.int4, "cpu")
    assert pool.shape == (3, 2, 32, 48) and pool.dtype == torch.uint8
    assert scales.shape == (3, 2, 2, 4 + 2, 16) and scales.dtype == torch.uint8
    assert A.empty_pool(3, 2, 16, 64, torch.float16, "cpu")[1] is None
    assert A.empty_pool(3, 2, 16, 64, torch.int8, "cpu")[1].shape == (3, 2, 16)
    for d, page in ((48, 16), (16, 16), (64, 8)):
        with pytest.raises(ValueError):
            A.empty_pool(3, 2, page, d, torch.int4, "cpu")
    with pytest.raises(ValueError):
        A.PagedKVCache(1, 4, 1, 80, dtype=torch.int4, device="cpu")


def test_abi_refusals_of_4_bits():
    lib = _lib.load()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)

    def attn(kv=4, d=64, ks=p, page=16, kp=p):
        return lib.vq2_paged_attention(p, 256, 64, 1, 0, 4, kp, p, kv, ks, ks, 8, 2, page, d, p, 4, 4, p, p, 2, 4, 64, 0.125, 1, 0,
                                       p, None, None, 0, None)

    def write(kv=4, d=64, ks=p):
        return lib.vq2_cache_write(None, 0, 0, 0, None, p, 128, 64, p, 128, 64, 1, 0, None, 0, 0, 1.0, p, p, kv, ks, ks, 8, 2, 16, d,
                                   p, 4, 4, p, p, 2, None)

    def read(kv=4, d=64, ks=p):
        return lib.vq2_cache_read(p, p, kv, ks, ks, 8, 2, 16, d, p, 4, 4, p, 2, p, p, 1, 0, None)
    for call in (attn, write, read):
        assert call() == _lib.VQ2_OK                             # no tokens
        assert call(ks=None) == _lib.VQ2_ERR_ARG and call(ks=odd) == _lib.VQ2_ERR_ALIGN
        assert call(d=48) == _lib.VQ2_ERR_SHAPE and call(d=288) == _lib.VQ2_ERR_SHAPE and call(kv=5) == _lib.VQ2_ERR_DTYPE
        assert call(kv=3, d=48) == _lib.VQ2_OK                   # int8 takes what it took
    assert attn(page=8) == _lib.VQ2_ERR_SHAPE and attn(kp=odd) == _lib.VQ2_ERR_ALIGN


def test_abi_refusals_of_page_copies():
    lib = _lib.load()

    class Pool(ctypes.Structure):
        _fields_ = [("base", ctypes.c_void_p), ("page_bytes", ctypes.c_int64)]

    def copy(base=256, size=64, n_pools=1, pages=4, src=256, n=0, pools=True):
        arr = (Pool * 2)(Pool(base, size), Pool(256, 16))
        return lib.vq2_copy_pages(arr if pools else None, n_pools, pages, src, src, n, None)
    assert copy() == _lib.VQ2_OK and copy(n_pools=0, pools=False) == _lib.VQ2_OK and copy(size=0, n=5) == _lib.VQ2_OK
    assert copy(pools=False) == _lib.VQ2_ERR_ARG and copy(base=None) == _lib.VQ2_ERR_ARG
    assert copy(src=None, n=1) == _lib.VQ2_ERR_ARG and copy(n=-1) == _lib.VQ2_ERR_ARG and copy(n_pools=-1) == _lib.VQ2_ERR_ARG
    assert copy(base=264) == _lib.VQ2_ERR_ALIGN and copy(size=24) == _lib.VQ2_ERR_ALIGN
    assert copy(pages=0) == _lib.VQ2_ERR_SHAPE and copy(size=1 << 31) == _lib.VQ2_ERR_SHAPE and copy(size=-16) == _lib.VQ2_ERR_SHAPE


def test_cpu_tensors_are_refused():
    pool, i = torch.zeros(4, 16), torch.zeros(1, dtype=torch.int32)
    for src, dst in ((i, i), ([0], [1])):
        with pytest.raises(ValueError, match="CUDA"):
            A.copy_pages([pool], src, dst)
    for src, dst in (([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0, 1], [2])):
        with pytest.raises(ValueError):
            A.copy_pages([pool], src, dst)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int4])
@pytest.mark.parametrize("to", [4, 20])
def test_resize_gives_a_pool_back_before_it_takes_the_next(dtype, to, monkeypatch):
    c = cache(dtype=dtype)
    a = c.add()
    c.begin([a], [40])
    old = [weakref.ref(x) for both in (c.pools, c.scales) for pair in both for x in pair if x is not None]
    real, alive = torch.Tensor.new_empty, []

    def new_empty(self, *shape):
        alive.append([r() is not None for r in old])
        return real(self, *shape)
    monkeypatch.setattr(torch.Tensor, "new_empty", new_empty)
    c.resize(to)
    assert alive == [[j >= i for j in range(len(old))] for i in range(len(old))]
    assert all(x.untyped_storage().nbytes() == x.nbytes for both in (c.pools, c.scales) for pair in both for x in pair if x is not None)


@pytest.mark.parametrize("to", [4, 20])
@pytest.mark.parametrize("again", [False, True])
def test_resize_that_runs_out_of_memory_keeps_no_more_than_it_says(to, again, monkeypatch):
    """The pools that were moved already go back to the size that is left, or, where there is no memory for that either, are cut."""
    c = cache(dtype=torch.int8)
    a = c.add()
    c.begin([a], [40])
    for i, pair in enumerate(c.pools + c.scales):
        for j, x in enumerate(pair):
            x[:3] = 10 * i + j
    real, calls = torch.Tensor.new_empty, []

    def new_empty(self, *shape):
        calls.append(shape)
        if len(calls) == 4 or again and len(calls) > 4:
            raise torch.OutOfMemoryError("full")
        return real(self, *shape)
    monkeypatch.setattr(torch.Tensor, "new_empty", new_empty)
    with pytest.raises(torch.OutOfMemoryError):
        c.resize(to)
    size = min(to, 8)
    assert len(c.users) == size and sorted(c.free) == list(range(3, size))
    for i, pair in enumerate(c.pools + c.scales):
        for j, x in enumerate(pair):
            assert x.shape[0] == size and x.is_contiguous() and (x[:3] == 10 * i + j).all()
            assert again or x.untyped_storage().nbytes() == x.nbytes
