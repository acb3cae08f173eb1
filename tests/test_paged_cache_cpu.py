"""PagedKVCache's bookkeeping on the host (no device needed): pages, tables, refusals."""
import pytest
import torch

from compressai_b200.attention import PagedKVCache


def cache(pages=6, **kw):
    return PagedKVCache(2, pages, 1, 16, page_size=16, device="cpu", **kw)


def test_pages_follow_lengths_and_come_back():
    c = cache()
    a, b = c.add(), c.add()
    c.begin([a, b], [17, 0])
    assert c.batch["lens"].tolist() == [17, 0] and c.batch["starts"].tolist() == [0, 17, 17]
    assert c.batch["table"].tolist() == [[0, 1], [-1, -1]] and c.batch["max_new"] == 17 and c.batch["max_len"] == 17
    c.begin([b, a], [1, 1])
    assert c.batch["lens"].tolist() == [1, 18] and c.batch["starts"] is None
    assert c.batch["table"].tolist() == [[2, -1], [0, 1]]
    c.release(a)
    c.begin([b], [64])
    assert c.lengths[b] == 65 and c.pages[b] == [2, 0, 1, 3, 4] and len(c.free) == 1
    d = c.add()
    c.begin([d], [16])
    assert c.pages[d] == [5] and not c.free


def test_refusals_change_nothing():
    c = cache(max_len=90)
    a, b = c.add(), c.add()
    c.begin([a], [33])
    before = (list(c.free), dict(c.lengths), c.batch["lens"].tolist())
    with pytest.raises(MemoryError):
        c.begin([a, b], [1, 64])
    for seqs, counts in (([a], [1, 2]), ([a, a], [1, 1]), ([a], [-1]), ([a], [58])):
        with pytest.raises(ValueError):
            c.begin(seqs, counts)
    assert before == (list(c.free), dict(c.lengths), c.batch["lens"].tolist())
    for args in ((0, 4, 1, 16), (1, 0, 1, 16)):
        with pytest.raises(ValueError):
            PagedKVCache(*args, device="cpu")


def test_int8_pools_have_scales():
    c = cache(dtype=torch.int8)
    assert c.pools[1][0].dtype == torch.int8 and c.scales[1][1].shape == (6, 1, 16)
    assert cache(dtype=torch.float16).scales[0] == (None, None)


def test_tokens_are_the_batch_s():
    """A write of fewer tokens than begun would leave rows that later steps read unwritten: refused ahead of the kernels."""
    c = cache()
    x = torch.zeros(5, 1, 16, dtype=torch.bfloat16)
    for call in (lambda: c.write(0, x, x), lambda: c.attend(0, x)):
        with pytest.raises(RuntimeError, match="begin"):
            call()
    a, b = c.add(), c.add()
    for counts in ([4, 0], [5, 1]):
        c.begin([a, b], counts)
        for call in (lambda: c.write(0, x, x), lambda: c.attend(0, x)):
            with pytest.raises(ValueError, match="new tokens"):
                call()


def test_a_failed_step_is_taken_back():
    """Begun again after a step that failed, the same tokens stand at the same positions on the same pages."""
    c = cache()
    a, b = c.add(), c.add()
    c.begin([a, b], [16, 3])
    before = (list(c.free), dict(c.lengths), {s: list(p) for s, p in c.pages.items()})
    c.begin([b, a], [20, 1])
    lens, table = c.batch["lens"].tolist(), c.batch["table"].tolist()
    c.cancel()
    assert before == (c.free, c.lengths, c.pages) and c.batch is None
    c.begin([b, a], [20, 1])
    assert c.batch["lens"].tolist() == lens and c.batch["table"].tolist() == table
    c.release(b)
    c.cancel()
    assert c.lengths == {a: 16} and len(c.free) == 5
    with pytest.raises(RuntimeError):
        c.cancel()


def test_a_begin_that_fails_late_changes_nothing(monkeypatch):
    c = cache()
    a = c.add()
    c.begin([a], [10])
    before = (list(c.free), dict(c.lengths), {s: list(p) for s, p in c.pages.items()})

    def full(*args):
        raise torch.OutOfMemoryError("full")
    monkeypatch.setattr(c, "_tables", full)
    with pytest.raises(torch.OutOfMemoryError):
        c.begin([a], [30])
    assert before == (c.free, c.lengths, c.pages) and c.batch is None
