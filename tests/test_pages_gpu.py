"""Pages copied within their pools, and sequences that share, copy, give back and move pages."""
import pytest
import torch

from compressai_b200 import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def bytes_of(x):
    return x.contiguous().view(torch.uint8)


@pytest.mark.parametrize("shapes", [[(9, 16)], [(9, 4, 32, 64), (9, 4, 32)], [(40, 2, 64, 256)] * 5, [(300, 1, 16, 8), (300, 16)],
                                    [(7, 3, 16, 1000)] * 2, [(5, 1 << 20)], [(12, 48)] * 300])
@pytest.mark.parametrize("n", [0, 1, 3, 10 ** 6])
def test_pages_are_copied(shapes, n):
    pages = shapes[0][0]
    n = min(n, pages // 2)
    kinds = [torch.bfloat16, torch.float32, torch.int8, torch.uint8]
    pools = [torch.randint(0, 256, s, generator=gen(i), device=DEV).to(kinds[i % 4 if s[-1] % 16 == 0 else 1]) for i, s in enumerate(shapes)]
    perm = torch.randperm(pages, generator=gen(1), device=DEV).to(torch.int32)
    src, dst = perm[:n], perm[n:2 * n]
    want = [p.clone() for p in pools]
    for w in want:
        w[dst.long()] = w[src.long()]
    assert A.copy_pages(pools, src, dst) is None
    for p, w in zip(pools, want):
        assert torch.equal(bytes_of(p), bytes_of(w))
    A.copy_pages(tuple(pools), src.tolist(), dst.tolist())
    for p, w in zip(pools, want):
        assert torch.equal(bytes_of(p), bytes_of(w))


def test_ids_that_are_no_pages_copy_nothing():
    pool = torch.randn(6, 4, 16, device=DEV)
    want = pool.clone()
    want[5] = want[0]
    ids = [[0, -1, 6, 2, 1, 3, 0], [5, 2, 3, 7, -3, 3, 2 ** 31 - 1]]
    A.copy_pages([pool], *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in ids))
    assert torch.equal(pool, want)


def test_pools_past_32_bits():
    pool = torch.empty(70000, 32768, dtype=torch.uint8, device=DEV)   # 2.3 GB
    pool[69999], pool[65536] = 7, 9
    A.copy_pages([pool], [69999, 65536], [0, 65535])
    assert (pool[0] == 7).all() and (pool[65535] == 9).all()


def test_a_replayed_copy_reads_its_ids_then():
    pool = torch.arange(8 * 64, device=DEV, dtype=torch.float32).view(8, 64)
    src, dst = (torch.tensor([v], dtype=torch.int32, device=DEV) for v in (0, 1))
    A.copy_pages([pool], src, dst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.copy_pages([pool], src, dst)
    src.fill_(5)
    dst.fill_(2)
    graph.replay()
    assert torch.equal(pool[2], pool[5]) and torch.equal(pool[1], pool[0])


def test_copy_refusals():
    pool, i = torch.zeros(4, 16, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    for pools, src, dst in (([pool.cpu()], i, i), (pool, i, i), ([pool], i.long(), i), ([pool], i, torch.cat([i, i])),
                            ([pool, pool[:3]], i, i), ([pool[:, :8]], i, i), ([torch.zeros(4, 3, device=DEV)], i, i),
                            ([pool], [0], [4]), ([pool], [-1], [0]), ([pool], [0, 1], [2, 2]), ([pool], [0, 1], [1, 2]),
                            ([pool], [0, 1], [2]), ([pool], i.cpu(), i.cpu())):
        with pytest.raises(ValueError):
            A.copy_pages(pools, src, dst)
    assert pool.abs().max() == 0


# ------------------------------------------------------------------------------------- a cache's sequences
KINDS = [torch.bfloat16, torch.int8, torch.int4]


class Twin:
    """A PagedKVCache beside one that shares nothing: every sequence written whole on pages of its own."""

    def __init__(self, dtype, pages=40, page=16):
        self.c = A.PagedKVCache(2, pages, 2, 64, page_size=page, dtype=dtype)
        self.dtype, self.page, self.g = dtype, page, gen(5)
        self.kv = {}   # (sequence, layer) -> k, v of its tokens

    def step(self, seqs, counts):
        self.c.begin(seqs, counts)
        for layer in range(2):
            k, v = (torch.randn(sum(counts), 2, 64, generator=self.g, device=DEV).to(torch.bfloat16) for _ in range(2))
            self.c.write(layer, k, v)
            at = 0
            for s, n in zip(seqs, counts):
                old = self.kv.get((s, layer))
                new = (k[at:at + n], v[at:at + n])
                self.kv[s, layer] = new if old is None else tuple(torch.cat([x, y]) for x, y in zip(old, new))
                at += n

    def fork(self, s):
        new = self.c.fork(s)
        for layer in range(2):
            if (s, layer) in self.kv:
                self.kv[new, layer] = self.kv[s, layer]
        return new

    def truncate(self, s, n):
        self.c.truncate(s, n)
        for layer in range(2):
            self.kv[s, layer] = tuple(x[:n] for x in self.kv[s, layer])

    def check(self):
        c = self.c
        users = [0] * len(c.users)
        for pages in c.pages.values():
            for p in pages:
                users[p] += 1
        assert users == c.users and sorted(c.free) == [p for p, u in enumerate(users) if not u]
        for s, pages in c.pages.items():
            n = c.lengths[s]
            assert len(pages) == -(-n // self.page)
            if not n:
                continue
            q = torch.randn(1, 4, 64, generator=gen(n), device=DEV).to(torch.bfloat16)
            lens, starts = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([n], [0, n]))
            table = torch.tensor([pages], dtype=torch.int32, device=DEV)
            own = torch.arange(len(pages), dtype=torch.int32, device=DEV)[None]
            for layer in range(2):
                k, v = self.kv[s, layer]
                assert k.shape[0] == n
                alone = [A.empty_pool(len(pages), 2, self.page, 64, self.dtype) for _ in range(2)]
                kw = dict(k_scale=alone[0][1], v_scale=alone[1][1])
                A.cache_write(k, v, alone[0][0], alone[1][0], own, lens, starts, **kw)
                here = dict(k_scale=c.scales[layer][0], v_scale=c.scales[layer][1])
                for got, want in zip(A.cache_read(*c.pools[layer], table, starts, n, **here),
                                     A.cache_read(alone[0][0], alone[1][0], own, starts, n, **kw)):
                    assert torch.equal(got, want)
                assert torch.equal(A.paged_attention(q, *c.pools[layer], table, lens, **here),
                                   A.paged_attention(q, alone[0][0], alone[1][0], own, lens, **kw))


@pytest.mark.parametrize("dtype", KINDS)
def test_forks_write_on_without_each_other(dtype):
    t = Twin(dtype)
    a = t.c.add()
    t.step([a], [37])
    b, d = t.fork(a), t.fork(a)
    assert len(t.c.free) == 37
    t.check()
    t.step([b, a, d], [3, 1, 20])    # two of the three write on in a copy of the third page
    t.check()
    e = t.fork(d)
    t.step([e], [1])
    t.c.release(a)
    t.check()
    t.step([d, b, e], [1, 16, 2])
    t.check()
    for s in (b, d, e):
        t.c.release(s)
    assert len(t.c.free) == 40


@pytest.mark.parametrize("dtype", KINDS)
def test_truncated_and_written_again(dtype):
    t = Twin(dtype)
    a = t.c.add()
    t.step([a], [50])
    b = t.fork(a)
    t.truncate(b, 21)        # ends inside a page that a has too
    t.check()
    t.step([b], [30])
    t.check()
    t.truncate(a, 0)
    t.step([a, b], [5, 1])
    t.check()
    with pytest.raises(ValueError):
        t.c.truncate(a, 6)
    with pytest.raises(ValueError):
        t.c.truncate(a, -1)


@pytest.mark.parametrize("dtype", KINDS)
def test_compacted_and_resized(dtype):
    t = Twin(dtype)
    seqs = [t.c.add() for _ in range(6)]
    for i, s in enumerate(seqs):
        t.step([s], [20 + 9 * i])
    b = t.fork(seqs[5])
    for s in (seqs[0], seqs[2], seqs[3]):
        t.c.release(s)
    used = sum(1 for u in t.c.users if u)
    assert t.c.compact() == used and sorted(p for ps in t.c.pages.values() for p in set(ps))[-1] < used
    t.check()
    t.step([seqs[1], b], [4, 4])
    t.check()
    assert t.c.compact() == t.c.compact()
    n = sum(1 for u in t.c.users if u)
    with pytest.raises(ValueError):
        t.c.resize(n - 1)
    t.check()
    t.c.resize(n + 1)
    assert all(x is None or x.shape[0] == n + 1 for both in (t.c.pools, t.c.scales) for pair in both for x in pair)
    t.check()
    t.step([seqs[1]], [1])
    with pytest.raises(MemoryError):
        t.c.begin([seqs[4]], [100])
    t.c.resize(60)
    t.step([seqs[4]], [100])
    t.check()


def test_a_step_on_forks_is_taken_back():
    t = Twin(torch.int4)
    a = t.c.add()
    t.step([a], [20])
    b = t.fork(a)
    before = ({s: list(p) for s, p in t.c.pages.items()}, dict(t.c.lengths), list(t.c.users))
    t.c.begin([a, b], [1, 30])
    t.c.cancel()
    assert before == (t.c.pages, t.c.lengths, t.c.users)
    t.check()
    t.step([a, b], [2, 1])
    t.check()


@pytest.mark.parametrize("kind", [list, tuple])
def test_pages_named_in_lists(kind):
    pools = [torch.randn(9, 4, 16, generator=gen(i), device=DEV) for i in range(3)]
    want = [p.clone() for p in pools]
    for w in want:
        w[4], w[0] = w[7], w[2]
    A.copy_pages(kind(pools), kind([7, 2]), kind([4, 0]))
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_a_replayed_copy_by_lists_keeps_its_ids():
    pool = torch.randn(8, 64, generator=gen(0), device=DEV)
    want = pool.clone()
    A.copy_pages([pool], [0], [1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.copy_pages([pool], [3], [4])
    others = [torch.tensor([5, 6], dtype=torch.int32).pin_memory() for _ in range(100)]
    for i in (3, 2):
        pool[3], want[3] = want[i], want[i].clone()
        graph.replay()
        want[1], want[4] = want[0], want[3]
        assert torch.equal(pool, want)
    del others
