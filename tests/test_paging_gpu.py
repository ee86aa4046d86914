"""Pages of paged caches on the GPU (palu_*_pages) against a model of the pool on the host: every value exact."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


class Model:
    """The pool's rules in plain Python: the lowest free page is taken first."""

    def __init__(self, n_pages, rows, per_row, bs):
        self.n, self.bs, self.per_row = n_pages, bs, per_row
        self.table = [[] for _ in range(rows)]
        self.page = {}                                  # page -> contents (any hashable)

    def refs(self):
        r = [0] * self.n
        for t in self.table:
            for b in t:
                r[b] += 1
        return r

    def free_pages(self):
        return [b for b, c in enumerate(self.refs()) if c == 0]

    def reserve(self, rows, lens):
        free = self.free_pages()
        for r, n in zip(rows, lens):
            while len(self.table[r]) < -(-n // self.bs) and free:
                self.table[r].append(free.pop(0))

    def fork(self, parents, children, lens, caches):
        free = self.free_pages()
        for p, c, n in zip(parents, children, lens):
            full, count = n // self.bs, -(-n // self.bs)
            if len(self.table[p]) < count or self.table[c]:
                continue
            if count > full and not free:
                continue
            self.table[c] = self.table[p][:full]
            if count > full:
                b = free.pop(0)
                for x in caches:
                    x[b] = x[self.table[p][full]]
                self.table[c].append(b)

    def free(self, rows):
        for r in rows:
            self.table[r] = []

    def compact(self, caches):
        refs = self.refs()
        used = sum(c > 0 for c in refs)
        src = [b for b in range(used, self.n) if refs[b]]
        dst = [b for b in range(used) if not refs[b]]
        to = dict(zip(src, dst))
        for x in caches:
            for a, b in to.items():
                x[b] = x[a]
        self.table = [[to.get(b, b) for b in t] for t in self.table]


def compare(pool, model, caches, plain):
    torch.cuda.synchronize()
    want = torch.full(pool.table.shape, -1, dtype=torch.int32)
    for r, t in enumerate(model.table):
        want[r, :len(t)] = torch.tensor(t, dtype=torch.int32)
    assert torch.equal(pool.table.cpu(), want)
    assert pool.refs.tolist() == model.refs()
    assert pool.mapped.tolist() == [len(t) for t in model.table]
    for a, b in zip(caches, plain):
        assert torch.equal(a.cpu(), b)


def make(cuda, n_pages=40, rows=12, per_row=6, bs=16, widths=(32, 48), dtype=torch.bfloat16):
    from palu_b200 import paging
    g = torch.Generator().manual_seed(0)
    plain = [torch.randn(n_pages, 2, bs, w, generator=g).to(dtype) for w in widths]
    caches = [p.to(cuda) for p in plain]
    return paging.PagePool(caches, rows=rows, blocks_per_row=per_row), Model(n_pages, rows, per_row, bs), caches, plain


def test_random_sequences_of_calls(cuda):
    rng = random.Random(3)
    pool, model, caches, plain = make(cuda)
    for step in range(60):
        what = rng.choice(["reserve", "reserve", "fork", "fork", "free", "compact"])
        if what == "reserve":
            rows = rng.sample(range(12), rng.randint(1, 4))
            lens = [rng.randint(0, 96) for _ in rows]
            pool.reserve(rows, lens)
            model.reserve(rows, lens)
        elif what == "fork":
            children = rng.sample(range(12), rng.randint(1, 4))
            rest = [r for r in range(12) if r not in children]
            parents = [rng.choice(rest) for _ in children]
            lens = [rng.randint(0, 16 * len(model.table[p]) + 10) for p in parents]
            lens = [min(n, 96) for n in lens]
            pool.fork(parents, children, lens)
            model.fork(parents, children, lens, plain)
        elif what == "free":
            rows = rng.sample(range(12), rng.randint(1, 5))
            pool.free(rows)
            model.free(rows)
        else:
            pool.compact()
            model.compact(plain)
        compare(pool, model, caches, plain)


def test_several_launches_of_many_rows(cuda):
    """More rows than one launch takes, pages past one scan step of the pool, a layer count past one launch's caches."""
    from palu_b200 import paging
    n, bs = 9000, 16
    plain = [torch.arange(n, dtype=torch.int32).view(n, 1, 1).repeat(1, 1, bs) + 10000 * i for i in range(130)]
    caches = [p.to(cuda) for p in plain]
    pool, model = paging.PagePool(caches, rows=1300, blocks_per_row=8), Model(n, 1300, 8, bs)
    rng = random.Random(1)
    rows = list(range(600))
    rng.shuffle(rows)
    lens = [rng.randint(1, 128) for _ in rows]
    pool.reserve(rows, lens)
    model.reserve(rows, lens)
    kids = list(range(600, 1200))
    pool.fork(rows, kids, lens)
    model.fork(rows, kids, lens, plain)
    gone = rng.sample(range(1200), 700)
    pool.free(gone)
    model.free(gone)
    pool.compact()
    model.compact(plain)
    compare(pool, model, caches, plain)
    pool.check()


def test_what_goes_wrong_is_told(cuda):
    pool, model, caches, plain = make(cuda, n_pages=5)
    pool.reserve([0, 1], [64, 64])                      # 4 pages, then one of four
    model.reserve([0, 1], [64, 64])
    compare(pool, model, caches, plain)
    with pytest.raises(RuntimeError, match="ran out of pages"):
        pool.check()
    pool.check()
    pool.fork([0, 1], [2, 3], [20, 17])                 # no page left; the parent is too short
    pool.fork([0], [1], [32])                           # the child is not empty
    compare(pool, model, caches, plain)
    with pytest.raises(RuntimeError, match="ran out.*fewer positions.*not empty"):
        pool.check()


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 64), (torch.uint8, 24), (torch.uint8, 5), (torch.float32, 3)])
def test_copies_of_any_type_and_size(cuda, dtype, width):
    from palu_b200 import paging
    g = torch.Generator().manual_seed(2)
    plain = [torch.randint(0, 200, (30, 3, 7, width), generator=g).to(dtype) for _ in range(2)]
    wide = torch.randint(0, 200, (30, 2, 3, 7, width), generator=g).to(dtype)   # K and V of a page side by side
    caches, both = [p.to(cuda) for p in plain], wide.to(cuda)
    src, dst = [1, 29, 1, 7, 5], [2, 0, 3, 7, 28]
    paging.copy_pages([*caches, both[:, 1]], src, dst)
    torch.cuda.synchronize()
    for s, d in zip(src, dst):
        for p in plain:
            p[d] = p[s]
        wide[d, 1] = wide[s, 1]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(caches, plain)) and torch.equal(both.cpu(), wide)


def test_many_copies_in_one_call(cuda):
    from palu_b200 import paging
    plain = torch.arange(2000).view(2000, 1, 1).repeat(1, 3, 100)
    cache = plain.to(cuda)
    src, dst = list(range(0, 2000, 2)), list(range(1, 2000, 2))
    paging.copy_pages([cache], src, dst)
    plain[dst] = plain[src]
    assert torch.equal(cache.cpu(), plain)


def test_captured_and_replayed(cuda):
    """A fork and its release in a graph: each replay forks the pages' current contents."""
    pool, model, caches, plain = make(cuda)
    pool.reserve([0], [40])
    model.reserve([0], [40])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pool.fork([0, 0], [1, 2], [40, 16])
        pool.free([1, 2])
    for step in range(2):
        for c, p in zip(caches, plain):
            c[2] += 1
            p[2] = (p[2] + 1)
        graph.replay()
        for p in plain:
            p[3] = p[2]                                  # the partial page of positions 32 .. 39
        compare(pool, model, caches, plain)


def test_compacting_an_empty_and_a_full_pool(cuda):
    pool, model, caches, plain = make(cuda, n_pages=6)
    pool.compact()
    compare(pool, model, caches, plain)
    pool.reserve([3], [96])
    model.reserve([3], [96])
    pool.compact()
    compare(pool, model, caches, plain)


def test_lengths_near_the_end_of_32_bits(cuda):
    """Blocks of 2^30 positions (no cache is named, so nothing has their size): the last lengths that 32 bits hold."""
    import ctypes
    from palu_b200 import _lib
    lib, n = _lib.load(), 4
    state = torch.tensor([-1] * 4 + [0] * n + [0] * 2 + [0], dtype=torch.int32, device=cuda)   # table [2][2], refs, mapped, status
    at = lambda i: state.data_ptr() + 4 * i
    pool = ctypes.byref(_lib.PagePoolInfo(at(0), at(4), at(4 + n), at(6 + n), 2, 2, n, 1 << 30))
    ints = lambda *x: (ctypes.c_int32 * len(x))(*x)
    ws = torch.zeros(int(lib.palu_page_workspace_bytes(n)), dtype=torch.uint8, device=cuda)
    most = 2**31 - 1
    _lib.check(lib.palu_reserve_pages(pool, ints(0), ints(most), 1, None))
    _lib.check(lib.palu_fork_pages(pool, None, 0, ints(0), ints(1), ints(most), 1, ws.data_ptr(), ws.numel(), None))
    torch.cuda.synchronize()
    assert state.tolist() == [0, 1, 0, 2, 2, 1, 1, 0, 2, 2, 0]     # the child shares page 0 and has a page of its own
