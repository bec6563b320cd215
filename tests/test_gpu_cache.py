"""The pages of a cache against a model in Python, operation by operation and in long runs, and the attention that reads them afterwards."""
import random

import pytest
import torch

from ditto_b200 import _lib, ops
from tests.masked_oracle import Oracle

pytestmark = pytest.mark.gpu


class Model:
    """Tables as lists; what is in a page is a number, its mark."""

    def __init__(self, sequences, columns, pages, page):
        self.table = [[-1] * columns for _ in range(sequences)]
        self.lengths, self.refs, self.page = [0] * sequences, [0] * pages, page
        self.marks = list(range(pages))

    def free_pages(self):
        return [i for i, r in enumerate(self.refs) if r <= 0]

    def reserve(self, counts):
        need = [max(0, -(-(n + c) // self.page) - -(-n // self.page)) for n, c in zip(self.lengths, counts)]
        free = self.free_pages()
        if sum(need) > len(free) or any(-(-(n + c) // self.page) > len(self.table[0]) for n, c in zip(self.lengths, counts)):
            return False
        for s, (k, c) in enumerate(zip(need, counts)):
            first = -(-self.lengths[s] // self.page)
            for i in range(k):
                p = free.pop(0)
                self.table[s][first + i], self.refs[p] = p, 1
            self.lengths[s] += c
        return True

    def fork(self, parents, children):
        free = self.free_pages()
        if sum(self.lengths[p] % self.page != 0 for p in parents) > len(free):
            return False
        for p, c in zip(parents, children):
            full, rest = divmod(self.lengths[p], self.page)
            row = self.table[p][:full] + [-1] * (len(self.table[p]) - full)
            if rest:
                row[full] = free.pop(0)
                self.marks[row[full]] = self.marks[self.table[p][full]]
            self.table[c], self.lengths[c] = row, self.lengths[p]
            for x in row:
                if x >= 0:
                    self.refs[x] += 1
        return True

    def free(self, sequences):
        for s in set(sequences):
            for x in self.table[s]:
                if x >= 0:
                    self.refs[x] -= 1
            self.table[s], self.lengths[s] = [-1] * len(self.table[s]), 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        moves = dict(zip([i for i in range(n, len(self.refs)) if self.refs[i] > 0], [i for i in range(n) if self.refs[i] <= 0]))
        for a, b in moves.items():
            self.refs[b], self.refs[a], self.marks[b] = self.refs[a], 0, self.marks[a]
        self.table = [[moves.get(x, x) for x in row] for row in self.table]


class Tables:
    def __init__(self, m, pools, device):
        self.m, self.device = m, device
        self.table = torch.tensor(m.table, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(m.lengths, dtype=torch.int32, device=device)
        self.refs = torch.tensor(m.refs, dtype=torch.int32, device=device)
        self.pools = pools

    def ids(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def check(self):
        assert self.table.tolist() == self.m.table
        assert self.lengths.tolist() == self.m.lengths
        assert self.refs.tolist() == self.m.refs
        for i, pool in enumerate(self.pools):
            marks = torch.tensor(self.m.marks, device=self.device).view(-1, 1) + 1000 * i
            assert torch.equal(pool.flatten(1).double(), marks.double().expand(-1, pool[0].numel()))


def _pools(n, pages, shape, dtype, device):
    marks = torch.arange(pages, device=device).view(-1, *[1] * len(shape))
    return [(marks + 1000 * i).to(dtype).expand(pages, *shape).contiguous() for i in range(n)]


# sequences, columns, pages, page, pools, shape of a page, type
CACHES = [(1, 1, 1, 1, 1, (8,), torch.float32), (6, 9, 40, 16, 3, (16, 2, 8), torch.float32), (40, 30, 700, 7, 2, (7, 1, 4), torch.float32),
          (300, 12, 5000, 16, 1, (16, 4, 2), torch.float64), (5, 70, 300, 1, 64, (4,), torch.float32), (3, 40, 100, 128, 2, (128, 33), torch.float64)]


@pytest.mark.parametrize("case", CACHES, ids=lambda c: "x".join(map(str, c[:5])))
def test_runs(cuda, case):
    sequences, columns, pages, page, n, shape, dtype = case
    rng = random.Random(sequences)
    m = Model(sequences, columns, pages, page)
    t = Tables(m, _pools(n, pages, shape, dtype, cuda), cuda)
    for step in range(25):
        live = [s for s in range(sequences) if m.lengths[s]]
        empty = [s for s in range(sequences) if not m.lengths[s]]
        what = rng.choice(["reserve", "reserve", "fork", "fork", "free", "compact"])
        status = 0
        if what == "reserve":
            counts = [rng.choice([0, 1, page, rng.randint(0, 3 * page)]) if rng.random() < 0.5 else 0 for _ in range(sequences)]
            if not m.reserve(counts):
                status = _lib.STATUS_NO_PAGES
            ops.cache_reserve(t.table, t.lengths, t.refs, t.ids(counts), page)
        elif what == "fork" and live and empty:
            children = rng.sample(empty, rng.randint(1, len(empty)))
            parents = [rng.choice(live) for _ in children]
            if not m.fork(parents, children):
                status = _lib.STATUS_NO_PAGES
            ops.cache_fork(t.pools, t.table, t.lengths, t.refs, t.ids(parents), t.ids(children), page)
        elif what == "free" and live:
            gone = [rng.choice(live) for _ in range(rng.randint(1, len(live)))]        # some of them twice
            m.free(gone)
            ops.cache_free(t.table, t.lengths, t.refs, t.ids(gone))
        elif what == "compact":
            m.compact()
            if step % 2:
                t.table, t.refs = ops.cache_compact(t.pools, t.table, t.refs)
            else:
                ops.cache_compact(t.pools, t.table, t.refs, out_table=t.table, out_references=t.refs)
        assert ops.device_status(cuda) == status, what
        t.check()


def test_copy(cuda):
    pools = _pools(300, 50, (3, 16), torch.float16, cuda)         # more pools than one launch takes
    want = [p.clone() for p in pools]
    source, target = [3, 7, 3, -1, 5, 9], [40, 41, 42, 43, -1, 44]
    for p in want:
        for a, b in zip(source, target):
            if a >= 0 and b >= 0:
                p[b] = p[a]
    ids = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    ops.cache_copy(pools, ids(source), ids(target))
    assert all(torch.equal(a, b) for a, b in zip(pools, want)) and ops.device_status(cuda) == 0
    for bad in (([50], [1]), ([1], [50]), ([2 ** 31 - 1], [2])):
        ops.cache_copy(pools, ids(bad[0]), ids(bad[1]))
        assert ops.device_status(cuda) == _lib.STATUS_BAD_PAGE
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    one = torch.arange(4 * 8, device=cuda).view(4, 8).float()     # a single tensor, pages with gaps between them
    room = torch.zeros(4, 12, device=cuda)
    room[:, :8] = one
    ops.cache_copy(room[:, :8], ids([0]), ids([3]))
    assert torch.equal(room[3, :8], one[0]) and (room[:, 8:] == 0).all()
    ops.cache_copy(pools, ids([]), ids([]))


def test_sequences_and_pages_out_of_range(cuda):
    m = Model(4, 3, 10, 4)
    m.reserve([5, 6, 0, 0])
    t = Tables(m, _pools(1, 10, (4, 4), torch.float32, cuda), cuda)
    ops.cache_free(t.table, t.lengths, t.refs, t.ids([-1, 4, 99]))
    t.check()
    ops.cache_fork(t.pools, t.table, t.lengths, t.refs, t.ids([9, -2, 1, 0]), t.ids([2, 3, -1, 0]), 4)
    t.check()
    assert ops.device_status(cuda) == 0
    t.table[0, 0] = 12                                  # a page that the pool does not have
    ops.cache_free(t.table, t.lengths, t.refs, t.ids([0]))
    assert ops.device_status(cuda) == _lib.STATUS_BAD_PAGE and t.table[0].tolist() == [-1, -1, -1]


def test_a_serving_run(cuda):
    """Prompts, samples forked from them, tokens appended to each, sequences freed, the pool compacted -- captured step by step where a
    program would -- and the attention over it against the definition."""
    H, Hk, d, page, layers = 4, 2, 64, 16, 2
    sequences, columns, pages = 8, 20, 90
    m = Model(sequences, columns, pages, page)
    pools = [torch.full((pages, page, Hk, d), float("nan"), device=cuda, dtype=torch.bfloat16) for _ in range(2 * layers)]
    t = Tables(m, pools, cuda)
    g = torch.Generator(device=cuda).manual_seed(2)
    rows = [[[torch.zeros(0, Hk, d, device=cuda, dtype=torch.bfloat16) for _ in range(2)] for _ in range(layers)] for _ in range(sequences)]

    def grow(counts):
        assert m.reserve(counts)
        ops.cache_reserve(t.table, t.lengths, t.refs, t.ids(counts), page)
        starts = t.ids([sum(counts[:i]) for i in range(sequences + 1)])
        for layer in range(layers):
            q = torch.randn(sum(counts), H, d, generator=g, device=cuda).bfloat16()
            k, v = (torch.randn(sum(counts), Hk, d, generator=g, device=cuda).bfloat16() for _ in range(2))
            kp, vp = pools[2 * layer], pools[2 * layer + 1]
            ops.cache_append(k, v, kp, vp, t.table, t.lengths, starts)
            out = ops.paged_attention(q, kp, vp, t.table, t.lengths, starts, scale=0.125, cap=20.0)
            first = 0
            for s, c in enumerate(counts):
                for i, x in enumerate((k, v)):
                    rows[s][layer][i] = torch.cat([rows[s][layer][i], x[first:first + c]])
                if c:
                    Oracle(q[None, first:first + c], *(x[None] for x in rows[s][layer]), scale=0.125, causal=True, cap=20.0).check(out[None, first:first + c])
                first += c
        assert t.table.tolist() == m.table and t.lengths.tolist() == m.lengths and t.refs.tolist() == m.refs
    grow([100, 33, 0, 0, 0, 0, 0, 0])
    parents, children = [0, 0, 1, 1], [2, 3, 4, 5]
    assert m.fork(parents, children)
    ops.cache_fork(t.pools, t.table, t.lengths, t.refs, t.ids(parents), t.ids(children), page)
    for a, b in zip(parents, children):
        rows[b] = [[x.clone() for x in layer] for layer in rows[a]]
    for _ in range(3):
        grow([1, 1, 1, 1, 1, 1, 0, 0])
    m.free([0, 4])
    ops.cache_free(t.table, t.lengths, t.refs, t.ids([0, 4]))
    for s in (0, 4):
        rows[s] = [[x[:0] for x in layer] for layer in rows[s]]
    m.compact()
    t.table, t.refs = ops.cache_compact(t.pools, t.table, t.refs)
    grow([200, 1, 5, 1, 0, 40, 0, 7])
    assert ops.device_status(cuda) == 0


def test_more_pools_than_a_launch_takes(cuda):
    """Fork and compaction of 300 pools: copies in two launches, the tables once."""
    m = Model(4, 5, 30, 4)
    t = Tables(m, _pools(300, 30, (4, 4), torch.float32, cuda), cuda)
    counts = [6, 9, 3, 0]
    m.reserve(counts)
    ops.cache_reserve(t.table, t.lengths, t.refs, t.ids(counts), 4)
    m.fork([1], [3])
    ops.cache_fork(t.pools, t.table, t.lengths, t.refs, t.ids([1]), t.ids([3]), 4)
    t.check()
    m.free([0])
    ops.cache_free(t.table, t.lengths, t.refs, t.ids([0]))
    m.compact()
    t.table, t.refs = ops.cache_compact(t.pools, t.table, t.refs)
    t.check()
    assert ops.device_status(cuda) == 0


def test_captured_fork(cuda):
    """A fork in a graph follows the tables' contents at each replay."""
    m = Model(6, 5, 40, 4)
    t = Tables(m, _pools(2, 40, (4, 4), torch.float32, cuda), cuda)
    m.reserve([6, 3, 0, 0, 0, 0])
    ops.cache_reserve(t.table, t.lengths, t.refs, t.ids([6, 3, 0, 0, 0, 0]), 4)
    parents, children, gone = t.ids([0, 1]), t.ids([2, 3]), t.ids([2, 3])
    ops.cache_fork(t.pools, t.table, t.lengths, t.refs, parents, children, 4)
    m.fork([0, 1], [2, 3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_free(t.table, t.lengths, t.refs, gone)
        ops.cache_fork(t.pools, t.table, t.lengths, t.refs, parents, children, 4)
    for p in ([0, 1], [1, 1], [0, 0]):
        parents.copy_(t.ids(p))
        graph.replay()
        m.free([2, 3])
        m.fork(p, [2, 3])
        torch.cuda.synchronize()
        t.check()
    assert ops.device_status(cuda) == 0


def test_refusals(cuda):
    m = Model(4, 3, 10, 4)
    t = Tables(m, _pools(2, 10, (4, 4), torch.float32, cuda), cuda)
    ids = t.ids
    for call in (lambda: ops.cache_reserve(t.table, t.lengths, t.refs, ids([1]), 4), lambda: ops.cache_reserve(t.table, t.lengths, t.refs, ids([1] * 4), 0),
                 lambda: ops.cache_reserve(t.table, t.lengths[:3], t.refs, ids([1] * 4), 4),
                 lambda: ops.cache_fork(t.pools, t.table, t.lengths, t.refs, ids([0]), ids([1, 2]), 4),
                 lambda: ops.cache_fork(t.pools, t.table, t.lengths, t.refs, ids([0] * 5), ids([1] * 5), 4),
                 lambda: ops.cache_fork([], t.table, t.lengths, t.refs, ids([0]), ids([1]), 4),
                 lambda: ops.cache_fork([p[:9] for p in t.pools], t.table, t.lengths, t.refs, ids([0]), ids([1]), 4),
                 lambda: ops.cache_fork([t.pools[0], t.pools[1][:, :2]], t.table, t.lengths, t.refs, ids([0]), ids([1]), 4),
                 lambda: ops.cache_compact([p.transpose(1, 2) for p in t.pools], t.table, t.refs),
                 lambda: ops.cache_compact(t.pools, t.table, t.refs, out_table=t.table[:2]),
                 lambda: ops.cache_compact([p[:, 0, :3] for p in t.pools], t.table, t.refs),
                 lambda: ops.cache_copy(t.pools, ids([1, 2]), ids([1])), lambda: ops.cache_free(t.table.t(), t.lengths, t.refs, ids([1]))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.cache_free(t.table, t.lengths, t.refs, ids([1]).long()), lambda: ops.cache_free(t.table.cpu(), t.lengths, t.refs, ids([1])),
                 lambda: ops.cache_copy([p.cpu() for p in t.pools], ids([1]), ids([2])), lambda: ops.cache_compact(t.pools, t.table.long(), t.refs)):
        with pytest.raises(TypeError):
            call()
    ops.cache_free(t.table, t.lengths, t.refs, ids([]))
    t.check()


def test_python_path_gives_the_same(cuda):
    def run():
        m = Model(6, 5, 40, 4)
        t = Tables(m, _pools(2, 40, (4, 4), torch.float32, cuda), cuda)
        ops.cache_reserve(t.table, t.lengths, t.refs, t.ids([6, 3, 9, 0, 0, 0]), 4)
        ops.cache_free(t.table, t.lengths, t.refs, t.ids([0]))
        ops.cache_fork(t.pools, t.table, t.lengths, t.refs, t.ids([1, 2]), t.ids([4, 5]), 4)
        table, refs = ops.cache_compact(t.pools, t.table, t.refs)
        return [table, refs, t.lengths, *t.pools]
    run()
    fast = ops._fast
    assert fast is not None
    want = run()
    try:
        ops._fast = None
        got = run()
    finally:
        ops._fast = fast
    assert all(torch.equal(a, b) for a, b in zip(want, got))
