"""Attention over a paged cache, and appending to it, against the definition in 64 bits sequence by sequence."""
import math

import pytest
import torch

from ditto_b200 import _lib, ops
from tests.masked_oracle import Oracle

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


class Cache:
    """Sequences of the given lengths in pages of a pool whose other slots hold NaN, and the new tokens at their ends."""

    def __init__(self, seed, lengths, new, H, Hk, d, page, dtype, spare=3, columns=None, device="cuda:0"):
        g = torch.Generator(device=device).manual_seed(seed)
        normal = lambda *s: torch.randn(s, generator=g, device=device).to(dtype)  # noqa: E731
        self.lengths_list, self.new = lengths, new
        n = [-(-x // page) for x in lengths]
        self.pages = sum(n) + spare
        self.keys, self.values = (torch.full((self.pages, page, Hk, d), math.nan, device=device, dtype=dtype) for _ in range(2))
        order = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)).int()
        columns = columns or max(max(n), 1) + 1
        table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
        self.rows, at = [], 0
        for b, x in enumerate(lengths):
            table[b, :n[b]] = order[at:at + n[b]]
            at += n[b]
            k, v = normal(x, Hk, d), normal(x, Hk, d)
            self.rows.append((k, v))
            for i in range(x - new[b]):
                page_id, slot = table[b, i // page].item(), i % page
                self.keys[page_id, slot], self.values[page_id, slot] = k[i], v[i]
        self.table = table.to(device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=device)
        self.query = normal(sum(new), H, d)
        self.new_keys = torch.cat([k[len(k) - m:] for (k, _), m in zip(self.rows, new)])
        self.new_values = torch.cat([v[len(v) - m:] for (_, v), m in zip(self.rows, new)])

    def append(self, starts=True):
        ops.cache_append(self.new_keys, self.new_values, self.keys, self.values, self.table, self.lengths, self.starts if starts else None)

    def attend(self, starts=True, **rules):
        return ops.paged_attention(self.query, self.keys, self.values, self.table, self.lengths, self.starts if starts else None, **rules)

    def check(self, out, **rules):
        first = 0
        for b, ((k, v), m) in enumerate(zip(self.rows, self.new)):
            if m:
                r = dict(rules)
                if r.get("prefix") is not None:
                    r["prefix"] = r["prefix"][b:b + 1]
                Oracle(self.query[None, first:first + m], k[None], v[None], causal=True, **r).check(out[None, first:first + m])
            first += m
        assert ops.device_status("cuda:0") == 0


def _slopes(H):
    return torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], device="cuda:0")


# lengths, heads, kv heads, d, page
SINGLE = [([1], 1, 1, 64, 16), ([128, 129, 127, 1], 4, 2, 128, 128), ([300, 17, 2000, 64, 65], 8, 2, 64, 16), ([5000], 32, 8, 128, 64),
          ([700] * 40, 7, 1, 80, 32), ([1000, 10], 128, 1, 128, 256), ([333, 1, 4097], 6, 2, 40, 384)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", SINGLE, ids=str)
def test_single_tokens(cuda, case, dtype):
    lengths, H, Hk, d, page = case
    c = Cache(1, lengths, [1] * len(lengths), H, Hk, d, page, dtype)
    c.append(starts=False)
    for b, (k, v) in enumerate(c.rows):                # what was appended, and only that
        i = lengths[b] - 1
        assert torch.equal(c.keys[c.table[b, i // page].item(), i % page], k[i]) and torch.equal(c.values[c.table[b, i // page].item(), i % page], v[i])
    written = sum(lengths)
    assert (~c.keys.isnan()).all(-1).all(-1).sum().item() == written
    c.check(c.attend(starts=False, scale=d ** -0.5), scale=d ** -0.5)


CHUNKS = [([200], [200], 2, 2, 64, 16), ([700, 129, 5], [200, 129, 1], 6, 2, 80, 64), ([3000, 1, 400, 256], [700, 1, 0, 1], 8, 1, 128, 32),
          ([2100, 2100], [2100, 3], 4, 4, 128, 128), ([130] * 9, [2] * 9, 16, 2, 64, 16), ([1500], [1500], 100, 1, 64, 256)]


@pytest.mark.parametrize("rule", ["plain", "cap", "slopes", "prefix"])
@pytest.mark.parametrize("case", CHUNKS, ids=str)
def test_chunks(cuda, case, rule):
    lengths, new, H, Hk, d, page = case
    c = Cache(2, lengths, new, H, Hk, d, page, BF16)
    c.append()
    rules = {"scale": d ** -0.5}
    if rule == "cap":
        rules["cap"] = 20.0
    if rule == "slopes":
        rules["slopes"] = _slopes(H)
    if rule == "prefix":
        rules["prefix"] = torch.tensor([(97 * b) % 300 for b in range(len(lengths))], dtype=torch.int32, device=cuda)
    c.check(c.attend(**rules), **rules)


# lengths, heads, kv heads, d, page: single tokens with rules, shares of the work that end inside a sequence among them
RULED = [([3000, 1, 129, 64], 8, 2, 128, 32), ([700] * 40, 21, 3, 80, 32), ([5000, 2], 64, 2, 128, 64), ([900, 31], 33, 1, 64, 128),
         ([9000, 4000, 100], 6, 6, 64, 256)]


@pytest.mark.parametrize("rule", ["cap", "slopes", "both", "prefix"])
@pytest.mark.parametrize("case", RULED, ids=str)
def test_single_tokens_with_rules(cuda, case, rule):
    lengths, H, Hk, d, page = case
    c = Cache(12, lengths, [1] * len(lengths), H, Hk, d, page, BF16)
    c.append(starts=False)
    rules = {"scale": d ** -0.5}
    if rule in ("cap", "both"):
        rules["cap"] = 4.0
    if rule in ("slopes", "both"):
        rules["slopes"] = _slopes(H)
    if rule == "prefix":
        rules["prefix"] = torch.tensor([(970 * b) % 3000 for b in range(len(lengths))], dtype=torch.int32, device=cuda)
    c.check(c.attend(starts=False, **rules), **rules)


@pytest.mark.parametrize("new", [1, 40, 700])
def test_far_keys_and_steep_slopes(cuda, new):
    """Biases of thousands, in parts of a sequence that hold far keys only; slopes of 0 and below."""
    c = Cache(13, [9000, 300], [new, 1], 6, 2, 128, 64, F16)
    c.append()
    rules = {"scale": 128 ** -0.5, "slopes": torch.tensor([2.0, 0.7, 0.0, 1e-3, 30.0, -1e-3], device=cuda)}
    c.check(c.attend(**rules), **rules)


def test_more_blocks_than_can_be_counted(cuda):
    """The reach of the table times the heads passes 2^31 blocks: refused, not cut."""
    pool = torch.zeros(4, 128, 256, 64, dtype=F16, device=cuda)
    table = torch.zeros(1, 2 ** 23, dtype=torch.int32, device=cuda)
    query, lengths = torch.zeros(1, 256, 64, dtype=F16, device=cuda), torch.tensor([100], dtype=torch.int32, device=cuda)
    with pytest.raises((ValueError, RuntimeError)):
        ops.paged_attention(query, pool, pool, table, lengths)
    assert (ops.paged_attention(query, pool, pool, table[:, :2 ** 22], lengths) == 0).all()


@pytest.mark.parametrize("columns", [12, 48, 49], ids=str)
@pytest.mark.parametrize("sequences", [1, 90, 300])
def test_short_reach(cuda, sequences, columns):
    """Tables of a few blocks' reach, on both sides of what is taken whole; more items than CTAs; lengths of 0 and beyond the table."""
    lengths = [1 + (b * 37) % (16 * columns) for b in range(sequences)]
    c = Cache(14, lengths, [1] * sequences, 6, 2, 64, 16, F16, columns=columns)
    c.append(starts=False)
    rules = {"scale": 0.125, "slopes": _slopes(6)}
    want = c.attend(starts=False, **rules)
    c.check(want, **rules)
    table = c.lengths.clone()
    c.lengths[0] = 0
    if sequences > 1:
        c.lengths[1] = 10 ** 9                          # (ids of -1 among what it reaches)
    out = c.attend(starts=False, **rules)
    assert (out[0] == 0).all()
    ops.device_status(cuda)
    for b in range(2, sequences):                       # (other lengths cut the work elsewhere, which regroups sums of 32 bits: the bound, not bits)
        k, v = c.rows[b]
        Oracle(c.query[None, b:b + 1], k[None], v[None], causal=True, **rules).check(out[None, b:b + 1])
    c.lengths.copy_(table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.attend(starts=False, **rules)
    graph.replay()
    assert torch.equal(out, want)


def test_tokens_behind_the_last_sequence_stay(cuda):
    c = Cache(3, [100, 300], [10, 20], 4, 2, 64, 16, F16)
    c.append()
    want = c.attend(scale=0.125)
    query = torch.cat([c.query, c.query[:7]])
    out = torch.full_like(query, 5.0)
    got = ops.paged_attention(query, c.keys, c.values, c.table, c.lengths, c.starts, out=out, scale=0.125)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out[:30], want) and (out[30:] == 5).all()
    # ... and their keys are not appended
    keys, values = c.keys.clone(), c.values.clone()
    more = lambda t: torch.cat([t, torch.full_like(t[:7], 9.0)])  # noqa: E731
    ops.cache_append(more(c.new_keys), more(c.new_values), c.keys, c.values, c.table, c.lengths, c.starts)
    assert torch.equal(c.keys.nan_to_num(), keys.nan_to_num()) and torch.equal(c.values.nan_to_num(), values.nan_to_num())


def test_sequences_without_keys(cuda):
    """Length 0, more new tokens than keys: rows of zeros; a sequence without new tokens costs nothing."""
    c = Cache(4, [50, 60], [4, 4], 2, 2, 64, 16, F16)
    c.append()
    c.lengths.copy_(torch.tensor([0, 2], dtype=torch.int32))
    out = c.attend(scale=0.125)
    assert (out[:4] == 0).all() and (out[4:6] == 0).all() and (out[6:] != 0).any()
    assert ops.device_status(cuda) == 0


def test_pages_and_lengths_out_of_range(cuda):
    """Ids out of the pool and lengths beyond the table are passed over, and the status says so."""
    c = Cache(5, [200, 200], [1, 1], 2, 2, 64, 16, F16, columns=13)
    c.append(starts=False)
    want = c.attend(starts=False, scale=0.125)
    for bad in (c.pages, -1, 2 ** 31 - 1, -2 ** 31):
        table = c.table.clone()
        table[1, 3] = bad
        out = ops.paged_attention(c.query, c.keys, c.values, table, c.lengths, scale=0.125)
        assert ops.device_status(cuda) == _lib.STATUS_BAD_PAGE
        assert torch.equal(out[0], want[0]) and torch.isfinite(out).all()
        before = c.keys.clone()
        table[:, 12] = bad
        ops.cache_append(c.new_keys, c.new_values, c.keys, c.values, table, c.lengths)
        assert ops.device_status(cuda) == _lib.STATUS_BAD_PAGE and torch.equal(c.keys.nan_to_num(), before.nan_to_num())
    lengths = c.lengths.clone()
    lengths[0], lengths[1] = 10 ** 6, -4
    c.keys.nan_to_num_()
    c.values.nan_to_num_()
    table = c.table.clamp(min=0)
    out = ops.paged_attention(c.query, c.keys, c.values, table, lengths, scale=0.125)
    assert torch.isfinite(out).all() and (out[1] == 0).all() and ops.device_status(cuda) == 0
    ops.cache_append(c.new_keys, c.new_values, c.keys, c.values, table, lengths)
    assert ops.device_status(cuda) == _lib.STATUS_BAD_PAGE


def test_broken_starts_stay_inside(cuda):
    c = Cache(6, [90, 90, 90], [8, 8, 8], 2, 2, 64, 16, F16)
    c.append()
    for starts in ([0, 100, 50, 24], [-5, 8, 16, 1000], [24, 16, 8, 0]):
        out = torch.full_like(c.query, 3.0)
        ops.paged_attention(c.query, c.keys, c.values, c.table, c.lengths, torch.tensor(starts, dtype=torch.int32, device=cuda), out=out, scale=0.125)
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()
    ops.device_status(cuda)


def test_layouts(cuda):
    """Pools inside one tensor, heads in front of slots, a query from a packed tensor: the same bits."""
    c = Cache(7, [250, 70], [1, 1], 8, 2, 64, 32, BF16)
    c.append(starts=False)
    want = c.attend(starts=False, scale=0.125)
    both = torch.stack([c.keys, c.values], 1)
    assert torch.equal(ops.paged_attention(c.query, both[:, 0], both[:, 1], c.table, c.lengths, scale=0.125), want)
    k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.keys, c.values))
    packed = torch.randn(2, 3, 8, 64, device=cuda).to(BF16)
    packed[:, 1] = c.query
    wide = torch.full((2, 20), 999, dtype=torch.int32, device=cuda)
    wide[:, :c.table.shape[1]] = c.table
    assert torch.equal(ops.paged_attention(packed[:, 1], k, v, wide[:, :c.table.shape[1]], c.lengths, scale=0.125), want)
    fresh = torch.full_like(both, math.nan)
    ops.cache_append(c.new_keys, c.new_values, fresh[:, 0], fresh[:, 1], c.table, c.lengths)
    assert (~fresh.isnan()).sum().item() == 2 * 2 * 2 * 64


def test_same_bits_and_graphs(cuda):
    """The shares of a call depend on the lengths; a captured step follows them, and repeats give the same bits."""
    c = Cache(8, [3000, 700, 64, 1500], [1, 1, 1, 1], 8, 2, 128, 64, BF16)
    c.append(starts=False)
    assert all(torch.equal(c.attend(starts=False, scale=0.1), c.attend(starts=False, scale=0.1)) for _ in range(3))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.append(starts=False)
            kept = c.attend(starts=False, scale=0.1)
        graphs.append((graph, kept))
    for lengths in ([3000, 700, 64, 1500], [100, 690, 1, 1499], [2999, 3, 5, 7]):
        c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        want = ops.paged_attention(c.query, *self_append(c), c.table, c.lengths, scale=0.1)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(want, kept) for _, kept in graphs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.attend(starts=False, scale=0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def self_append(c):
    c.append(starts=False)
    return c.keys, c.values


def test_many_sequences(cuda):
    """More sequences than a CTA has threads, most of them without new tokens."""
    lengths = [(37 * i) % 300 + 1 for i in range(900)]
    new = [1 if i % 7 == 0 else 0 for i in range(900)]
    c = Cache(9, lengths, new, 4, 1, 64, 32, F16)
    c.append()
    c.check(c.attend(scale=0.125), scale=0.125)


def test_refusals(cuda):
    c = Cache(10, [40, 50], [1, 1], 4, 2, 64, 16, F16)
    good = [c.query, c.keys, c.values, c.table, c.lengths]
    def bad(kind, at, value, **more):
        args = list(good)
        args[at] = value
        with pytest.raises(kind):
            ops.paged_attention(*args, **more)
    bad(TypeError, 0, c.query.float())
    bad(TypeError, 0, c.query.cpu())
    bad(ValueError, 0, c.query[:1])                    # one token for two sequences
    bad(ValueError, 0, c.query[:, :3])
    bad(ValueError, 0, c.query[..., :56])
    bad(TypeError, 1, c.keys.to(BF16))
    bad(ValueError, 1, c.keys[:, :8])
    bad(TypeError, 3, c.table.long())
    bad(ValueError, 3, c.table[:1])
    bad(ValueError, 3, c.table[:, :0])
    bad(ValueError, 3, c.table.t().contiguous().t())
    bad(TypeError, 4, c.lengths.long())
    bad(ValueError, 4, c.lengths[:1])
    with pytest.raises(ValueError):
        ops.paged_attention(*good, c.starts[:2])
    with pytest.raises(ValueError):
        ops.paged_attention(*good, cap=-1.0)
    with pytest.raises(ValueError):
        ops.paged_attention(*good, out=torch.empty_like(c.query[:1]))
    small = torch.zeros(4, 24, 2, 64, device=cuda, dtype=F16)
    with pytest.raises(ValueError):
        ops.paged_attention(c.query, small, small, c.table, c.lengths)
    with pytest.raises(ValueError):
        ops.cache_append(c.new_keys[:, :1], c.new_values[:, :1], c.keys, c.values, c.table, c.lengths)
    with pytest.raises(TypeError):
        ops.cache_append(c.new_keys.float(), c.new_values, c.keys, c.values, c.table, c.lengths)
    with pytest.raises(ValueError):
        ops.cache_append(c.new_keys[:1], c.new_values[:1], c.keys, c.values, c.table, c.lengths)
    assert ops.paged_attention(c.query[:0], c.keys, c.values, c.table, c.lengths, torch.zeros(3, dtype=torch.int32, device=cuda)).shape == (0, 4, 64)
    assert ops.device_status(cuda) == 0


def test_python_path_gives_the_same(cuda):
    c = Cache(11, [400, 90], [33, 1], 4, 2, 64, 16, F16)
    c.append()
    want = c.attend(scale=0.125, cap=9.0)
    fast, keys = ops._fast, c.keys.clone()
    assert fast is not None
    try:
        ops._fast = None
        c.append()
        got = c.attend(scale=0.125, cap=9.0)
    finally:
        ops._fast = fast
    assert torch.equal(got, want) and torch.equal(keys.nan_to_num(), c.keys.nan_to_num())


def test_long_cache_offsets(cuda):
    """A pool whose offsets pass 2^31 elements and 2^32 bytes."""
    free, _ = torch.cuda.mem_get_info(cuda)
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    pages, page, Hk, d = 70000, 128, 2, 128            # 4.6 GB a pool
    keys = torch.zeros(pages, page, Hk, d, dtype=F16, device=cuda)
    values = torch.zeros_like(keys)
    ids = torch.tensor([[pages - 1, 3, 66000]], dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    k, v = (torch.randn(300, Hk, d, generator=g, device=cuda).to(F16) for _ in range(2))
    lengths, starts = torch.tensor([300], dtype=torch.int32, device=cuda), torch.tensor([0, 300], dtype=torch.int32, device=cuda)
    ops.cache_append(k, v, keys, values, ids, lengths, starts)
    q = torch.randn(300, 4, d, generator=g, device=cuda).to(F16)
    out = ops.paged_attention(q, keys, values, ids, lengths, starts, scale=d ** -0.5)
    Oracle(q[None], k[None], v[None], scale=d ** -0.5, causal=True).check(out[None])
    assert ops.device_status(cuda) == 0
