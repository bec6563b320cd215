"""Masked attention and its gradients against the definition in 64 bits (tests/masked_oracle.py says what the bounds count)."""
import math

import pytest
import torch

from ditto_b200 import ops
from tests.masked_oracle import Oracle

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _operands(seed, B, M, L, H, Hk, d, dtype, device="cuda:0"):
    g = torch.Generator(device=device).manual_seed(seed)
    return [torch.randn(shape, generator=g, device=device).to(dtype) for shape in ((B, M, H, d), (B, L, Hk, d), (B, L, Hk, d), (B, M, H, d))]


def _documents(B, L, lengths, padding=0, device="cuda:0"):
    rows = []
    for b in range(B):
        ids, n = [], 0
        while len(ids) < L - padding * b:
            ids += [7 * b + n] * lengths[(b + n) % len(lengths)]
            n += 1
        rows.append((ids[:L - padding * b] + [-1] * L)[:L])
    return torch.tensor(rows, dtype=torch.int32, device=device)


def _slopes(H):
    return torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], device="cuda:0")


def _both(ops_args, grad, rules, dtype):
    q, k, v = ops_args
    out, lse = ops.masked_attention(q, k, v, return_lse=True, **rules)
    oracle = Oracle(q, k, v, **rules)
    oracle.check(out, lse)
    grads = ops.masked_attention_backward(grad, q, k, v, out, lse, **rules)
    oracle.check_gradients(grad, grads)
    assert ops.device_status("cuda:0") == 0
    return out, lse, grads


# (B, M, L, H, Hk, d): one tile and less, tile and block borders on either side, odd lengths, groups that do not divide 128, head
# dimensions that are no multiple of 16 or 64, fewer and more queries than keys
SHAPES = [(1, 1, 1, 1, 1, 64), (2, 3, 5, 2, 1, 8), (1, 127, 127, 1, 1, 64), (1, 128, 128, 2, 2, 128), (1, 129, 129, 2, 1, 128),
          (2, 255, 257, 3, 3, 72), (1, 300, 300, 6, 2, 40), (1, 200, 90, 4, 2, 96), (2, 65, 700, 7, 1, 80), (1, 513, 513, 16, 2, 128),
          (1, 40, 1000, 100, 1, 64), (1, 33, 65, 128, 1, 16), (3, 384, 384, 5, 5, 120)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(cuda, shape, causal, dtype):
    q, k, v, g = _operands(sum(shape), *shape, dtype)
    _both((q, k, v), g, dict(scale=shape[-1] ** -0.5, causal=causal), dtype)


@pytest.mark.parametrize("rule", ["cap", "slopes", "both", "small cap"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("shape", [(2, 150, 150, 6, 2, 64), (1, 260, 390, 4, 4, 128)], ids=["64", "128"])
def test_modified_scores(cuda, shape, causal, rule):
    q, k, v, g = _operands(5, *shape, BF16)
    rules = dict(scale=shape[-1] ** -0.5, causal=causal)
    if rule in ("cap", "both"):
        rules["cap"] = 30.0
    if rule == "small cap":
        rules.update(cap=0.5, scale=1.0)              # most scores are saturated
    if rule in ("slopes", "both"):
        rules["slopes"] = _slopes(shape[3])
    _both((q, k, v), g, rules, BF16)


@pytest.mark.parametrize("scale", [2.0 ** -40, 2.0 ** -21, 2.0 ** -20, 1.0, 2.0 ** 21], ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_bias_at_any_scale(cuda, causal, scale):
    """The bias in units of scores far from 1; three tiles and more keys than queries, so that tiles begin inside a block of keys."""
    q, k, v, g = _operands(21, 2, 300, 700, 4, 2, 64, BF16)
    q = (q.float() * (0.125 / scale)).to(BF16)
    rules = dict(scale=scale, causal=causal, slopes=_slopes(4))
    out, lse = ops.masked_attention(q, k, v, return_lse=True, **rules)
    Oracle(q, k, v, **rules).check(out, lse)
    assert ops.device_status(cuda) == 0


def test_bias_of_documents_and_prefixes(cuda):
    q, k, v, g = _operands(22, 2, 500, 640, 6, 2, 128, BF16)
    ids = torch.full((2, 640), -1, dtype=torch.int32)
    ids[0, :300], ids[0, 300:], ids[1, 5:77], ids[1, 77:600] = 4, 9, 1, 2
    _both((q, k, v), g, dict(scale=128 ** -0.5, causal=True, slopes=_slopes(6), documents=ids.to(cuda)), BF16)
    prefix = torch.tensor([600, 150], dtype=torch.int32, device=cuda)
    _both((q, k, v), g, dict(scale=128 ** -0.5, causal=True, slopes=_slopes(6), prefix=prefix), BF16)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("rule", ["plain", "cap", "slopes"])
def test_rows_that_see_one_key(cuda, rule, d, dtype):
    """Their weight is 1 whatever the score: gradients of queries and keys are exactly 0, that of a value its rows' sum."""
    rules = dict(scale=d ** -0.5, causal=True)
    if rule == "cap":
        rules["cap"] = 30.0
    if rule == "slopes":
        rules["slopes"] = _slopes(8)
    ids = torch.arange(200, dtype=torch.int32, device=cuda).expand(3, 200).contiguous()
    for M, documents in ((1, None), (200, ids)):
        q, k, v, g = _operands(23, 3, M, M, 8, 2, d, dtype)
        out, lse = ops.masked_attention(q, k, v, return_lse=True, documents=documents, **rules)
        dq, dk, dv = ops.masked_attention_backward(g, q, k, v, out, lse, documents=documents, **rules)
        assert torch.equal(out, v.repeat_interleave(4, 2)) and (dq == 0).all() and (dk == 0).all()
        want = g.double().view(3, M, 2, 4, d).sum(3)
        u = torch.finfo(dtype).eps / 2                  # (rounded once; weights within 2^-20 of 1 are 1 in 16 bits)
        assert ((dv.double() - want).abs() <= u * want.abs() + 2.0 ** -20 * g.double().abs().amax() * 4).all()


@pytest.mark.parametrize("prefix", [[0, 0], [1, 400], [129, 128], [-5, 127], [10 ** 9, 300]], ids=str)
def test_prefix(cuda, prefix):
    q, k, v, g = _operands(6, 2, 300, 400, 4, 2, 64, F16)
    _both((q, k, v), g, dict(scale=0.125, causal=True, prefix=torch.tensor(prefix, dtype=torch.int32, device=cuda)), F16)


@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("lengths,padding", [([1000], 0), ([1], 0), ([130, 3, 255], 40), ([128], 128), ([64, 1, 1, 500], 300)], ids=str)
@pytest.mark.parametrize("M", [500, 131])
def test_documents(cuda, M, lengths, padding, causal):
    q, k, v, g = _operands(7, 2, M, 500, 6, 2, 64, BF16)
    _both((q, k, v), g, dict(scale=0.125, causal=causal, documents=_documents(2, 500, lengths, padding)), BF16)


def test_documents_in_any_order(cuda):
    """Ids that come back, and blocks whose ranges of ids meet although no id does."""
    q, k, v, g = _operands(8, 2, 700, 700, 2, 2, 128, BF16)
    ids = torch.randint(0, 5, (2, 700), generator=torch.Generator().manual_seed(3)).int()
    ids[1, :300] = torch.arange(300) % 2 * 10
    ids[1, 300:600] = 5
    ids[1, 600:] = -3
    for causal in (False, True):
        rules = dict(scale=128 ** -0.5, causal=causal, documents=ids.to(cuda), slopes=_slopes(2), cap=20.0)
        _both((q, k, v), g, rules, BF16)
    prefix = torch.tensor([350, 10], dtype=torch.int32, device=cuda)
    _both((q, k, v), g, dict(scale=128 ** -0.5, causal=True, documents=ids.to(cuda), prefix=prefix), BF16)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_long_rows_and_many_items(cuda, dtype):
    """Two tiles an item, several items and parts of key blocks a CTA; few key heads, whose sums several CTAs share."""
    for shape in ((3, 700, 700, 60, 60, 64), (1, 2500, 2500, 8, 1, 128)):
        q, k, v, g = _operands(9, *shape, dtype)
        _both((q, k, v), g, dict(scale=shape[-1] ** -0.5, causal=True), dtype)


def test_rows_that_see_nothing(cuda):
    """More queries than keys under a causal mask, and rows of padding: zeros, -inf and zero gradients, whatever stands in the operands."""
    q, k, v, g = _operands(10, 2, 200, 100, 2, 2, 64, F16)
    out, lse, (dq, dk, dv) = _both((q, k, v), g, dict(scale=0.125, causal=True), F16)
    assert (out[:, :100] == 0).all() and (lse[:, :100] == -math.inf).all() and (dq[:, :100] == 0).all() and (out[:, 100:] != 0).any()
    ids = torch.full((2, 300), -1, dtype=torch.int32, device=cuda)
    q, k, v, g = _operands(11, 2, 300, 300, 2, 1, 64, F16)
    out, lse, grads = _both((q, k, v), g, dict(scale=0.125, documents=ids), F16)
    assert (out == 0).all() and (lse == -math.inf).all() and all((x == 0).all() for x in grads)


def test_keys_that_nobody_sees_may_be_large(cuda):
    """Masked scores are replaced, not added to: the type's largest values, and scores beyond its range, do not show."""
    q, k, v, g = _operands(12, 1, 256, 256, 2, 2, 64, BF16)
    ids = _documents(1, 256, [100])
    ids[:, 200:] = -1
    rules = dict(scale=0.125, causal=True, documents=ids)
    want = ops.masked_attention(q, k, v, **rules)
    k[:, 200:] = 3e38
    v[:, 200:] = -3e38
    assert torch.equal(want, ops.masked_attention(q, k, v, **rules))
    k[:, 200:] = math.inf
    assert torch.equal(want, ops.masked_attention(q, k, v, **rules))


def test_nan_where_it_is_seen(cuda):
    q, k, v, _ = _operands(13, 1, 100, 100, 1, 1, 64, BF16)
    k[0, 60] = math.nan
    out = ops.masked_attention(q, k, v, scale=0.125, causal=True)
    assert torch.isfinite(out[:, :60]).all() and out[:, 60:].isnan().all()


def test_large_scores(cuda):
    """Scores of thousands: references whose product with the scale is subtracted from the scores."""
    q, k, v, g = _operands(14, 1, 200, 300, 2, 2, 64, BF16)
    out, lse = ops.masked_attention(q * 30, k * 30, v, scale=1.0, return_lse=True)
    oracle = Oracle(q * 30, k * 30, v, scale=1.0)
    top = oracle.p.amax(-1)
    sure = top > 0.999                                 # rows that one key decides: the others hang on the last bits of scores of 50000
    assert sure.float().mean() > 0.9
    err = (out.double().transpose(1, 2) - oracle.o).abs().amax(-1)
    assert (err[sure] <= 0.02).all()


def test_strides(cuda):
    """Views of a packed tensor, heads in front of tokens, a result with gaps: the same bits as contiguous operands."""
    B, T, H, Hk, d = 2, 200, 4, 2, 64
    packed = torch.randn(B, T, (H + 2 * Hk) * d, device=cuda).to(BF16)
    q = packed[..., :H * d].view(B, T, H, d)
    k = packed[..., H * d:(H + Hk) * d].view(B, T, Hk, d)
    v = packed[..., (H + Hk) * d:].view(B, T, Hk, d)
    rules = dict(scale=0.125, causal=True)
    out, lse = ops.masked_attention(q.contiguous(), k.contiguous(), v.contiguous(), return_lse=True, **rules)
    got, lse2 = ops.masked_attention(q, k, v, return_lse=True, **rules)
    assert torch.equal(out, got) and torch.equal(lse, lse2)
    room = torch.full((B, H, T, d + 8), 7.0, device=cuda, dtype=BF16)
    view = room[..., :d].transpose(1, 2)
    assert ops.masked_attention(q, k, v, out=view, **rules).data_ptr() == room.data_ptr()
    assert torch.equal(view, out) and (room[..., d:] == 7).all()
    g = torch.randn(B, H, T, d, device=cuda).to(BF16).transpose(1, 2)
    want = ops.masked_attention_backward(g.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), out, lse, **rules)
    for x, y in zip(want, ops.masked_attention_backward(g, q, k, v, view, lse, **rules)):
        assert torch.equal(x, y)


def test_same_bits_every_time(cuda):
    q, k, v, g = _operands(15, 1, 1500, 1500, 8, 1, 128, F16)
    rules = dict(scale=128 ** -0.5, causal=True, cap=30.0)
    first = None
    for _ in range(4):
        out, lse = ops.masked_attention(q, k, v, return_lse=True, **rules)
        now = (out, lse, *ops.masked_attention_backward(g, q, k, v, out, lse, **rules))
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


def test_empty_operands(cuda):
    z = lambda *s: torch.zeros(s, dtype=BF16, device=cuda)  # noqa: E731
    out, lse = ops.masked_attention(z(2, 3, 4, 64), z(2, 0, 4, 64), z(2, 0, 4, 64), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert ops.masked_attention(z(0, 3, 4, 64), z(0, 5, 4, 64), z(0, 5, 4, 64)).shape == (0, 3, 4, 64)
    assert ops.masked_attention(z(2, 0, 4, 64), z(2, 5, 4, 64), z(2, 5, 4, 64)).shape == (2, 0, 4, 64)
    grads = ops.masked_attention_backward(z(2, 0, 4, 64), z(2, 0, 4, 64), z(2, 5, 2, 64), z(2, 5, 2, 64), z(2, 0, 4, 64),
                                          torch.zeros(2, 0, 4, device=cuda))
    assert [tuple(x.shape) for x in grads] == [(2, 0, 4, 64), (2, 5, 2, 64), (2, 5, 2, 64)] and all((x == 0).all() for x in grads)


def test_autograd_and_differences(cuda):
    """Gradients through autograd: those of the explicit call, with shared heads and an expanded key, and near central differences of the
    definition in 64 bits."""
    q, k, v, g = _operands(16, 2, 90, 90, 4, 2, 64, BF16)
    rules = dict(scale=0.125, causal=True, cap=10.0, slopes=_slopes(4))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = ops.masked_attention(*leaves, **rules)
    out.backward(g)
    o, lse = ops.masked_attention(q, k, v, return_lse=True, **rules)
    for x, y in zip(leaves, ops.masked_attention_backward(g, q, k, v, o, lse, **rules)):
        assert torch.equal(x.grad, y)
    # one key row for the whole batch: its gradient is the sum
    one = k[:1].clone().requires_grad_()
    ops.masked_attention(q, one.expand(2, -1, -1, -1).contiguous(), v, **rules).backward(g)
    parts = ops.masked_attention_backward(g, q, k[:1].expand(2, -1, -1, -1).contiguous(), v,
                                          *ops.masked_attention(q, k[:1].expand(2, -1, -1, -1).contiguous(), v, return_lse=True, **rules), **rules)
    assert torch.equal(one.grad, parts[1].sum(0, keepdim=True))
    # only what asks for one gets one; a gradient that is expanded is no fault
    leaf = q.clone().requires_grad_()
    ops.masked_attention(leaf, k, v, **rules).float().sum().backward()
    assert torch.isfinite(leaf.grad).all()
    # differences: f(x + h e) - f(x - h e) of the definition, along random directions
    gen = torch.Generator(device=cuda).manual_seed(1)
    grads = [x.grad.double() for x in leaves]
    for i in range(3):
        e = torch.randn(leaves[i].shape, generator=gen, device=cuda, dtype=torch.float64)
        f = []
        for h in (1e-4, -1e-4):
            moved = [t.double() for t in (q, k, v)]
            moved[i] = moved[i] + h * e
            f.append((Oracle(*moved, **rules).out * g.double()).sum())
        slope = (f[0] - f[1]) / 2e-4
        got = (grads[i] * e).sum()
        # a sum of n rounded terms with random signs: a few times u sqrt(sum of squares)
        assert (got - slope).abs() <= 8 * 2.0 ** -8 * (grads[i] * e).square().sum().sqrt() + 1e-3 * slope.abs()


def test_streams_and_graphs(cuda):
    """On a side stream, captured and replayed with new contents; two graphs have scratch memory of their own."""
    B, T, H, d = 2, 400, 4, 64
    q, k, v, g = _operands(17, B, T, T, H, H, d, BF16)
    ids = _documents(B, T, [90, 33])
    rules = dict(scale=0.125, causal=True, documents=ids)

    def step():
        out, lse = ops.masked_attention(q, k, v, return_lse=True, **rules)
        return (out, lse, *ops.masked_attention_backward(g, q, k, v, out, lse, **rules))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step()
        graphs.append((graph, kept))
    q.copy_(torch.randn_like(q))
    ids.copy_(_documents(B, T, [17, 200]))
    want = step()
    for graph, kept in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, kept in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, kept))
    assert ops.device_status(cuda) == 0


def test_backward_of_autograd_under_capture(cuda):
    """A training step captured whole, its leaves used by no other graph."""
    q, k, v, g = (t.requires_grad_() if i < 3 else t for i, t in enumerate(_operands(18, 1, 130, 130, 2, 2, 64, BF16)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            grads = torch.autograd.grad(ops.masked_attention(q, k, v, scale=0.125, causal=True), (q, k, v), g)
    torch.cuda.current_stream().wait_stream(side)
    want = [x.clone() for x in grads]
    del grads
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ops.masked_attention(q, k, v, scale=0.125, causal=True), (q, k, v), g)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals(cuda):
    q, k, v, g = _operands(19, 2, 32, 32, 4, 2, 64, BF16)
    call = ops.masked_attention
    for bad, kind in ((dict(scale=0.0), ValueError), (dict(scale=math.inf), ValueError), (dict(scale=math.nan), ValueError), (dict(cap=-1.0), ValueError),
                      (dict(cap=0.0), ValueError), (dict(prefix=torch.zeros(2, dtype=torch.int32, device=cuda)), ValueError),
                      (dict(causal=True, prefix=torch.zeros(3, dtype=torch.int32, device=cuda)), ValueError),
                      (dict(causal=True, prefix=torch.zeros(2, dtype=torch.int64, device=cuda)), TypeError),
                      (dict(slopes=torch.zeros(3, device=cuda)), ValueError), (dict(slopes=torch.zeros(4, device=cuda, dtype=BF16)), TypeError),
                      (dict(slopes=torch.zeros(4, device=cuda, requires_grad=True)), ValueError),
                      (dict(documents=torch.zeros(2, 31, dtype=torch.int32, device=cuda)), ValueError),
                      (dict(documents=torch.zeros(2, 64, dtype=torch.int32, device=cuda)[:, ::2]), ValueError),
                      (dict(out=torch.empty(2, 32, 4, 64, device=cuda)), TypeError), (dict(out=torch.empty(2, 31, 4, 64, device=cuda, dtype=BF16)), ValueError)):
        with pytest.raises(kind):
            call(q, k, v, **bad)
    for bad, kind in (((q.float(), k, v), TypeError), ((q, k.half(), v), TypeError), ((q.cpu(), k, v), TypeError), ((q, k[:1], v[:1]), ValueError),
                      ((q, k, v[:, :16]), ValueError), ((q[:, :, :3], k, v), ValueError), ((q[..., :60], k[..., :60], v[..., :60]), ValueError),
                      ((q.transpose(2, 3), k, v), ValueError), ((q[0], k, v), ValueError), ((q[:1].expand(2, -1, -1, -1), k, v), ValueError),
                      ((torch.zeros(2, 32, 4, 136, device=cuda, dtype=BF16),) * 3, ValueError),
                      ((torch.zeros(2 * 32 * 4 * 64 + 1, device=cuda, dtype=BF16)[1:].view(2, 32, 4, 64), k, v), ValueError)):
        with pytest.raises(kind):
            call(*bad)
    with pytest.raises(ValueError):
        call(q, k[:, :16], v[:, :16], documents=torch.zeros(2, 16, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError):
        call(q.clone().requires_grad_(), k, v, out=torch.empty_like(q))
    out, lse = call(q, k, v, return_lse=True)
    for bad in ((g[:1], q, k, v, out, lse), (g, q, k, v, out, lse[:, :1]), (g, q, k, v, out[:1], lse)):
        with pytest.raises(ValueError):
            ops.masked_attention_backward(*bad)
    with pytest.raises(TypeError):
        ops.masked_attention_backward(g.half(), q, k, v, out, lse)
    assert ops.device_status(cuda) == 0


def test_python_path_gives_the_same(cuda):
    """The checked path in Python, which serves calls where the native one was not built."""
    q, k, v, g = _operands(20, 2, 140, 140, 4, 2, 72, F16)
    rules = dict(scale=0.1, causal=True, prefix=torch.tensor([9, 130], dtype=torch.int32, device=cuda), slopes=_slopes(4), cap=9.0)
    def step():
        out, lse = ops.masked_attention(q, k, v, return_lse=True, **rules)
        return (out, lse, *ops.masked_attention_backward(g, q, k, v, out, lse, **rules))
    step()
    fast = ops._fast
    assert fast is not None
    want = step()
    try:
        ops._fast = None
        got = step()
    finally:
        ops._fast = fast
    assert all(torch.equal(a, b) for a, b in zip(want, got))
