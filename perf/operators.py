"""Masked attention with its gradients, attention over a paged key/value cache, and the cache's page operations, as
cases that can be timed.

A case is a dict of plain values.  `kind` names the operator:

  masked   attention over dense tensors whose scores are capped by a tanh or get a bias by distance, under a causal,
           prefix or document mask; with "train" the pass returns the gradients too
  paged    one step of a serving program: the new tokens' keys and values are appended to a paged cache, and the new
           tokens attend to their sequences (a chunk of tokens each, a single token each, or a mixture)
  fork     sequences of a paged cache are freed and forked again from others: full pages are shared, the last is copied
  compact  the live pages of a pool move to its front

`own` False computes an operator in its plain form, with elementary torch operations in 32 bits; True makes the calls
of `ditto_b200.ops`.
"""
import math
import random

import torch

own = False

_DTYPE = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # a short prompt that sees itself whole, with the tokens that follow it: the smallest call, inference
        {"name": "prefix-197-tokens", "kind": "masked", "train": False, "batch": 1, "M": 197, "L": 197, "heads": 12, "kv_heads": 12,
         "d": 64, "dtype": "float16", "mask": "prefix", "slopes": False, "cap": 0.0},
        # a training step over rows packed with documents of many lengths
        {"name": "documents-4x4096-train", "kind": "masked", "train": True, "batch": 4, "M": 4096, "L": 4096, "heads": 16, "kv_heads": 16,
         "d": 64, "dtype": "bfloat16", "mask": "documents", "slopes": False, "cap": 0.0},
        # a training step with capped scores and shared key heads, an odd length
        {"name": "capped-2x2047-train", "kind": "masked", "train": True, "batch": 2, "M": 2047, "L": 2047, "heads": 16, "kv_heads": 4,
         "d": 128, "dtype": "bfloat16", "mask": "causal", "slopes": False, "cap": 30.0},
        # one long text with a bias by distance: the largest training work
        {"name": "distance-8192-train", "kind": "masked", "train": True, "batch": 1, "M": 8192, "L": 8192, "heads": 16, "kv_heads": 2,
         "d": 128, "dtype": "float16", "mask": "causal", "slopes": True, "cap": 0.0},
        # four short conversations, a token each: all latency
        {"name": "decode-4-short", "kind": "paged", "new": "single", "batch": 4, "longest": 600, "chunk": 1, "heads": 8, "kv_heads": 2,
         "d": 64, "page": 16, "dtype": "float16", "slopes": False, "cap": 0.0, "prefix": False},
        # a full serving batch of ragged lengths, a token each: reads the cache
        {"name": "decode-64-ragged", "kind": "paged", "new": "single", "batch": 64, "longest": 16384, "chunk": 1, "heads": 32, "kv_heads": 8,
         "d": 128, "page": 64, "dtype": "bfloat16", "slopes": False, "cap": 0.0, "prefix": False},
        # chunks of some sequences among single tokens of the others, capped scores
        {"name": "mixed-16-capped", "kind": "paged", "new": "mixed", "batch": 16, "longest": 4500, "chunk": 500, "heads": 32, "kv_heads": 8,
         "d": 128, "page": 32, "dtype": "bfloat16", "slopes": False, "cap": 50.0, "prefix": False},
        # the second half of a long prompt over the first, with a bias by distance: the largest chunk
        {"name": "chunk-8192-of-16384", "kind": "paged", "new": "chunk", "batch": 1, "longest": 16384, "chunk": 8192, "heads": 16,
         "kv_heads": 2, "d": 128, "page": 128, "dtype": "float16", "slopes": True, "cap": 0.0, "prefix": False},
        # two prompts sampled three times each
        {"name": "fork-2x3", "kind": "fork", "parents": 2, "children": 3, "longest": 300, "layers": 4, "kv_heads": 2, "d": 64, "page": 16,
         "dtype": "float16"},
        # a batch of beams: 32 prompts, eight each
        {"name": "fork-32x8", "kind": "fork", "parents": 32, "children": 8, "longest": 2000, "layers": 8, "kv_heads": 8, "d": 128, "page": 64,
         "dtype": "bfloat16"},
        # a small pool, half in use
        {"name": "compact-200-pages", "kind": "compact", "pages": 200, "sequences": 10, "per": 12, "layers": 4, "kv_heads": 2, "d": 64,
         "page": 16, "dtype": "float16"},
        # a pool of some GB after many sequences have ended
        {"name": "compact-2000-pages", "kind": "compact", "pages": 2000, "sequences": 50, "per": 24, "layers": 8, "kv_heads": 8, "d": 128,
         "page": 64, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["masked", "masked", "masked", "paged", "paged", "paged", "fork", "compact"])
    dtype = rng.choice(["float16", "bfloat16"])
    heads, kv_heads = rng.choice([(12, 12), (16, 16), (16, 4), (16, 2), (8, 1), (6, 2), (32, 8), (7, 1), (10, 2), (24, 4)])
    d = rng.choice([64, 64, 128, 128, 128, 80, 96, 40])
    slopes, cap = rng.choice([(False, 0.0), (False, 0.0), (True, 0.0), (False, 30.0), (False, 50.0), (True, 20.0)])
    if kind == "masked":
        while True:
            batch, L = _log(rng, 1, 6), _log(rng, 1, 8192)
            M = L if rng.random() < 0.8 else _log(rng, 1, L)
            if batch * heads * M * L <= 1.0e9:
                break
        return {"kind": kind, "train": rng.random() < 0.7, "batch": batch, "M": M, "L": L, "heads": heads, "kv_heads": kv_heads, "d": d,
                "dtype": dtype, "mask": rng.choice(["causal", "prefix", "documents", "documents", "both-ways", "full"]), "slopes": slopes,
                "cap": cap}
    page = rng.choice([16, 16, 32, 64, 64, 128, 256])
    if kind == "paged":
        while True:
            batch, longest = _log(rng, 1, 128), _log(rng, 16, 32768)
            new = rng.choice(["single", "single", "mixed", "chunk"])
            chunk = 1 if new == "single" else _log(rng, 2, min(longest, 4096))
            if batch * longest * kv_heads * d <= 6.0e8 and batch * heads * chunk * longest <= 1.5e9:
                break
        return {"kind": kind, "new": new, "batch": batch, "longest": longest, "chunk": chunk, "heads": heads, "kv_heads": kv_heads, "d": d,
                "page": page, "dtype": dtype, "slopes": slopes, "cap": cap, "prefix": rng.random() < 0.2}
    while True:
        layers = _log(rng, 1, 16)
        if kind == "fork":
            c = {"kind": kind, "parents": _log(rng, 1, 32), "children": _log(rng, 1, 8), "longest": _log(rng, 1, 4000)}
            pages = c["parents"] * (-(-c["longest"] // page) + 2 * c["children"])
        else:
            c = {"kind": kind, "pages": _log(rng, 4, 4000), "per": _log(rng, 1, 32)}
            c["sequences"] = max(1, int(c["pages"] * rng.uniform(0.2, 0.95)) // c["per"])
            pages = max(c["pages"], c["sequences"] * c["per"])
            c["pages"] = pages
        if pages * layers * 2 * page * kv_heads * d <= 2.0e9:
            break
    return {**c, "layers": layers, "kv_heads": kv_heads, "d": d, "page": page, "dtype": dtype}


# ------------------------------------------------------------------ what a case fixes apart from the seed


def _rng(case):
    return random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))


def _documents(case):
    """Document of each position, a list for each row: lengths spread over the logarithm, the rest of a row is padding (-1)."""
    rng, L, rows = _rng(case), case["L"], []
    for _ in range(case["batch"]):
        ids, end = [], L - (rng.randint(0, L // 16) if rng.random() < 0.5 else 0)
        while len(ids) < end:
            ids += [len(rows) * 1000 + len(set(ids))] * min(end - len(ids), _log(rng, max(1, L // 32), max(1, L // 2)))
        rows.append(ids + [-1] * (L - end))
    return rows


def _prefixes(case, longest):
    rng = _rng(case)
    return [rng.randint(0, longest) for _ in range(case["batch"])]


def _lengths(case):
    """Lengths with the new tokens, and how many of them are new, for each sequence."""
    rng, top = _rng(case), case["longest"]
    lengths = [top] + [rng.randint(max(1, top // 8), top) for _ in range(case["batch"] - 1)]
    if case["new"] == "single":
        new = [1] * len(lengths)
    elif case["new"] == "chunk":
        new = [min(n, case["chunk"]) for n in lengths]
    else:
        new = [min(n, case["chunk"]) if i % 4 == 0 else 1 for i, n in enumerate(lengths)]
    return lengths, new


def _parents(case):
    rng = _rng(case)
    return [case["longest"]] + [rng.randint(max(1, case["longest"] // 8), case["longest"]) for _ in range(case["parents"] - 1)]


def _live(case):
    """How many pages a compact case has in use (every second sequence shares half its pages with the one before), and where."""
    n = case["sequences"] * case["per"] - (case["sequences"] // 2) * (case["per"] // 2)
    return n, _rng(case).sample(range(case["pages"]), n)


def _pairs(case):
    """(query, key) pairs that the masks leave, for one head over all rows."""
    M, L, mask = case["M"], case["L"], case["mask"]
    if mask == "full":
        return case["batch"] * M * L
    pos = range(L - M, L)
    if mask in ("causal", "prefix"):
        p = _prefixes(case, L) if mask == "prefix" else [0] * case["batch"]
        return sum(max(i + 1, p[b]) for b in range(case["batch"]) for i in pos)
    total = 0
    for ids in _documents(case):
        first, count = {}, {}
        for j, x in enumerate(ids):
            first.setdefault(x, j)
            count[x] = count.get(x, 0) + 1
        total += sum(0 if ids[i] < 0 else (i - first[ids[i]] + 1 if mask == "documents" else count[ids[i]]) for i in pos)
    return total


def work(case):
    """Every input read once and every result written once; two operations per multiply-add of the products over the
    visible pairs: two products forward, five backward."""
    if case["kind"] == "masked":
        b, h, kh, d = case["batch"], case["heads"], case["kv_heads"], case["d"]
        q, kv, rows = b * case["M"] * h * d, b * case["L"] * kh * d, b * case["M"] * h
        each = 2.0 * d * h * _pairs(case)
        if not case["train"]:
            return {"bytes": 2.0 * (2 * q + 2 * kv) + 4.0 * rows, "flops": 2 * each}
        # forward: q, k, v, out, lse; backward: the same read, with the gradient of out, and three gradients written
        return {"bytes": 2.0 * (2 * q + 2 * kv) + 4.0 * rows + 2.0 * (4 * q + 4 * kv) + 4.0 * rows, "flops": 7 * each}
    if case["kind"] == "paged":
        lengths, new = _lengths(case)
        kv = case["kv_heads"] * case["d"] * 2 * 2.0
        pairs = sum(n * m - m * (m - 1) // 2 for n, m in zip(lengths, new))
        if case["prefix"]:
            pairs = sum(max(n - m + t + 1, min(p, n)) for n, m, p in zip(lengths, new, _prefixes(case, case["longest"])) for t in range(m))
        return {"bytes": kv * sum(lengths) + 2 * kv * sum(new) + 2 * 2.0 * sum(new) * case["heads"] * case["d"],
                "flops": 4.0 * case["heads"] * case["d"] * pairs}
    page = case["layers"] * 2 * case["page"] * case["kv_heads"] * case["d"] * 2.0
    if case["kind"] == "fork":
        lengths, c = _parents(case), case["children"]
        tables = 8.0 * sum(-(-n // case["page"]) for n in lengths) * (1 + 2 * c)
        return {"bytes": 2 * page * c * sum(n % case["page"] != 0 for n in lengths) + tables, "flops": 0.0}
    n, at = _live(case)
    return {"bytes": 2 * page * sum(p >= n for p in at) + 8.0 * (case["pages"] + case["sequences"] * case["per"]), "flops": 0.0}


# ------------------------------------------------------------------ inputs


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kh, d = _DTYPE[case["dtype"]], case["kv_heads"], case["d"]

    def normal(*shape):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)

    def order(n):
        return torch.randperm(n, generator=gen, device="cuda")

    state = {"case": case}
    if case["kind"] in ("masked", "paged"):
        state["rules"] = {"scale": d ** -0.5, "cap": case["cap"] or None, "slopes": _slopes(case["heads"]) if case["slopes"] else None}
    if case["kind"] == "masked":
        b, M, L, h = case["batch"], case["M"], case["L"], case["heads"]
        state["q"], state["k"], state["v"] = normal(b, M, h, d), normal(b, L, kh, d), normal(b, L, kh, d)
        state["rules"]["causal"] = case["mask"] in ("causal", "prefix", "documents")
        if case["mask"] == "prefix":
            state["rules"]["prefix"] = _int(_prefixes(case, L))
        if case["mask"] in ("documents", "both-ways"):
            state["rules"]["documents"] = _int(_documents(case))
        if case["train"]:
            state["grad"] = normal(b, M, h, d)
        return state
    if case["kind"] == "paged":
        lengths, new = _lengths(case)
        page, n = case["page"], [-(-x // case["page"]) for x in lengths]
        pages = sum(n) + sum(n) // 16 + 1
        state["kp"], state["vp"] = normal(pages, page, kh, d), normal(pages, page, kh, d)
        table = torch.full((len(n), max(n)), -1, dtype=torch.int32, device="cuda")
        used = torch.arange(max(n), device="cuda")[None, :] < _int(n)[:, None]
        table[used] = order(pages)[: sum(n)].int()
        tokens = sum(new)
        state.update(table=table, lengths=_int(lengths), q=normal(tokens, case["heads"], d), k=normal(tokens, kh, d), v=normal(tokens, kh, d),
                     most=max(new), longest=max(lengths))
        # the slots behind a sequence's end hold what other sequences left there
        state["starts"] = None if case["new"] == "single" else _int([sum(new[:i]) for i in range(len(new) + 1)])
        if case["prefix"]:
            state["rules"]["prefix"] = _int(_prefixes(case, case["longest"]))
        return state
    page, layers = case["page"], case["layers"]
    if case["kind"] == "fork":
        # the state behind an earlier fork: the children share their parents' full pages and own a last page at the pool's end
        lengths, c = _parents(case), case["children"]
        n, P = [-(-x // page) for x in lengths], case["parents"]
        tails = sum(x % page != 0 for x in lengths) * c
        pages = sum(n) + 2 * tails
        table = torch.full((P * (1 + c), max(n)), -1, dtype=torch.int32)
        own_pages = order(sum(n) + tails)[: sum(n)].int().cpu()
        at, tail, refs = 0, pages - tails, torch.zeros(pages, dtype=torch.int32)
        for i, x in enumerate(lengths):
            rows = [i] + [P + i * c + k for k in range(c)]
            table[rows, : n[i]] = own_pages[at: at + n[i]]
            refs[own_pages[at: at + n[i]].long()] = 1 + c
            if x % page:
                refs[own_pages[at + n[i] - 1]] = 1
                for r in rows[1:]:
                    table[r, n[i] - 1], refs[tail] = tail, 1
                    tail += 1
            at += n[i]
        parents = [i for i in range(P) for _ in range(c)]
        state.update(table=table.cuda(), references=refs.cuda(), lengths=_int(lengths + [lengths[i] for i in parents]),
                     parents=_int(parents), children=_int(list(range(P, P * (1 + c)))), pools=normal(2 * layers, pages, page, kh, d))
        return state
    n, at = _live(case)
    S, per, half = case["sequences"], case["per"], case["per"] // 2
    mine = torch.tensor(at, device="cuda")[order(n)].int().cpu()
    table, taken = torch.empty((S, per), dtype=torch.int32), 0
    for s in range(S):
        shared = half if s % 2 else 0
        if shared:
            table[s, :shared] = table[s - 1, :shared]
        table[s, shared:] = mine[taken: taken + per - shared]
        taken += per - shared
    refs = torch.bincount(table.reshape(-1).long(), minlength=case["pages"]).int()
    state.update(table=table.cuda(), references=refs.cuda(), pools=normal(2 * layers, case["pages"], page, kh, d), most=min(n, case["pages"] - n))
    return state


# ------------------------------------------------------------------ the plain forms


def _modified(s, rules, distance):
    """Scores behind the cap and the bias by distance, and what the cap's derivative is made of."""
    t = None
    if rules["cap"]:
        t = torch.tanh(s / rules["cap"])
        s = rules["cap"] * t
    if rules["slopes"] is not None:
        s = s - rules["slopes"].view(s.shape[1], s.shape[2], 1, 1) * distance.abs()
    return s, t


def _softmax(s, seen):
    """exp(s - lse) over what is seen, and lse; rows that see nothing get zeros and -inf."""
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total), (top + torch.log(total)).squeeze(-1)


def _plain_masked(state):
    case, rules = state["case"], state["rules"]
    q, k, v = state["q"], state["k"], state["v"]
    b, M, h, d = q.shape
    L, kh = k.shape[1], k.shape[2]
    qf = q.float().view(b, M, kh, h // kh, d).permute(0, 2, 3, 1, 4)
    kf, vf = (t.float().permute(0, 2, 1, 3).unsqueeze(2) for t in (k, v))
    pos, key = torch.arange(L - M, L, device=q.device), torch.arange(L, device=q.device)
    seen = torch.ones((1, M, L), dtype=torch.bool, device=q.device)
    if rules["causal"]:
        seen = (key[None, :] <= pos[:, None]).unsqueeze(0)
    if rules.get("prefix") is not None:
        seen = seen | (key[None, None, :] < rules["prefix"][:, None, None])
    if rules.get("documents") is not None:
        doc = rules["documents"]
        mine = doc[:, L - M:, None]
        seen = seen & (mine == doc[:, None, :]) & (mine >= 0)
    seen = seen.view(seen.shape[0], 1, 1, M, L)
    s, t = _modified(rules["scale"] * (qf @ kf.transpose(-1, -2)), rules, (pos[:, None] - key[None, :]).float())
    p, lse = _softmax(s, seen)
    o = p @ vf
    rows = lambda x: x.permute(0, 3, 1, 2, 4).reshape(b, M, h, d)  # noqa: E731
    answer = {"out": rows(o).to(q.dtype), "lse": lse.permute(0, 3, 1, 2).reshape(b, M, h)}
    if case["train"]:
        g = state["grad"].float().view(b, M, kh, h // kh, d).permute(0, 2, 3, 1, 4)
        ds = p * (g @ vf.transpose(-1, -2) - (g * o).sum(-1, keepdim=True))
        if t is not None:
            ds = ds * (1 - t * t)
        ds = ds * rules["scale"]
        columns = lambda x: x.sum(2).permute(0, 2, 1, 3).to(q.dtype)  # noqa: E731
        answer.update(dq=rows(ds @ kf).to(q.dtype), dk=columns(ds.transpose(-1, -2) @ qf), dv=columns(p.transpose(-1, -2) @ g))
    return answer


def _plain_paged(state):
    case, rules, q = state["case"], state["rules"], state["q"]
    kp, vp, table, lengths = state["kp"], state["vp"], state["table"], state["lengths"]
    batch, page, tokens, h, d = len(lengths), case["page"], len(q), case["heads"], case["d"]
    kh, dev = case["kv_heads"], q.device
    starts = state["starts"] if state["starts"] is not None else torch.arange(batch + 1, device=dev, dtype=torch.int32)
    new = starts[1:] - starts[:-1]
    # append
    token = torch.arange(tokens, device=dev)
    seq = torch.bucketize(token, starts[1:].contiguous(), right=True)
    slot = lengths[seq] - new[seq] + (token - starts[seq])
    where = (table[seq, (slot // page).long()].long(), (slot % page).long())
    kp[where], vp[where] = state["k"], state["v"]
    # the sequences side by side, the new tokens of each in a row
    key = torch.arange(state["longest"], device=dev)
    at = table[:, key // page].clamp(min=0).long()
    kf, vf = (t[at, key % page].float().permute(0, 2, 1, 3).unsqueeze(2) for t in (kp, vp))
    step = torch.arange(state["most"], device=dev)
    qf = q[(starts[:-1, None] + step).clamp(max=tokens - 1).long()].float().view(batch, len(step), kh, h // kh, d).permute(0, 2, 3, 1, 4)
    pos = (lengths - new)[:, None] + step
    seen = key[None, None, :] <= pos[:, :, None]
    if rules.get("prefix") is not None:
        seen = seen | (key[None, None, :] < rules["prefix"][:, None, None])
    seen = seen & (key[None, None, :] < lengths[:, None, None])
    distance = (pos[:, :, None] - key[None, None, :]).float()[:, None, None]
    s, _ = _modified(rules["scale"] * (qf @ kf.transpose(-1, -2)), rules, distance)
    p, _ = _softmax(s, seen[:, None, None])
    o = (p @ vf).permute(0, 3, 1, 2, 4).reshape(batch, len(step), h, d)
    return {"out": o[seq, (token - starts[seq]).long()].to(q.dtype), "keys": kp, "values": vp}


def _plain_fork(state):
    table, lengths, refs, pools = state["table"], state["lengths"], state["references"], state["pools"]
    parents, children, page = state["parents"].long(), state["children"].long(), state["case"]["page"]
    # free the children
    old = table[children]
    refs.index_add_(0, old.clamp(min=0).reshape(-1).long(), -(old >= 0).int().reshape(-1))
    # the k-th child that needs a page takes the k-th free one
    free = torch.sort((refs > 0).int(), stable=True).indices
    full, partial = lengths[parents] // page, lengths[parents] % page != 0
    target = free[(torch.cumsum(partial, 0) - 1).clamp(min=0)]
    column = torch.arange(table.shape[1], device=table.device)
    row = torch.where(column < full[:, None], table[parents], -1)
    row = torch.where((column == full[:, None]) & partial[:, None], target[:, None].int(), row)
    table[children] = row
    lengths[children] = lengths[parents]
    refs.index_add_(0, row.clamp(min=0).reshape(-1).long(), (row >= 0).int().reshape(-1))
    source = table[parents, full.clamp(max=table.shape[1] - 1).long()].long().clamp(min=0)
    pools[:, torch.where(partial, target, source)] = pools[:, source]
    return {"table": table, "lengths": lengths, "references": refs, "pools": pools}


def _plain_compact(state):
    table, refs, pools = state["table"], state["references"], state["pools"]
    pages, most = len(refs), state["most"]
    live = refs > 0
    n = live.sum()
    at = torch.arange(pages, device=refs.device)
    # the k-th live page behind the first n places moves to the k-th free one among them; lists longer than the moves repeat the
    # first of them, or copy a page onto itself where there is none
    source = torch.sort((~(live & (at >= n))).int(), stable=True).indices[:most]
    target = torch.sort((~(~live & (at < n))).int(), stable=True).indices[:most]
    moves = live[source] & (source >= n)
    target = torch.where(moves, target, source)
    source, target = torch.where(moves, source, source[:1]), torch.where(moves, target, target[:1])
    pools[:, target] = pools[:, source]
    renamed = at.clone()
    renamed[source] = target
    counts = refs.clone()
    counts[source] = 0
    counts[target] = refs[source]
    return {"table": torch.where(table >= 0, renamed[table.clamp(min=0).long()].int(), table), "references": counts, "pools": pools}


# ------------------------------------------------------------------ a pass


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"masked": _plain_masked, "paged": _plain_paged, "fork": _plain_fork, "compact": _plain_compact}[kind](state)
    from ditto_b200 import ops
    if kind == "masked":
        out, lse = ops.masked_attention(state["q"], state["k"], state["v"], return_lse=True, **state["rules"])
        if not state["case"]["train"]:
            return {"out": out, "lse": lse}
        dq, dk, dv = ops.masked_attention_backward(state["grad"], state["q"], state["k"], state["v"], out, lse, **state["rules"])
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if kind == "paged":
        ops.cache_append(state["k"], state["v"], state["kp"], state["vp"], state["table"], state["lengths"], state["starts"])
        out = ops.paged_attention(state["q"], state["kp"], state["vp"], state["table"], state["lengths"], state["starts"], **state["rules"])
        return {"out": out, "keys": state["kp"], "values": state["vp"]}
    pools = list(state["pools"].unbind(0))
    if kind == "fork":
        ops.cache_free(state["table"], state["lengths"], state["references"], state["children"])
        ops.cache_fork(pools, state["table"], state["lengths"], state["references"], state["parents"], state["children"],
                       state["case"]["page"])
        return {"table": state["table"], "lengths": state["lengths"], "references": state["references"], "pools": state["pools"]}
    table, references = ops.cache_compact(pools, state["table"], state["references"])
    return {"table": table, "references": references, "pools": state["pools"]}


# ------------------------------------------------------------------ the definition in 64 bits


def _exact_head(q, k, v, rules, slope, pos, seen, g=None):
    """One head in 64 bits: q [M, d], k and v [L, d], seen [M, L]; out, lse and, with g, the three gradients."""
    q, k, v = q.double(), k.double(), v.double()
    x = (q @ k.T).mul_(rules["scale"])
    t = None
    if rules["cap"]:
        t = torch.tanh(x / rules["cap"])
        x = t * rules["cap"]
    if slope is not None:
        x -= slope.double() * (pos[:, None] - torch.arange(len(k), device=q.device)).abs()
    x.masked_fill_(~seen, -math.inf)
    lse = torch.logsumexp(x, 1)
    w = x.sub_(torch.where(lse == -math.inf, 0.0, lse)[:, None]).exp_()
    out = w @ v
    if g is None:
        return out, lse
    g = g.double()
    dv = w.T @ g
    ds = (g @ v.T).sub_((g * out).sum(1, keepdim=True)).mul_(w).mul_(rules["scale"])
    if t is not None:
        ds *= 1 - t * t
    return out, lse, ds @ k, ds.T @ q, dv


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None
    state = prepare(case, seed)
    rules, h, kh, d = state["rules"], case["heads"], case["kv_heads"], case["d"]
    slope = lambda i: None if rules["slopes"] is None else rules["slopes"][i]  # noqa: E731
    if case["kind"] == "masked":
        b, M, L = case["batch"], case["M"], case["L"]
        q, k, v = state["q"], state["k"], state["v"]
        pos, key = torch.arange(L - M, L, device="cuda"), torch.arange(L, device="cuda")
        zero = lambda *s: torch.zeros(s, dtype=torch.float64, device="cuda")  # noqa: E731
        answer = {"out": zero(b, M, h, d), "lse": zero(b, M, h)}
        if case["train"]:
            answer.update(dq=zero(b, M, h, d), dk=zero(b, L, kh, d), dv=zero(b, L, kh, d))
        for i in range(b):
            seen = torch.ones(M, L, dtype=torch.bool, device="cuda")
            if rules["causal"]:
                seen = pos[:, None] >= key
                if rules.get("prefix") is not None:
                    seen = seen | (key < rules["prefix"][i])
            if rules.get("documents") is not None:
                ids = rules["documents"][i]
                seen = seen & (ids[pos][:, None] == ids) & (ids >= 0)
            for j in range(h):
                n = j * kh // h
                r = _exact_head(q[i, :, j], k[i, :, n], v[i, :, n], rules, slope(j), pos, seen, state["grad"][i, :, j] if case["train"] else None)
                answer["out"][i, :, j], answer["lse"][i, :, j] = r[0], r[1]
                if case["train"]:
                    answer["dq"][i, :, j] = r[2]
                    answer["dk"][i, :, n] += r[3]
                    answer["dv"][i, :, n] += r[4]
        return answer
    lengths, new = _lengths(case)
    if sum(m * n for m, n in zip(new, lengths)) * h > 4e9 or case["batch"] * h > 8192:
        return None
    out, first = torch.zeros(sum(new), h, d, dtype=torch.float64, device="cuda"), 0
    for i, (n, m) in enumerate(zip(lengths, new)):
        at = torch.arange(n, device="cuda")
        where = (state["table"][i, at // case["page"]].long(), at % case["page"])
        k, v = (torch.cat([p[where][: n - m], t[first: first + m]]) for p, t in ((state["kp"], state["k"]), (state["vp"], state["v"])))
        seen = at <= at[n - m:, None]
        if case["prefix"]:
            seen = seen | (at < rules["prefix"][i])
        for j in range(h):
            out[first: first + m, j] = _exact_head(state["q"][first: first + m, j], k[:, j * kh // h], v[:, j * kh // h], rules, slope(j),
                                                   at[n - m:], seen)[0]
        first += m
    return {"out": out, "keys": None, "values": None}
