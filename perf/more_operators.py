"""Measured cases of the serving operators for drafted trees and shared pages.

A step that verifies drafted tokens lays out every request's tree and takes over what the sampled tokens confirm
(tree), lets all its new tokens attend to the request's pages and to the nodes above them (attend) and applies
penalties, biases and grammar masks to every row of logits (rules); between steps requests are forked, reordered, cut
and ended over pages that they share (fork).  Each case is one call of one of them (the tree's two calls, the fork with
the copies that it asks for), as a program that serves a model makes it: in its plain form in elementary torch
operations, or (own) through llm-project_amd/qllama.py.

Shapes are those of the benchmark's models: "tiny" (6 query and 2 KV heads of 48), "1b" (32 and 8 of 64), "8b" (32
and 8 of 128), with their context lengths and vocabularies.  Lengths, trees and settings of a case follow from its "mix"
number, the contents from the seed.
"""
import importlib.util
import math
import os
import random

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADS = {"tiny": (6, 2, 48), "1b": (32, 8, 64), "8b": (32, 8, 128)}      # query heads, KV heads, head_dim
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


def listed():
    return [
        # a few requests' small trees: latency is all of it
        {"name": "tree_few", "kind": "tree", "requests": 4, "nodes": 8, "mix": 1},
        # a full batch with large trees
        {"name": "tree_batch", "kind": "tree", "requests": 200, "nodes": 64, "mix": 2},
        # one request of a small model with a small tree
        {"name": "attend_tiny", "kind": "attend", "shape": "tiny", "type": "f32", "page": 16, "requests": 1, "most": 200, "nodes": 8, "chain": False, "mix": 3},
        # the headline model's layer: 32 ragged requests with trees of up to 16 nodes
        {"name": "attend_8b", "kind": "attend", "shape": "8b", "type": "bf16", "page": 16, "requests": 32, "most": 2560, "nodes": 16, "chain": False, "mix": 4},
        # pieces of prompts, every token behind the one before
        {"name": "attend_chunk", "kind": "attend", "shape": "1b", "type": "f32", "page": 16, "requests": 6, "most": 2048, "nodes": 200, "chain": True, "mix": 5},
        # two requests over long documents with large trees, pages of 64
        {"name": "attend_long", "kind": "attend", "shape": "8b", "type": "f16", "page": 64, "requests": 2, "most": 60000, "nodes": 48, "chain": False, "mix": 6},
        # a large batch on an 8-bit cache, a short draft each
        {"name": "attend_i8", "kind": "attend", "shape": "8b", "type": "i8", "page": 32, "requests": 64, "most": 4100, "nodes": 7, "chain": False, "mix": 7},
        # two prompts continued by four samples each
        {"name": "fork_samples", "kind": "fork", "shape": "1b", "type": "f16", "page": 16, "layers": 2, "groups": 2, "old": 1, "new": 4, "most": 700, "mix": 8},
        # 32 searches of 8 beams each change places, in all 16 layers
        {"name": "fork_beams", "kind": "fork", "shape": "1b", "type": "bf16", "page": 16, "layers": 16, "groups": 32, "old": 8, "new": 8, "most": 600, "mix": 9},
        # a few rows with a common repetition penalty
        {"name": "rules_few", "kind": "rules", "requests": 4, "nodes": 1, "vocab": 128256, "history": 1500, "masks": 0, "mix": 10},
        # the rows of drafted trees, some requests behind a grammar
        {"name": "rules_tree", "kind": "rules", "requests": 40, "nodes": 9, "vocab": 32000, "history": 1000, "masks": 60, "mix": 11},
        # a full batch of long conversations, every request with settings of its own
        {"name": "rules_batch", "kind": "rules", "requests": 192, "nodes": 1, "vocab": 128256, "history": 8000, "masks": 40, "mix": 12},
    ]


def _log(rng, lo, hi):
    hi = max(lo, int(hi))
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["tree", "attend", "attend", "attend", "fork", "rules"])
    mix = rng.randint(100, 10 ** 9)
    if kind == "tree":
        return {"kind": kind, "requests": _log(rng, 1, 250), "nodes": _log(rng, 2, 64), "mix": mix}
    if kind == "attend":
        shape, typ, chain = rng.choice(["tiny", "1b", "8b", "8b"]), rng.choice(["f32", "f16", "bf16", "i8"]), rng.random() < 0.25
        H, kvh, hd = HEADS[shape]
        nodes, n = _log(rng, 2, 250 if chain else 64), _log(rng, 1, 64)
        room = 500_000_000 // (n * 2 * kvh * (hd * ESIZE[typ] + (4 if typ == "i8" else 0)))      # tokens within the largest case's cost
        work = 60_000_000_000 // (4 * H * hd * nodes * n)
        return {"kind": kind, "shape": shape, "type": typ, "page": rng.choice([8, 16, 20, 32, 64, 256]), "requests": n,
                "most": max(nodes, _log(rng, nodes, min(60000, room, work, 400_000 // n))), "nodes": nodes, "chain": chain, "mix": mix}
    if kind == "fork":
        groups, new = _log(rng, 1, 32), rng.randint(1, 8)
        return {"kind": kind, "shape": rng.choice(["tiny", "1b"]), "type": rng.choice(["f32", "f16", "bf16", "i8"]), "page": rng.choice([8, 16, 20, 64]),
                "layers": rng.randint(1, 8), "groups": groups, "old": rng.randint(1, 8), "new": new, "most": _log(rng, 10, 1000), "mix": mix}
    vocab, nodes = _log(rng, 1000, 151936), rng.choice([1, 1, 4, 13])
    return {"kind": kind, "requests": _log(rng, 1, max(1, min(192, 150 * 128256 // (vocab * nodes)))), "nodes": nodes, "vocab": vocab,
            "history": _log(rng, 1, 8000), "masks": rng.choice([0, 5, 60]), "mix": mix}


# ---------------------------------------------------------------------------
# What follows from a case alone
# ---------------------------------------------------------------------------
def _forest(r, n, nodes, chain=False):
    """Rows of n requests (most have all of their tree, some less) and the rows' parents (-1: none, or no row)."""
    rows = [nodes if r.random() < 0.7 else r.randint(1, nodes) for _ in range(n)]
    parents = np.full((n, nodes), -1, np.int32)
    for i, m in enumerate(rows):
        for j in range(1, m):
            parents[i, j] = j - 1 if chain else r.randint(max(0, (j - 1) // 2 - 1), (j - 1) // 2 + (j - 1) % 2)
    return np.array(rows, np.int32), parents


def _above(parents):
    """[request, row, other]: whether the other row is the row itself or above it."""
    n, N = parents.shape
    up = np.zeros((n, N, N), bool)
    for j in range(N):
        p = parents[:, j]
        up[:, j] = np.where((p >= 0)[:, None], up[np.arange(n), p], False)
        up[:, j, j] = True
    return up


def _attend_lengths(case):
    """Cached tokens of every request, its new rows among them: the longest has `most`, the others spread below it."""
    r = random.Random(case["mix"])
    rows, parents = _forest(r, case["requests"], case["nodes"], case["chain"])
    lens = [max(int(m), int(case["most"] * (1.0 if i == 0 else r.uniform(0.05, 1.0)))) for i, m in enumerate(rows)]
    return np.array(lens, np.int32), rows, parents


def _fork_lengths(case):
    """Of groups of requests: tokens of the old ones, and how many of them all share; which old request each new one continues
    (-1: none), and how much of it."""
    r = random.Random(case["mix"])
    lens, shared, source, keep = [], [], [], []
    for g in range(case["groups"]):
        common = r.randint(1, case["most"])
        first = len(lens)
        for _ in range(case["old"]):
            lens.append(min(case["most"], common + r.randint(0, max(1, case["most"] // 8))))
            shared.append(common)
        for _ in range(case["new"]):
            source.append(-1 if r.random() < 0.05 else first + r.randrange(case["old"]))
            keep.append(10 ** 6 if r.random() < 0.8 else r.randint(0, case["most"]))
    return tuple(np.array(x, np.int32) for x in (lens, shared, source, keep))


def _rules(case):
    """Per request: rows, tokens so far, tokens of its prompt, and settings; per row its mask (-1: none)."""
    r = random.Random(case["mix"])
    n = case["requests"]
    rows, parents = _forest(r, n, case["nodes"])
    tokens = np.array([case["history"]] + [r.randint(0, case["history"]) for _ in range(n - 1)], np.int32)
    prompt = np.array([r.randint(0, int(t)) for t in tokens], np.int32)
    pick = lambda *a: np.array([r.choice(a) for _ in range(n)], np.float32)  # noqa: E731
    behind = [r.random() < 0.6 for _ in range(n)]
    allowed = np.array([r.randrange(case["masks"]) if case["masks"] and behind[i] else -1 for i in range(n) for _ in range(rows[i])], np.int32)
    return rows, parents, tokens, prompt, pick(1.0, 1.1, 1.3, 0.9), pick(0.0, 0.5, 1.5), pick(0.0, 0.1, -0.2), allowed


def work(case):
    kind = case["kind"]
    if kind == "tree":
        rows, _ = _forest(random.Random(case["mix"]), case["requests"], case["nodes"])
        # row: parent read twice, token, choice and slot read; position, mask, path, source and destination written
        return {"bytes": int(rows.sum()) * 44 + case["requests"] * 28, "flops": 0}
    if kind == "attend":
        H, KVH, hd = HEADS[case["shape"]]
        lens, rows, parents = (x.astype(np.int64) for x in _attend_lengths(case))
        each = 2 * KVH * (hd * ESIZE[case["type"]] + (4 if case["type"] == "i8" else 0))
        seen = int(((lens - rows) * rows).sum())
        for m, up in zip(rows, _above(parents)):
            seen += int(up[:m].sum())
        pages = int((-(-lens // case["page"])).sum())
        row = 2 * H * hd * 4 + 4 * H + (0 if case["chain"] else 8)
        return {"bytes": int(lens.sum()) * each + int(rows.sum()) * row + 8 * len(lens) + 4 * pages, "flops": 4 * H * hd * seen}
    if kind == "fork":
        _, KVH, hd = HEADS[case["shape"]]
        lens, _, source, keep = _fork_lengths(case)
        page = case["page"]
        t = np.where(source >= 0, np.minimum(lens[source.clip(0)], keep), 0)
        each = 2 * KVH * (hd * ESIZE[case["type"]] + (4 if case["type"] == "i8" else 0)) * case["layers"]
        # all but the requests that keep the page, about one a source, copy the tokens of their last page
        copied = int((t % page).sum()) - sum(int((t[source == s] % page).max(initial=0)) for s in set(source.tolist()))
        return {"bytes": 2 * each * max(copied, 0) + 4 * int((-(-lens // page)).sum() + (-(-t // page)).sum()) + 24 * len(source) + 4 * len(lens), "flops": 0}
    rows, _, tokens, _, _, _, _, allowed = _rules(case)
    V = case["vocab"]
    masks = len(set(allowed[allowed >= 0].tolist()))
    return {"bytes": int(rows.sum()) * 8 * V + masks * 4 * -(-V // 32) + 4 * int(tokens.sum()) + 16 * int(rows.sum()) + 150 * len(rows), "flops": 2 * int(rows.sum()) * V}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _cuda(x, dtype=None):
    return torch.as_tensor(x, dtype=dtype, device="cuda")


def _i32(*shape):
    return torch.full(shape, -1, dtype=torch.int32, device="cuda")


def _cache(g, typ, shape):
    """Keys and values as a model caches them (N(0, 1), some channels larger), every slot of every page holding some."""
    gain = torch.ones(shape[-1], device="cuda")
    gain[::16] = 3.0
    made = []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device="cuda") * gain
        if typ == "i8":
            scale = x.abs().amax(-1) / 127.0
            made.append((torch.round(x / scale[..., None]).to(torch.int8), scale))
        else:
            made.append((x.to(TYPES[typ]), None))
        del x
    (k, ks), (v, vs) = made
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _starts(rows):
    return _cuda(np.concatenate([[0], np.cumsum(rows)]), torch.int32)


def _words(up, rows):
    """Ancestors as bits: a row of 64-bit words for every row of every request."""
    n, N, _ = up.shape
    W = -(-N // 64)
    bits = np.zeros((n, N, W * 64), np.uint64)
    bits[..., :N] = up
    words = (bits.reshape(n, N, W, 64) << np.arange(64, dtype=np.uint64)).sum(-1, dtype=np.uint64)
    return _cuda(words[np.arange(N)[None, :] < np.asarray(rows)[:, None]].view(np.int64))


def _prepare_tree(case, g):
    rows, parents = _forest(random.Random(case["mix"]), case["requests"], case["nodes"])
    n, N, R = len(rows), case["nodes"], int(rows.sum())
    at = _cuda(np.arange(N)[None, :] < rows[:, None])
    tokens = torch.randint(0, 32000, (n, N), generator=g, device="cuda", dtype=torch.int32)
    # a draft is right about two times in three: what follows a row is then one of its children's tokens
    par = _cuda(parents).long()
    lucky = torch.rand((n, N, N), generator=g, device="cuda").masked_fill(par[:, None, :] != torch.arange(N, device="cuda")[None, :, None], -1.0)
    best, child = lucky.max(-1)
    right = (best >= 0) & (torch.rand((n, N), generator=g, device="cuda") < 0.67)
    chosen = torch.where(right, tokens.gather(1, child), torch.randint(0, 32000, (n, N), generator=g, device="cuda", dtype=torch.int32))
    lens = torch.randint(100, 2500, (n,), generator=g, device="cuda", dtype=torch.int32) + _cuda(rows)
    return {"starts": _starts(rows), "lens": lens, "parents": _cuda(parents), "tokens": tokens[at], "chosen": chosen[at],
            "slots": torch.randperm(4 * R, generator=g, device="cuda")[:R].to(torch.int32), "rows": R,
            "out": {"positions": _i32(R), "mask": torch.zeros((R, -(-N // 64)), dtype=torch.int64, device="cuda"), "accepted": _i32(n), "last": _i32(n),
                    "lens": _i32(n), "path": _i32(R), "src": _i32(R), "dst": _i32(R)}}


def _prepare_attend(case, g):
    H, KVH, hd = HEADS[case["shape"]]
    lens, rows, parents = _attend_lengths(case)
    page = case["page"]
    have = -(-lens // page)
    total, width = int(have.sum()), int(have.max()) + 2           # a table has room for what is still to come
    s = _cache(g, case["type"], (total + 5, KVH, page, hd))
    perm = torch.randperm(total + 5, generator=g, device="cuda").to(torch.int32)
    col = np.arange(width)[None, :]
    at = _cuda(np.where(col < have[:, None], (np.cumsum(have) - have)[:, None] + col, -1))
    q = torch.randn((int(rows.sum()), H, hd), generator=g, device="cuda") * 1.5
    s.update(table=torch.where(at >= 0, perm[at.clamp(min=0)], -1), lens=_cuda(lens), starts=_starts(rows), q=q, nodes=case["nodes"],
             mask=None if case["chain"] else _words(_above(parents), rows), o=torch.empty_like(q),
             lse=torch.empty(q.shape[:2], device="cuda"), most=int(lens.max()), page=page)
    return s


def _prepare_fork(case, g):
    _, KVH, hd = HEADS[case["shape"]]
    lens, shared, source, keep = _fork_lengths(case)
    page, n, m = case["page"], len(lens), len(source)
    have, common = -(-lens // page), shared // page                # whole pages of the common beginning are shared
    width = int(have.max()) + 1
    table, extra, used = np.full((n, width), -1, np.int64), [], 0
    for i in range(n):
        first = i - i % case["old"]
        c = int(common[i]) if i != first else 0
        table[i, :c] = table[first, :c]
        table[i, c:have[i]] = used + np.arange(have[i] - c)
        if i == first:
            extra += [case["old"] - 1] * int(common[i]) + [0] * int(have[i] - common[i])
        else:
            extra += [0] * int(have[i] - c)
        used += int(have[i]) - c
    pages = used + m + 9
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    count = torch.zeros(pages, dtype=torch.int32, device="cuda")
    count[perm[:used].long()] = _cuda(extra, torch.int32)
    head = int(torch.randint(0, pages, (1,), generator=g, device="cuda"))
    ring = _i32(pages)
    ring[(head + torch.arange(pages - used, device="cuda")) % pages] = perm[used:]
    s = _cache(g, case["type"], (case["layers"], pages, KVH, page, hd))
    s.update(lens=_cuda(lens), table=torch.where(_cuda(table) >= 0, perm[_cuda(table).clamp(min=0)], -1), source=_cuda(source), keep=_cuda(keep),
             extra=count, ring=ring, state=_cuda([head, pages - used], torch.int32), page=page, type=case["type"],
             out={"table": _i32(m, width), "lens": _i32(m), "status": _i32(m), "extra": torch.empty_like(count), "state": _i32(2),
                  "src": _i32(m), "dst": _i32(m), "count": _i32(m)})
    return s


def _prepare_rules(case, g):
    rows, parents, n_tokens, n_prompt, rep, pres, freq, allowed = _rules(case)
    n, V, R = case["requests"], case["vocab"], int(rows.sum())
    x = torch.randn((R, V), generator=g, device="cuda") * 2.2                  # a language model's rows: a wide floor
    few = min(64, V // 4)
    x.scatter_(1, torch.randint(0, V, (R, few), generator=g, device="cuda"), 6.0 + 9.0 * torch.rand((R, few), generator=g, device="cuda"))
    # text repeats itself: token t about as often as 1 / t
    some = lambda *shape: torch.exp(torch.rand(shape, generator=g, device="cuda") * math.log(V)).to(torch.int32).clamp(max=V - 1)  # noqa: E731
    s = {"logits": x, "out": torch.empty_like(x), "requests": _cuda(np.repeat(np.arange(n), rows), torch.int32),
         "tokens": some(n, max(1, case["history"])), "n_tokens": _cuda(n_tokens), "n_prompt": _cuda(n_prompt),
         "repetition": _cuda(rep), "presence": _cuda(pres), "frequency": _cuda(freq),
         "bias_tokens": torch.rand((n, V), generator=g, device="cuda").topk(8)[1].to(torch.int32), "bias": torch.randn((n, 8), generator=g, device="cuda") * 4,
         "starts": None, "drafted": None, "mask": None, "allowed": None, "allowed_rows": None}
    if case["nodes"] > 1:
        s.update(starts=_starts(rows), drafted=some(R), mask=_words(_above(parents), rows))
    if case["masks"]:
        # a grammar's states: most let few tokens through, some nearly all
        share = torch.rand((case["masks"], 1), generator=g, device="cuda") ** 4
        words = -(-V // 32)
        bits = (torch.rand((case["masks"], words * 32), generator=g, device="cuda") < share).view(case["masks"], words, 32)
        packed = (bits.long() << torch.arange(32, device="cuda")).sum(-1)
        s.update(allowed=torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32), allowed_rows=_cuda(allowed))
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"tree": _prepare_tree, "attend": _prepare_attend, "fork": _prepare_fork, "rules": _prepare_rules}[case["kind"]](case, g)
    s["kind"] = case["kind"]
    return s


# ---------------------------------------------------------------------------
# The operators in their plain form
# ---------------------------------------------------------------------------
def _plain_tree(s):
    n, N = s["parents"].shape
    starts, rows, i32 = s["starts"].long(), s["rows"], torch.int32
    req = torch.searchsorted(starts[1:], torch.arange(rows, device="cuda"), right=True)
    node = torch.arange(rows, device="cuda") - starts[req]
    m = starts[1:] - starts[:-1]
    ctx = s["lens"].long() - m
    j = torch.arange(N, device="cuda")
    par = s["parents"].long()
    up = ((par[:, :, None] == j) & (j < j[:, None]) | (j == j[:, None])).float()
    for _ in range(max(1, (N - 1).bit_length())):         # twice the distance each time
        up = (torch.matmul(up, up) > 0).float()
    W = -(-N // 64)
    bits = torch.zeros((n, N, W * 64), dtype=torch.int64, device="cuda")
    bits[..., :N] = up.long()
    mask = (bits.view(n, N, W, 64) << torch.arange(64, device="cuda")).sum(-1)
    depth = up.sum(-1).long() - 1

    def spread(x):
        d = torch.full((n, N), -1, dtype=torch.int64, device="cuda")
        d[req, node] = x.long()
        return d

    tokens, chosen, slots = spread(s["tokens"]), spread(s["chosen"]), spread(s["slots"])
    fits = (par >= 0) & (tokens >= 0) & (tokens == chosen.gather(1, par.clamp(min=0)))
    among = fits[:, None, :] & (par[:, None, :] == par[:, :, None]) & (j[None, :] < j[:, None])      # an earlier sibling that fits too
    good = fits & ~among.any(-1)
    good[:, 0] = True
    there = j[None, :] < m[:, None]
    taken = ((up * ~good[:, None, :]).sum(-1) == 0) & (up[:, :, 0] > 0) & there
    count = taken.sum(1)
    k = taken.long().cumsum(1) - 1
    path = torch.full((n, N + 1), -1, dtype=torch.int64, device="cuda")
    path.scatter_(1, torch.where(taken, k, N), torch.where(taken, j.expand(n, N), -1))
    path = path[:, :N]
    moved = (path >= 0) & (path != j)
    src = torch.where(moved, slots.gather(1, path.clamp(min=0)), -1)
    dst = torch.where(moved, slots, -1)
    end = torch.where(count > 0, path.gather(1, (count - 1).clamp(min=0)[:, None])[:, 0], 0)
    last = torch.where(count > 0, chosen.gather(1, end[:, None])[:, 0], -1)
    path = torch.where(path >= 0, path + starts[:-1, None], -1)
    pick = lambda x: x[req, node].to(i32)  # noqa: E731
    return {"positions": pick(ctx[:, None] + depth), "mask": mask[req, node], "accepted": count.to(i32), "last": last.to(i32),
            "lens": (ctx + count).to(i32), "path": pick(path), "src": pick(src), "dst": pick(dst)}


def _plain_attend(s):
    q, table, lens, starts = s["q"], s["table"], s["lens"].long(), s["starts"].long()
    R, H, hd = q.shape
    n, N, KVH, page = lens.numel(), s["nodes"], s["k"].shape[1], s["page"]
    G, cols = H // KVH, -(-s["most"] // page)
    T = cols * page
    at = table[:, :cols].long().clamp(min=0)
    req = torch.searchsorted(starts[1:], torch.arange(R, device="cuda"), right=True)
    node = torch.arange(R, device="cuda") - starts[req]
    ctx = lens - (starts[1:] - starts[:-1])

    def rows(x, scale):
        x = x[at].float()
        if scale is not None:
            x = x * scale[at][..., None]
        return x.transpose(1, 2).reshape(n, KVH, T, hd)

    dense = torch.zeros((n, N, H, hd), device="cuda")
    dense[req, node] = q
    dense = dense.view(n, N, KVH, G, hd).permute(0, 2, 1, 3, 4).reshape(n, KVH, N * G, hd)
    k = rows(s["k"], s["k_scale"]).transpose(2, 3).contiguous()
    scores = torch.matmul(dense, k) * (1.0 / math.sqrt(hd))
    del k
    b = torch.arange(T, device="cuda")[None, :] - ctx[:, None]                # a token's place among the new ones
    if s["mask"] is None:
        seen = b[:, None, :] <= torch.arange(N, device="cuda")[None, :, None]
    else:
        words = torch.zeros((n, N, s["mask"].shape[1]), dtype=torch.int64, device="cuda")
        words[req, node] = s["mask"]
        inside = ((b >= 0) & (b < 64 * words.shape[2]))[:, None, :]
        c = b.clamp(0, 64 * words.shape[2] - 1)[:, None, :].expand(n, N, T)
        seen = (b < 0)[:, None, :] | (inside & ((words.gather(2, c >> 6) >> (c & 63)) & 1).bool())
    seen = seen & (torch.arange(T, device="cuda")[None, :] < lens[:, None])[:, None, :]
    scores = scores.view(n, KVH, N, G, T).masked_fill(~seen[:, None, :, None, :], float("-inf")).view(n, KVH, N * G, T)
    del seen
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top > float("-inf"), top, 0.0)                          # of a row that is none of the request's
    e = torch.exp(scores - top)
    del scores
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, rows(s["v"], s["v_scale"])) / total
    back = lambda x: x.view(n, KVH, N, G, -1).transpose(1, 2).reshape(n, N, H, -1)[req, node]  # noqa: E731
    return {"o": back(o), "lse": back(top + torch.log(total))[..., 0]}


def _plain_fork(s):
    page, ring, extra = s["page"], s["ring"], s["extra"]
    n, width = s["table"].shape
    m, R, P = s["source"].numel(), ring.numel(), extra.numel()
    lens, src, i32 = s["lens"].long(), s["source"].long(), torch.int32
    head, free = s["state"].long()
    col = torch.arange(width, device="cuda")
    tokens = torch.where(src >= 0, torch.minimum(lens[src.clamp(min=0)], s["keep"].long()), 0)
    have, want = (lens + page - 1) // page, (tokens + page - 1) // page
    old = torch.where(col < have[:, None], s["table"].long(), P)
    new = torch.where(col < want[:, None], s["table"].long()[src.clamp(min=0)], P)
    ones = lambda x: torch.ones_like(x).flatten()  # noqa: E731
    holders = torch.cat([extra.long() + 1, extra.new_zeros(1).long()])
    outside = holders.scatter_add(0, old.flatten(), -ones(old))
    # who may keep a page that it will write to: the one that has most of it, the first of these; all others copy it
    covered = (tokens[:, None] - col * page).clamp(max=page)
    rank = torch.where(new < P, covered * m + (m - 1 - torch.arange(m, device="cuda"))[:, None], -1)
    best = torch.full((P + 1,), -1, dtype=torch.int64, device="cuda").scatter_reduce(0, new.flatten(), rank.flatten(), "amax")
    copies = (new < P) & (covered < page) & ((rank != best[new]) | (outside[new] > 0))
    need = copies.any(1).long()
    refused = (need > 0) & (need.cumsum(0) > free)
    need = torch.where(refused, 0, need)
    taken = need.sum()
    got = ring[(head + need.cumsum(0) - need) % R].long()
    copies, new = copies & ~refused[:, None], torch.where(refused[:, None], P, new)
    after = outside.scatter_add(0, torch.where(copies, P, new).flatten(), ones(new))
    table = torch.where(copies, got[:, None], new)
    first = torch.full((P + 1,), n * width, dtype=torch.int64, device="cuda").scatter_reduce(
        0, old.flatten(), torch.arange(n * width, device="cuda"), "amin")
    gone = (old < P) & (after[old] <= 0) & (first[old] == torch.arange(n * width, device="cuda").view(n, width))
    order = gone.flatten().long().cumsum(0).view(n, width) - 1
    given = gone & (order < R - free)
    ring_out = torch.cat([ring, ring[:1]]).scatter(0, torch.where(given, (head + free + order) % R, R).flatten(), s["table"].flatten())[:R]
    touched = torch.zeros(P + 1, dtype=torch.bool, device="cuda").scatter(0, old.flatten(), True)
    extra_out = torch.where(touched[:P], (after[:P] - 1).clamp(min=0), extra.long())
    page_from = torch.where(copies, new, 0).sum(1)
    moved = need > 0
    k, v, ks, vs = s["k"], s["v"], s["k_scale"], s["v_scale"]
    inside = torch.arange(page, device="cuda") < (tokens % page)[:, None]
    at = (moved[:, None] & inside).nonzero()
    a, b, slot = page_from[at[:, 0]], got[at[:, 0]], at[:, 1]
    k[:, b, :, slot] = k[:, a, :, slot]
    v[:, b, :, slot] = v[:, a, :, slot]
    if ks is not None:
        ks[:, b, :, slot] = ks[:, a, :, slot]
        vs[:, b, :, slot] = vs[:, a, :, slot]
    o = {"table": torch.where(table < P, table, -1), "lens": torch.where(refused, 0, tokens), "status": torch.where(refused, 3, 0),
         "extra": extra_out, "state": torch.stack([(head + taken) % R, free - taken + torch.minimum(gone.sum(), R - free)]),
         "src": torch.where(moved, page_from * page, -1), "dst": torch.where(moved, got * page, -1), "count": torch.where(moved, tokens % page, 0)}
    return {**{x: y.to(i32) for x, y in o.items()}, "ring": ring_out, **_held(s)}


def _held(s):
    """The caches; 8-bit rows as the values they stand for."""
    if s["type"] == "i8":
        return {"k": s["k"] * s["k_scale"][..., None], "v": s["v"] * s["v_scale"][..., None]}
    return {"k": s["k"], "v": s["v"]}


def _plain_rules(s):
    x, req = s["logits"], s["requests"].long()
    R, V = x.shape
    place = torch.arange(s["tokens"].shape[1], device="cuda")
    tokens = s["tokens"].long()
    live, told = place < s["n_tokens"][:, None], place < s["n_prompt"][:, None]
    n = s["n_tokens"].numel()
    seen = torch.zeros((n, V), device="cuda").scatter_add_(1, tokens, live.float())
    made = torch.zeros((n, V), device="cuda").scatter_add_(1, tokens, (live & ~told).float())
    seen, made = seen[req], made[req]
    if s["mask"] is not None:
        N = 64 * s["mask"].shape[1]
        b = torch.arange(N, device="cuda")
        bit = ((s["mask"][:, b >> 6] >> (b & 63)) & 1).float()
        at = (s["starts"].long()[req][:, None] + b).clamp(max=R - 1)
        token = s["drafted"].long()[at]
        seen.scatter_add_(1, token, bit)
        made.scatter_add_(1, token, bit)
    col = lambda y: y[req][:, None]  # noqa: E731
    rep = torch.where(seen > 0, col(s["repetition"]), 1.0)
    y = torch.where(x > 0, x / rep, x * rep)
    y = y - (col(s["frequency"]) * made + col(s["presence"]) * (made > 0))
    bias = torch.zeros((n, V), device="cuda").scatter_(1, s["bias_tokens"].long(), s["bias"])
    y = y + bias[req]
    if s["allowed"] is not None:
        t = torch.arange(V, device="cuda")
        bits = ((s["allowed"][:, t >> 5] >> (t & 31)) & 1).bool()
        a = s["allowed_rows"].long()
        y = y.masked_fill(~(bits[a.clamp(min=0)] | (a < 0)[:, None]), float("-inf"))
    return {"out": y}


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
_q = None


def _lib():
    global _q
    if _q is None:
        spec = importlib.util.spec_from_file_location("qllama", os.path.join(ROOT, "llm-project_amd", "qllama.py"))
        _q = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_q)
    return _q


def _own(s):
    Q, kind = _lib(), s["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "tree":
        o = s["out"]
        Q.tree_plan(s["starts"], s["lens"], s["parents"], o["positions"], o["mask"], stream=stream)
        Q.tree_accept(s["starts"], s["lens"], s["parents"], s["tokens"], s["chosen"], s["slots"], o["accepted"], o["last"], o["lens"],
                      o["path"], o["src"], o["dst"], stream=stream)
        return o
    if kind == "attend":
        if "cache" not in s:
            s["cache"] = Q.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
            s["work"] = torch.empty(Q.tree_attention_work(s["cache"], s["q"].shape[0], s["lens"].numel(), s["q"].shape[1], s["nodes"]),
                                    dtype=torch.uint8, device="cuda")
        Q.tree_attention(s["cache"], s["q"], s["starts"], s["table"], s["lens"], s["o"], s["work"], mask=s["mask"], lse=s["lse"],
                         nodes=s["nodes"], stream=stream)
        return {"o": s["o"], "lse": s["lse"]}
    if kind == "fork":
        o = s["out"]
        if "caches" not in s:
            sc = s["type"] == "i8"
            s["caches"] = Q.PagedCaches([Q.PagedKV(s["k"][i], s["v"][i], s["k_scale"][i] if sc else None, s["v_scale"][i] if sc else None)
                                         for i in range(s["k"].shape[0])])
            s["work"] = torch.empty(Q.paged_fork_work(s["lens"].numel(), s["source"].numel(), s["extra"].numel()), dtype=torch.uint8, device="cuda")
        Q.paged_fork(s["lens"], s["table"], s["source"], s["extra"], s["ring"], s["state"], s["page"], o["table"], o["lens"], o["status"],
                     o["extra"], o["state"], o["src"], o["dst"], o["count"], s["work"], keep=s["keep"], stream=stream)
        Q.paged_move(s["caches"], o["src"], o["dst"], count=o["count"], stream=stream)
        return {**o, "ring": s["ring"], **_held(s)}
    Q.logit_rules(s["logits"], s["out"], requests=s["requests"], tokens=s["tokens"], n_tokens=s["n_tokens"], n_prompt=s["n_prompt"],
                  repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"], starts=s["starts"], drafted=s["drafted"],
                  mask=s["mask"], bias_tokens=s["bias_tokens"], bias=s["bias"], allowed=s["allowed"], allowed_rows=s["allowed_rows"],
                  stream=stream)
    return {"out": s["out"]}


def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "attend": _plain_attend, "fork": _plain_fork, "rules": _plain_rules}[state["kind"]](state)


# ---------------------------------------------------------------------------
# The same from the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_attend(s, case):
    R, H, hd = s["q"].shape
    KVH, page = s["k"].shape[1], s["page"]
    G = H // KVH
    lens, rows, parents = _attend_lengths(case)
    o, lse = torch.zeros((R, H, hd), dtype=torch.float64, device="cuda"), torch.zeros((R, H), dtype=torch.float64, device="cuda")
    up, first = _above(parents), 0
    for r, (length, m) in enumerate(zip(lens.tolist(), rows.tolist())):
        pages = s["table"][r, :-(-length // page)].long()
        hidden = torch.zeros((m, length), dtype=torch.bool, device="cuda")
        hidden[:, length - m:] = _cuda(~up[r, :m, :m])
        for h in range(KVH):
            k, v = s["k"][pages, h].double(), s["v"][pages, h].double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][pages, h].double()[..., None], v * s["v_scale"][pages, h].double()[..., None]
            k, v = k.reshape(-1, hd)[:length], v.reshape(-1, hd)[:length]
            q = s["q"][first:first + m, h * G:(h + 1) * G].double().reshape(m * G, hd)
            w = (q @ k.t().contiguous()) / hd ** 0.5
            w = w.view(m, G, length).masked_fill(hidden[:, None, :], float("-inf")).view(m * G, length)
            z = torch.logsumexp(w, 1, keepdim=True)
            o[first:first + m, h * G:(h + 1) * G] = (torch.exp(w - z) @ v).view(m, G, hd)
            lse[first:first + m, h * G:(h + 1) * G] = z.view(m, G)
        first += m
    return {"o": o, "lse": lse}


def _exact_rules(s, case):
    rows, parents, n_tokens, n_prompt, rep, pres, freq, allowed = _rules(case)
    V = case["vocab"]
    logits, tokens = s["logits"].double().cpu().numpy(), s["tokens"].cpu().numpy()
    bias_at, bias = s["bias_tokens"].cpu().numpy(), s["bias"].double().cpu().numpy()
    rep, pres, freq = rep.astype(np.float64), pres.astype(np.float64), freq.astype(np.float64)
    drafted = None if s["drafted"] is None else s["drafted"].cpu().numpy()
    words = None if s["allowed"] is None else s["allowed"].cpu().numpy().view(np.uint32)
    up, out, i = _above(parents), np.empty_like(logits), 0
    for r in range(case["requests"]):
        first = i
        for j in range(rows[r]):
            more = drafted[first:first + rows[r]][up[r, j, :rows[r]]] if drafted is not None else tokens[:0, 0]
            history = tokens[r, :n_tokens[r]]
            times = np.bincount(np.concatenate([history[n_prompt[r]:], more]), minlength=V)
            x = logits[i].copy()
            known = np.unique(np.concatenate([history, more]))
            x[known] = np.where(x[known] > 0, x[known] / rep[r], x[known] * rep[r])
            x -= freq[r] * times + pres[r] * (times > 0)
            x[bias_at[r]] += bias[r]
            if words is not None and allowed[i] >= 0:
                x[np.unpackbits(words[allowed[i]].view(np.uint8), bitorder="little")[:V] == 0] = -np.inf
            out[i] = x
            i += 1
    return {"out": out}


def exact(case, seed):
    if case["kind"] in ("tree", "fork"):
        return None                       # whole numbers and copies only
    s = prepare(case, seed)
    return _exact_attend(s, case) if case["kind"] == "attend" else _exact_rules(s, case)
