"""Drafted trees over a paged cache (include/qserve.h) on the GPU against plain definitions in whole numbers and 64 bits:
positions and ancestors, attention of several new tokens a request, and what the chosen tokens confirm."""
import math
import random

import pytest
from test_gpu_qserve import EPS, Buffer, Dev, Graph, Q, Work, dev_i32, i32, make_cache, pages_for, same, widened  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def i64(*shape):
    return Dev(torch.zeros(shape, dtype=torch.int64))


def forest(r, m, kind="tree"):
    """Parents of m rows; kind "tree": anything before them, "chain": the row before, "wild": also what is no row."""
    if kind == "chain":
        return [j - 1 for j in range(m)]
    if kind == "wild":
        return [r.choice([-7, -1, j, j + 1, 2 ** 31 - 1, -2 ** 31, r.randrange(max(1, j))]) for j in range(m)]
    return [-1 if j == 0 or r.random() < 0.1 else r.randrange(max(0, j - 9), j) for j in range(m)]


def above(parents):
    """Rows that every row may attend to among its request's new ones."""
    up = []
    for j, p in enumerate(parents):
        up.append({j} | (up[p] if 0 <= p < j else set()))
    return up


def signed(x):
    return x - 2 ** 64 if x >= 2 ** 63 else x


# ---------------------------------------------------------------------------
# Positions and masks
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("sizes,nodes,words,kind", [
    ([1], 1, 1, "tree"), ([0, 3, 0, 1], 4, 1, "tree"), ([64, 63, 1, 0, 17], 64, 1, "tree"), ([65, 64, 2], 70, 2, "tree"),
    ([256, 200, 129], 256, 4, "tree"), ([256, 31], 256, 4, "chain"), ([70, 3], 70, 1, "tree"), ([40, 5], 10, 1, "tree"), ([300, 1], 1024, 4, "chain"),
    ([30, 0, 64], 64, 1, "wild"), ([8] * 700, 8, 1, "tree")])
def test_tree_plan(Q, sizes, nodes, words, kind):  # noqa: F811
    r = random.Random(len(sizes) + nodes)
    n, rows, spare = len(sizes), sum(sizes), 3
    table = torch.full((n, nodes + 2), 99, dtype=torch.int32)          # a stride, and parents of rows that are not there
    want_p, want_m = [], []
    starts, lens = [0], []
    for i, m in enumerate(sizes):
        par = forest(r, min(m, nodes), kind)
        table[i, :len(par)] = torch.tensor(par, dtype=torch.int32)
        starts.append(starts[-1] + m)
        lens.append(m + r.randrange(0, 5000))
        up = above((par + [-1] * m)[:m])
        for j in range(m):
            inside = j < 64 * words
            want_p.append(lens[i] - m + (len(up[j]) - 1 if inside else j))
            bits = sum(1 << b for b in up[j]) if inside else 0
            want_m.append([signed(bits >> 64 * w & (2 ** 64 - 1)) for w in range(words)])
    pos, mask = Dev(torch.full((rows + spare,), 55, dtype=torch.int32)), Dev(torch.full((rows + spare, words), 77, dtype=torch.int64))
    parents = Dev(table)[:, :nodes]
    for _ in range(2):
        Q.tree_plan(dev_i32(starts), dev_i32(lens), parents, pos, mask)
        assert pos.get().tolist() == want_p + [55] * spare
        assert mask.get().tolist() == want_m + [[77] * words] * spare


def test_tree_plan_starts_out_of_range(Q):  # noqa: F811
    """Rows are cut to the outputs; a falling start is a request without rows."""
    pos, mask = Dev(torch.full((5,), -9, dtype=torch.int32)), Dev(torch.full((5, 1), -9, dtype=torch.int64))
    Q.tree_plan(dev_i32([-4, 2, 1, 2 ** 31 - 1]), dev_i32([10, 20, 30]), Dev(torch.tensor([[-1, 0, 1, 2]] * 3, dtype=torch.int32)), pos, mask)
    # request 0: rows 0, 1; request 1: none; request 2: rows 1 .. 4 (row 1 by either)
    assert pos.get().tolist()[0] == 8 and pos.get().tolist()[1] in (9, 26) and pos.get().tolist()[2:] == [27, 28, 29]
    assert mask.get().flatten().tolist()[2:] == [3, 7, 15]


# ---------------------------------------------------------------------------
# Acceptance
# ---------------------------------------------------------------------------
def accept_ref(m, parents, tokens, chosen, nodes):
    if m == 0:
        return []
    path, at = [0], 0
    while True:
        c = [j for j in range(at + 1, min(m, nodes)) if parents[j] == at and tokens[j] == chosen[at] and chosen[at] >= 0]
        if not c or at >= nodes:
            return path
        at = c[0]
        path.append(at)


@pytest.mark.parametrize("sizes,nodes,kind", [([1], 1, "tree"), ([0, 5, 1, 64, 0, 65, 200], 200, "tree"), ([700, 3], 1024, "chain"), ([1024], 1024, "chain"),
                                              ([1030, 9], 8, "tree"), ([12] * 900, 12, "tree"), ([40, 30], 64, "wild")])
def test_tree_accept(Q, sizes, nodes, kind):  # noqa: F811
    r = random.Random(nodes + len(sizes))
    n, rows = len(sizes), sum(sizes)
    table = torch.full((n, nodes + 1), 3, dtype=torch.int32)
    starts, lens, tokens, chosen = [0], [], [], []
    slots = [r.randrange(2 ** 31 - 1) for _ in range(rows)]
    acc, last, lens_out, path, src, dst = [], [], [], [], [], []
    for i, m in enumerate(sizes):
        par = forest(r, min(m, nodes), kind)
        table[i, :len(par)] = torch.tensor(par, dtype=torch.int32)
        t = [r.randrange(-1, 4) for _ in range(m)]                    # siblings that are alike, and tokens below 0
        c = [r.randrange(-1, 4) if kind != "chain" or r.random() < 0.02 else t[min(j + 1, m - 1)] for j in range(m)]
        got = accept_ref(m, par, t, c, nodes)
        s0 = starts[-1]
        lens.append(m + r.randrange(3000))
        acc.append(len(got))
        last.append(c[got[-1]] if got else -1)
        lens_out.append(lens[i] - m + len(got))
        for k in range(m):
            row = got[k] if k < len(got) else -1
            path.append(s0 + row if row >= 0 else -1)
            src.append(slots[s0 + row] if row >= 0 and row != k else -1)
            dst.append(slots[s0 + k] if row >= 0 and row != k else -1)
        tokens += t
        chosen += c
        starts.append(s0 + m)
    out = [i32(n), i32(n), i32(n)] + [Dev(torch.full((rows + 2,), -5, dtype=torch.int32)) for _ in range(3)]
    pad = [0, 0]
    Q.tree_accept(dev_i32(starts), dev_i32(lens), Dev(table)[:, :nodes], dev_i32(tokens + pad), dev_i32(chosen + pad), dev_i32(slots + pad), *out)
    for x, want in zip(out[:3], (acc, last, lens_out)):
        assert x.get().tolist() == want
    for x, want in zip(out[3:], (path, src, dst)):
        assert x.get().tolist() == want + [-5, -5]


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def attend_ref(kv, q, starts, table, lens, seen):
    """o, lse, and a bound of what 32-bit arithmetic may differ from them, all in 64 bits: the terms of the one-token
    attention's bound (test_gpu_qserve.py).  A sum over len tokens is taken in groups of 16 or 32, whose order differs and
    whose additions its 3 len counts; parts of a tile that meet add 6 EPS of a weight each, and there are fewer than len / 16
    of them and three rounds more: within 3 len + 16 from 32 tokens on, and 18 more below."""
    R, H, hd = q.shape
    KVH, page = kv.k.shape[1], kv.k.shape[2]
    G, scale = H // KVH, 1.0 / math.sqrt(hd)
    o, lse, bound, lse_bound = (torch.zeros(s, dtype=torch.float64) for s in ((R, H, hd), (R, H), (R, H, hd), (R, H)))
    lse.fill_(-math.inf)
    k_all, v_all = kv.k.get().double(), kv.v.get().double()
    if kv.k_scale is not None:
        k_all, v_all = k_all * kv.k_scale.get().double()[..., None], v_all * kv.v_scale.get().double()[..., None]
    q = q.double()
    for r in range(len(lens)):
        m, length = starts[r + 1] - starts[r], min(max(lens[r], 0), table.shape[1] * page)
        ctx = max(length - m, 0)
        for j in range(m):
            i = starts[r] + j
            t = torch.tensor(sorted(set(range(ctx)) | {ctx + b for b in seen[i] if b < m and ctx + b < length}), dtype=torch.long)
            p = table[r, t // page].long()
            t = t[(p >= 0) & (p < k_all.shape[0])]
            p = table[r, t // page].long()
            if not len(t):
                continue
            for h in range(KVH):
                k, v, hs = k_all[p, h, t % page], v_all[p, h, t % page], slice(h * G, h * G + G)
                s = (q[i, hs] @ k.t()) * scale
                z = torch.logsumexp(s, 1, keepdim=True)
                w = torch.exp(s - z)
                ds = ((3 * hd + 4) * EPS * (q[i, hs].abs() @ k.abs().t()) * scale + 2 * EPS * s.abs()).amax(1, keepdim=True)
                dw = 2 * ds + 4 * EPS * s.abs().amax(1, keepdim=True) + 8 * EPS
                o[i, hs], lse[i, hs] = w @ v, z[:, 0]
                bound[i, hs] = (2 * dw + (3 * len(t) + 34) * EPS) * (w @ v.abs())
                lse_bound[i, hs] = (dw + (len(t) + 34) * EPS + 4 * EPS * z.abs())[:, 0]
    return o, lse, bound, lse_bound


def attend(Q, kv, q, starts, table, lens, mask, nodes=0, spare=2, **kw):  # noqa: F811
    """o and lse; behind the requests' rows lie rows that stay as they were."""
    R, H, hd = q.shape
    full = torch.cat([q, torch.zeros(spare, H, hd)])
    o, lse = Dev(torch.full((R + spare, H, hd), 7.0)), Dev(torch.full((R + spare, H), 7.0))
    if mask is not None:
        mask = Dev(torch.cat([mask, torch.full((spare, mask.shape[1]), -1, dtype=torch.int64)]))
    work = Buffer(Q.tree_attention_work(kv, R + spare, len(lens), H, nodes))
    Q.tree_attention(kv, Dev(full), dev_i32(starts), Dev(table), dev_i32(lens), o, Work(work), mask=mask, lse=lse, nodes=nodes, **kw)
    o, lse = o.get(), lse.get()
    assert bool((o[R:] == 7.0).all()) and bool((lse[R:] == 7.0).all())
    return o[:R], lse[:R]


def case(typ, H, KVH, hd, page, order, lens, sizes, words, seed, Q, kind="bits"):  # noqa: F811
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    need = sum(-(-max(x, 0) // page) for x in lens)
    kv = make_cache(Q, typ, need + 3, KVH, page, hd, order, g)
    starts = [0]
    for m in sizes:
        starts.append(starts[-1] + m)
    q = torch.randn((starts[-1], H, hd), generator=g) * 1.5
    table = pages_for(lens, page, max(1, -(-max(lens) // page)) + 1, need + 3, seed)
    if words == 0:
        return kv, q, starts, table, lens, [set(range(j + 1)) for m in sizes for j in range(m)], None
    seen, mask = [], torch.zeros((starts[-1], words), dtype=torch.int64)
    for m in sizes:
        up = above(forest(r, m))
        for j in range(m):
            s = up[j] if kind == "tree" else {b for b in range(64 * words) if r.random() < 0.4} if r.random() < 0.8 else set()
            s = {b for b in s if b < 64 * words}
            for w in range(words):
                mask[len(seen), w] = signed(sum(1 << (b - 64 * w) for b in s if 64 * w <= b < 64 * w + 64))
            seen.append(s)
    return kv, q, starts, table, lens, seen, mask


def check(Q, kv, q, starts, table, lens, seen, mask, hints=(0,), tables=None):  # noqa: F811
    wo, wl, bound, lb = attend_ref(kv, q, starts, table, lens, seen)
    empty = torch.isinf(wl)
    for t in tables or (table, widened(table, kv.k.shape[2])):
        for nodes in hints:
            o, lse = attend(Q, kv, q, starts, t, lens, mask, nodes)
            o, lse = o.double(), lse.double()
            assert bool(((o - wo).abs() <= bound).all()), ((o - wo).abs() - bound).max()
            assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all()) and bool((o[empty] == 0).all())
            assert bool(((lse - wl).abs()[~empty] <= lb[~empty]).all())


SHAPES = [(6, 2, 48), (8, 2, 64), (4, 1, 128), (3, 3, 128), (5, 1, 8), (20, 1, 72), (2, 1, 256), (4, 2, 160)]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("H,KVH,hd", SHAPES)
@pytest.mark.parametrize("page,order,words", [(16, "head", 1), (5, "slot", 0), (48, "slot", 2), (1, "head", 1)])
def test_tree_attention_matches_the_definition(Q, typ, H, KVH, hd, page, order, words):  # noqa: F811
    """Requests without rows, without tokens, with nothing but new rows, with more rows than tokens, and masks of any bits, rows
    that see nothing among them; lengths around the steps; every hint."""
    lens = [0, 1, 2, 9, 16, 33, 64, 65, 130, 257, 3, -4, 40]
    sizes = [0, 1, 2, 9, 1, 0, 7, 13, 3, 5, 6, 2, 40]
    c = case(typ, H, KVH, hd, page, order, lens, sizes, words, H + hd + page, Q)
    check(Q, *c, hints=(0, 1, 5, 11, 30, 40) if (H, KVH, hd) in SHAPES[:4] else (0, 9))


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("lens,sizes,page,words", [([5000], [5], 16, 1), ([4097, 3], [17, 2], 64, 1), ([1, 6001, 40], [1, 70, 33], 24, 2), ([300] * 70, [4] * 70, 16, 1),
                                                   ([900, 0, 31, 1700] * 9, [3, 1, 20, 11] * 9, 128, 1), ([1500, 700], [256, 200], 16, 4),
                                                   ([1500, 700], [256, 200], 16, 0), ([2200], [600], 32, 0)])
def test_tree_attention_split_and_joined(Q, typ, lens, sizes, page, words):  # noqa: F811
    """Long and many requests, many rows: shares that end inside a tile, begin in another's, and hold several."""
    c = case(typ, 6, 2, 64, page, "head", lens, sizes, words, len(lens) + page, Q, "tree")
    check(Q, *c, hints=(0, 3, 60), tables=(widened(c[3], page),))


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("page,words,most", [(16, 1, 400), (7, 0, 400), (16, 2, 2500)])
def test_what_is_masked_has_no_effect(Q, typ, page, words, most):  # noqa: F811
    """New rows' keys, values and scales that are not finite reach the rows that see them, and leave the others' bits alone; slots
    behind the tokens and pages outside the cache count for nothing."""
    lens, sizes = [most, 70, 66, 30], [40, 70, 3, 30]
    kv, q, starts, table, lens, seen, mask = case(typ, 4, 2, 64, page, "head", lens, sizes, words, page, Q)
    table[0, 1] = -1
    table[1, -(-70 // page):] = 2 ** 31 - 1
    for t in (table, widened(table, page)):
        o, lse = attend(Q, kv, q, starts, t, lens, mask)
        for bad in (float("nan"), float("inf")):
            odd = {0: [0, 11, 39], 1: [5, 64, 69], 3: [29]}
            keep = [x.get() for x in ((kv.k_scale, kv.v_scale) if typ == "i8" else (kv.k, kv.v))]
            now = [x.clone() for x in keep]
            for r, rows in odd.items():
                for b in rows:
                    at = lens[r] - sizes[r] + b
                    p, s = int(table[r, at // page]), at % page
                    for x in now:
                        if typ == "i8":
                            x[p, :, s] = bad
                        else:
                            x[p, :, s, 3::7] = bad
            for x, y in zip((kv.k_scale, kv.v_scale) if typ == "i8" else (kv.k, kv.v), now):
                x.set(y)
            o2, lse2 = attend(Q, kv, q, starts, t, lens, mask)
            for x, y in zip((kv.k_scale, kv.v_scale) if typ == "i8" else (kv.k, kv.v), keep):
                x.set(y)
            for r in range(4):
                for j in range(sizes[r]):
                    i = starts[r] + j
                    if any(b in seen[i] for b in odd.get(r, [])):
                        assert not bool(torch.isfinite(o2[i]).all(-1).any()), (r, j)
                    else:
                        assert torch.equal(o2[i], o[i]) and torch.equal(lse2[i], lse[i]), (r, j)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("most", [100, 3000])
def test_values_that_are_not_finite(Q, typ, most):  # noqa: F811
    """Of an earlier token, in the step that the new rows lie in and in another: every row that attends to it gets no finite
    output at that dim, and keeps the others."""
    kv, q, starts, table, lens, seen, mask = case(typ, 4, 2, 64, 16, "head", [most], [9], 1, 3, Q, "tree")
    clean, _ = attend(Q, kv, q, starts, widened(table, 16), lens, mask)
    for at in (most - 10, 20):
        keep = kv.v.get()
        x = keep.clone()
        x[int(table[0, at // 16]), 1, at % 16, 5] = float("nan")
        kv.v.set(x)
        o, lse = attend(Q, kv, q, starts, widened(table, 16), lens, mask)
        kv.v.set(keep)
        assert bool(o[:, 2:, 5].isnan().all()) and bool(torch.isfinite(lse).all())
        o[:, 2:, 5] = clean[:, 2:, 5]
        assert torch.equal(o, clean)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
def test_one_row_is_the_one_token_attention(Q, typ):  # noqa: F811
    """Requests of a row each: as paged_attention, within both bounds."""
    lens = [1, 40, 700, 0, 33]
    kv, q, starts, table, lens, seen, mask = case(typ, 6, 2, 48, 16, "head", lens, [1] * 5, 1, 2, Q, "tree")
    check(Q, kv, q, starts, table, lens, seen, mask)


def test_strided_rows_scale_and_no_lse(Q):  # noqa: F811
    kv, q, starts, table, lens, seen, _ = case("bf16", 4, 2, 64, 16, "slot", [90, 20], [8, 3], 0, 5, Q)
    R = len(q)
    wide = torch.zeros(R, 3, 4, 64)
    wide[:, 1] = q * 2.0
    dq, do = Dev(wide), Dev(torch.full((R, 2, 4, 64), 7.0))
    work = Work(Buffer(Q.tree_attention_work(kv, R, 2, 4, 8)))
    Q.tree_attention(kv, dq[:, 1], dev_i32(starts), Dev(table), dev_i32(lens), do[:, 0], work, nodes=8, scale=0.0625)      # 1 / sqrt(64) / 2
    want, _ = attend(Q, kv, q, starts, table, lens, None, spare=0, nodes=8)
    got = do.get()
    assert torch.equal(got[:, 0], want) and bool((got[:, 1] == 7.0).all())


def test_starts_out_of_range(Q):  # noqa: F811
    """Starts outside the rows, and falling ones, read and write nothing outside: rows 0 .. 3 are request 0's, the rest no one's."""
    kv, q, starts, table, lens, seen, _ = case("f16", 4, 2, 64, 16, "head", [50, 30, 20], [4, 4, 4], 0, 6, Q)
    for far in (False, True):
        t = widened(table, 16) if far else table
        want, _ = attend(Q, kv, q[:4], [0, 4], t[:1], lens[:1], None, nodes=4)
        o, _ = attend(Q, kv, q, [-5, 4, 1, -2 ** 31], t, lens, None, nodes=4)
        assert torch.equal(o[:4], want) and bool((o[4:] == 7.0).all())


def test_equal_inputs_give_equal_bits(Q):  # noqa: F811
    c = case("bf16", 8, 2, 128, 16, "head", [3000, 500, 1200], [30, 3, 16], 1, 8, Q, "tree")
    kv, q, starts, table, lens, seen, mask = c
    first = attend(Q, kv, q, starts, widened(table, 16), lens, mask)
    for _ in range(3):
        again = attend(Q, kv, q, starts, widened(table, 16), lens, mask)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("typ,H,KVH,hd,nodes", [("bf16", 16, 1, 256, 8), ("f32", 16, 2, 128, 12), ("i8", 4, 4, 128, 9)])
def test_in_a_graph(Q, typ, H, KVH, hd, nodes):  # noqa: F811
    """The largest tiles in LDS (set as the launch's own size), and both launches of a split call, under capture."""
    kv, q, starts, table, lens, seen, mask = case(typ, H, KVH, hd, 16, "head", [2000, 77, 300], [nodes, 2, nodes], 1, 4, Q, "tree")
    for t in (table, table[1:2, :5].contiguous()):
        n, s = len(t), starts if len(t) == 3 else [0, 2]
        x, m, L = (q, mask, lens) if n == 3 else (q[nodes:nodes + 2].contiguous(), mask[nodes:nodes + 2].contiguous(), lens[1:2])
        want = attend(Q, kv, x, s, t, L, m, nodes, spare=0)
        dq, dm, dt, dn, ds, o, lse = Dev(x), Dev(m), Dev(t), dev_i32(L), dev_i32(s), Dev(torch.zeros_like(x)), Dev(torch.zeros(x.shape[:2]))
        work = Work(Buffer(Q.tree_attention_work(kv, len(x), n, H, nodes)))
        graph = Graph(lambda stream: Q.tree_attention(kv, dq, ds, dt, dn, o, work, mask=dm, lse=lse, nodes=nodes, stream=stream))
        for _ in range(3):
            o.set(torch.zeros_like(x))
            graph.replay()
            assert same(o, want[0]) and same(lse, want[1])


# ---------------------------------------------------------------------------
# f32 rows in 16-bit parts (heads of up to 128, from 33 columns on)
# ---------------------------------------------------------------------------
LN2 = float(torch.tensor(0.69314718056))             # what a sum of exponents of 2 is multiplied by, as a 32-bit number
UNIT = 0.6931471824645996                             # scale: times log2 e, in 32 bits, it is 1


def alone(Q, k, q, hd, nodes):  # noqa: F811
    """Scores of single products: row i of a request attends to itself alone, and key and queries of a row have one dim that is
    not 0 (its own).  k (requests, rows), q (requests, rows, heads); what comes back is each lse."""
    n, m, H = q.shape
    page = 16
    per = -(-m // page)
    kv = Q.PagedKV(*(Dev(torch.zeros((n * per, 1, page, hd))) for _ in range(2)))
    keys, rows, queries = torch.zeros((n, per * page, hd)), torch.arange(m), torch.zeros((n, m, H, hd))
    keys[:, rows, rows % hd] = k
    queries[:, rows, :, rows % hd] = q.transpose(0, 1)
    kv.k.set(keys.view(n * per, 1, page, hd))
    table = torch.arange(n * per, dtype=torch.int32).view(n, per)
    mask = torch.tensor([signed(1 << j) for j in range(m)], dtype=torch.int64)[:, None].repeat(n, 1)
    _, lse = attend(Q, kv, queries.view(n * m, H, hd), [m * i for i in range(n + 1)], table, [m] * n, mask, nodes=nodes, scale=UNIT)
    return lse.view(n, m, H).double()


@pytest.mark.parametrize("hd,nodes", [(64, 64), (64, 5), (128, 64), (64, 1), (128, 1)])
def test_f32_products_are_as_close_as_32_bits(Q, hd, nodes):  # noqa: F811
    """Keys and queries whose low halves are worst for parts that are cut (0xff7f and 0xffff: cut queries lose 5.6 x 2^-24 of
    every product, toward 0).  Parts to nearest leave out 2^-24 of a product at most.  The roundings beside them (five sums, the
    product with ln 2: 2^-24 each) go either way: over 4096 products of random signs and exponents their mean stays below
    4 x 6 x 2^-24 / 64 < 2^-25.  Of a single one: 2^-24 and six roundings.  The same in tiles that take f32 products."""
    g = torch.Generator().manual_seed(hd + nodes)

    def numbers(shape, low):
        bits = (torch.randint(0, 2, shape, generator=g) << 31) | (torch.randint(120, 134, shape, generator=g) << 23) | (torch.randint(0, 8, shape, generator=g) << 16) | low
        return bits.to(torch.int64).where(bits < 2 ** 31, bits - 2 ** 32).to(torch.int32).view(torch.float32)

    k, q = numbers((8, 64), 0xff7f), numbers((8, 64, 8), 0xffff)
    want = k.double()[..., None] * q.double() * LN2
    off = alone(Q, k, q, hd, nodes) / want - 1
    assert float(off.abs().max()) <= 7 * EPS, off.abs().max() / EPS
    assert abs(float(off.mean())) <= 2 * EPS, off.mean() / EPS


@pytest.mark.parametrize("hd,nodes", [(64, 1), (64, 4), (72, 4), (128, 1), (128, 4), (160, 8), (256, 64)])
def test_f32_products_of_few_columns_are_rounded_once(Q, hd, nodes):  # noqa: F811
    """Up to 32 columns (8 a row here), and with heads of more than 128, f32 rows are not taken apart: a product has one rounding,
    its product with ln 2 another."""
    g = torch.Generator().manual_seed(hd + nodes)
    k, q = torch.randn((8, 64), generator=g), torch.randn((8, 64, 8), generator=g)
    off = alone(Q, k, q, hd, nodes) / (k.double()[..., None] * q.double() * LN2) - 1
    assert float(off.abs().max()) <= 2 * EPS * (1 + EPS), off.abs().max() / EPS

@pytest.mark.parametrize("hd,nodes", [(64, 5), (64, 64), (72, 8), (128, 5), (128, 64)])
def test_f32_products_of_parts_add_up_from_the_smallest(Q, hd, nodes):  # noqa: F811
    """A product of parts leaves out 1.001 x 2^-24; its small products sum up to 2^-6.9 of it, so that five roundings of them
    take 0.05 x 2^-24; the largest product, added last, takes one of 2^-24, and ln 2 another.  (From the largest on: six.)"""
    g = torch.Generator().manual_seed(hd + nodes)
    k, q = torch.randn((8, 64), generator=g), torch.randn((8, 64, 8), generator=g)
    off = alone(Q, k, q, hd, nodes) / (k.double()[..., None] * q.double() * LN2) - 1
    assert float(off.abs().max()) <= 3.06 * EPS, off.abs().max() / EPS

@pytest.mark.parametrize("hd", [64, 128])
def test_f32_weights_are_as_close_as_32_bits(Q, hd):  # noqa: F811
    """All values of a request are alike, so that o = v whatever the weights are.  Weights that are cut make every product 2^-25.5
    smaller on average, and o with them; what is rounded to nearest goes either way: some ten roundings of 2^-24 / sqrt(3) on
    average, over 8 x hd different values (each with hundreds of weights) a mean below 4 x 10 ^ 0.5 x 2^-24 / (3 x 512) ^ 0.5 < 2^-25
    even if all weights of a value agreed, and 2^-27 as they do not (tens of different ones)."""
    g = torch.Generator().manual_seed(hd)
    n, m, H, ctx, page = 8, 64, 8, 48, 16
    per = (ctx + m) // page
    kv = Q.PagedKV(*(Dev(torch.zeros((n * per, 1, page, hd))) for _ in range(2)))
    v = torch.randn((n, 1, hd), generator=g).repeat(1, per * page, 1)
    kv.k.set(torch.randn((n * per, 1, page, hd), generator=g))
    kv.v.set(v.reshape(n * per, 1, page, hd))
    q = torch.randn((n * m, H, hd), generator=g)
    table = torch.arange(n * per, dtype=torch.int32).view(n, per)
    o, _ = attend(Q, kv, q, [m * i for i in range(n + 1)], table, [ctx + m] * n, None, nodes=m)
    off = o.double().view(n, m * H, hd) / v[:, :1].double() - 1
    assert abs(float(off.mean())) <= EPS / 8, off.mean() / EPS


@pytest.mark.parametrize("hd,nodes", [(64, 1), (64, 64), (128, 64), (64, 5)])
def test_f32_products_at_the_end_of_the_range(Q, hd, nodes):  # noqa: F811
    """1.998 x 1.7e38 is a 32-bit number, 2 x 2^127, which the first parts are rounded to, is not; likewise the largest number
    times 1.  The scores of either sign come out, with the roundings of any other product (one more of each sum)."""
    most = float(torch.finfo(torch.float32).max)
    k = torch.tensor([1.7e38, -1.7e38, most, -most, 1.0, 2.0 ** 127, 3.3e38, -3e38]).repeat(8)[None]
    q = torch.tensor([1.998, 1.998, 1.0, 1.0, 1.7e38, 1.99, 1.03, 1.1]).repeat(8)[None, :, None].repeat(1, 1, 8)
    off = alone(Q, k, q, hd, nodes) / (k.double()[..., None] * q.double() * LN2) - 1
    assert float(off.abs().max()) <= 7 * EPS

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes", [1, 11, 40])
def test_an_infinite_f32_key(Q, hd, nodes):  # noqa: F811
    """A score of -inf is a weight of 0, in every tile: rows whose queries turn an infinite key to that have the outputs that they
    have without the token, the others none that is a number.  Both for an earlier token and for a new one."""
    ctx, m = 70, 40
    kv, q, starts, table, lens, _, _ = case("f32", 8, 2, hd, 1, "head", [ctx + m], [m], 1, 3, Q)
    r = random.Random(hd)
    seen = above(forest(r, m))
    mask = torch.tensor([[signed(sum(1 << b for b in s))] for s in seen], dtype=torch.int64)
    q[:, :, 3] = q[:, :, 3].abs() + 0.125
    q[1::2, :, 3] *= -1.0
    for t in (7, ctx + 2):
        keep = kv.k.get()
        x = keep.clone()
        x[int(table[0, t]), :, 0, 3] = -math.inf
        without = table.clone()
        without[0, t] = -1
        wo, wl, bound, lb = attend_ref(kv, q, starts, without, lens, seen)
        kv.k.set(x)
        for tab in (table, widened(table, 1)):
            o, lse = (y.double() for y in attend(Q, kv, q, starts, tab, lens, mask, nodes))
            for i in range(m):
                if i % 2 and (t < ctx or t - ctx in seen[i]):
                    assert not bool(torch.isfinite(o[i]).any()), i
                else:
                    assert bool(((o - wo)[i].abs() <= bound[i]).all()) and bool(((lse - wl)[i].abs() <= lb[i]).all()), i
        kv.k.set(keep)


def test_no_row_behind_the_mask_is_accepted(Q):  # noqa: F811
    """A chain of 100 drafted rows whose tokens all fit, with a mask of one word: rows 64 .. 99 have mask 0 and are left out."""
    m = 100
    par, starts, lens = Dev(torch.arange(-1, m - 1, dtype=torch.int32).view(1, m)), dev_i32([0, m]), dev_i32([300])
    for words, want in ((1, 64), (2, 100)):
        pos, mask = i32(m), Dev(torch.zeros((m, words), dtype=torch.int64))
        Q.tree_plan(starts, lens, par, pos, mask)
        assert (mask.get() != 0).any(1).sum().item() == want
        out, rows = [i32(1), i32(1), i32(1)], [i32(m), i32(m), i32(m)]
        Q.tree_accept(starts, lens, par, dev_i32([5] * m), dev_i32([5] * m), dev_i32(list(range(m))), *out, *rows, mask=mask)
        assert [x.get().item() for x in out] == [want, 5, 200 + want]
        assert rows[0].get().tolist() == list(range(want)) + [-1] * (m - want) and rows[1].get().tolist() == [-1] * m


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_f32_values_in_parts_that_are_not_finite(Q, hd, bad):  # noqa: F811
    """Of an earlier token, alone in its step and beside new ones: no row has a number at that dim, and the others stay."""
    kv, q, starts, table, lens, seen, mask = case("f32", 4, 2, hd, 16, "head", [700], [40], 1, 3, Q, "tree")
    clean, _ = attend(Q, kv, q, starts, widened(table, 16), lens, mask)
    for at in (20, 657):
        keep = kv.v.get()
        x = keep.clone()
        x[int(table[0, at // 16]), 1, at % 16, 5] = bad
        kv.v.set(x)
        o, lse = attend(Q, kv, q, starts, widened(table, 16), lens, mask)
        kv.v.set(keep)
        assert not bool(torch.isfinite(o[:, 2:, 5]).any()) and bool(torch.isfinite(lse).all())
        o[:, 2:, 5] = clean[:, 2:, 5]
        assert torch.equal(o, clean)
