"""Pages that several requests hold, and rows of the cache to other slots (include/qserve.h) on the GPU, against sequential
accounts of the same rules."""
import random

import pytest
from test_gpu_qserve import Buffer, Dev, Q, Work, dev_i32, i32, make_cache  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Fork
# ---------------------------------------------------------------------------
def fork_ref(lens, table, source, keep, extra, ring, state, page, out, width):
    """The rules one request and one page after another.  out: table rows as they were before the call."""
    n, P, R = len(lens), len(extra), len(ring)
    head, count = state
    head = 0 if not 0 <= head < R else head
    count = min(max(count, 0), R)
    lens = [min(max(x, 0), width * page) for x in lens]
    pages = lambda t: -(-t // page)  # noqa: E731
    held = [[p if 0 <= p < P else -1 for p in table[r][:pages(lens[r])]] for r in range(n)]
    tokens = [0 if not 0 <= s < n else lens[s] if keep is None else min(max(keep[i], 0), lens[s]) for i, s in enumerate(source)]
    outside = {}
    for row in held:
        for p in row:
            if p >= 0:
                outside.setdefault(p, extra[p] + 1)
                outside[p] -= 1
    best = {}
    for i, t in enumerate(tokens):
        for e in range(pages(t)):
            p = held[source[i]][e]
            if p >= 0:
                best[p] = max(best.get(p, (0, 0)), (min(page, t - e * page), -i))
    free, asked = [ring[(head + k) % R] for k in range(count)], 0
    after, res = dict(outside), {k: [] for k in ("lens", "status", "src", "dst", "count")}
    new_table = [list(row) for row in out]
    for i, t in enumerate(tokens):
        row, part = [held[source[i]][e] for e in range(pages(t))], t % page
        p = row[-1] if part else -1
        copies = p >= 0 and (outside[p] > 0 or best[p] != (part, -i))
        asked += copies
        refused = copies and asked > count
        move = (-1, -1, 0)
        if refused:
            t, row = 0, []
        elif copies:
            got = free[asked - 1]
            row[-1] = got if 0 <= got < P else -1
            if row[-1] >= 0:
                move = (p * page, got * page, part)
        for e, x in enumerate(row):
            if x >= 0 and not (copies and e == len(row) - 1):
                after[x] += 1
            new_table[i][e] = x
        for k, v in zip(("lens", "status", "src", "dst", "count"), (t, 3 if refused else 0) + move):
            res[k].append(v)
    taken = min(asked, count)
    extra, ring, back = list(extra), list(ring), 0
    done = set()
    for row in held:
        for p in row:
            if p < 0 or p in done:
                continue
            done.add(p)
            extra[p] = max(after[p] - 1, 0)
            if after[p] <= 0:
                if back < R - count:
                    ring[(head + count + back) % R] = p
                back += 1
    res.update(table=new_table, extra=extra, ring=ring, state=[(head + taken) % R, count - taken + min(back, R - count)])
    return res


def fork_run(Q, lens, table, source, keep, extra, ring, state, page, width, in_place=False):  # noqa: F811
    n, m, P = len(lens), len(source), len(extra)
    wide = torch.full((max(n, 1), width + 3), 12345, dtype=torch.int32)
    for r in range(n):
        wide[r, :width] = torch.tensor(table[r], dtype=torch.int32)
    o = {"table": Dev(torch.full((max(m, 1), width + 1), -77, dtype=torch.int32)), "lens": i32(m), "status": i32(m), "state": i32(2), "src": i32(m),
         "dst": i32(m), "count": i32(m), "ring": dev_i32(ring)}
    e = dev_i32(extra)
    o["extra"] = e if in_place else i32(P)
    work = Work(Buffer(Q.paged_fork_work(n, m, P)))
    Q.paged_fork(dev_i32(lens), Dev(wide)[:, :width], dev_i32(source), e, o["ring"], dev_i32(state), page, o["table"][:, :width], o["lens"], o["status"],
                 o["extra"], o["state"], o["src"], o["dst"], o["count"], work, keep=None if keep is None else dev_i32(keep))
    got = {k: v.get().tolist() for k, v in o.items()}
    got["table"] = [row[:width] for row in got["table"][:m]]
    return got


def check_fork(Q, *args, **kw):  # noqa: F811
    lens, table, source, keep, extra, ring, state, page, width = args
    want = fork_ref(*args[:-1], [[-77] * width for _ in source], width)
    got = fork_run(Q, *args, **kw)
    for k, v in want.items():
        assert got[k] == v, k
    return got


class Pool:
    """Requests over pages with counts, as a server keeps them."""

    def __init__(self, pages, page, seed):
        self.r, self.page = random.Random(seed), page
        self.free = list(range(pages))
        self.r.shuffle(self.free)
        self.extra = [0] * pages

    def request(self, t, width, of=None, common=0):
        """A request of t tokens; of: shares the first `common` whole pages of another's."""
        n = -(-t // self.page)
        row = [of[e] if of is not None and e < common else self.free.pop() for e in range(n)]
        for p in row[:common] if of is not None else []:
            self.extra[p] += 1
        return row + [-1] * (width - n)

    def ring(self, size, head):
        ring = [-9] * size
        for k, p in enumerate(self.free):
            ring[(head + k) % size] = p
        return ring, [head, len(self.free)]


@pytest.mark.parametrize("seed,old,new,page,most", [(1, 1, 1, 16, 40), (2, 3, 8, 16, 100), (3, 40, 40, 4, 60), (4, 200, 100, 16, 300), (5, 7, 300, 1, 12),
                                                    (6, 30, 30, 64, 200), (7, 600, 1200, 8, 30), (8, 2, 5, 16, 9000)])
@pytest.mark.parametrize("cut", [False, True])
def test_fork_matches_the_account(Q, seed, old, new, page, most, cut):  # noqa: F811
    """Requests that share beginnings are continued by none, one or several, whole or cut; some pages are held from outside;
    with few free pages, some copies are refused."""
    width = -(-most // page) + 1
    pool = Pool(old * width + new + 20, page, seed)
    r, lens, table = pool.r, [], []
    for i in range(old):
        t = r.choice([0, 1, page, r.randint(0, most), r.randint(0, most)])
        t = min(t, most)
        if i and r.random() < 0.6:
            j = r.randrange(i)
            common = r.randint(0, min(t, lens[j]) // page)
            table.append(pool.request(t, width, table[j], common))
        else:
            table.append(pool.request(t, width))
        lens.append(t)
    for row in table[:3]:
        if row[0] >= 0:
            pool.extra[row[0]] += 1                     # a kept beginning
    source = [r.choice([-1, old, r.randrange(old), r.randrange(old), r.randrange(max(1, old // 4))]) for _ in range(new)]
    keep = [r.choice([-3, 0, 10 ** 9, page, r.randint(0, most)]) for _ in range(new)] if cut else None
    for few in (None, 2, 0):
        ring, state = pool.ring(len(pool.extra), r.randrange(len(pool.extra)))
        if few is not None:
            state = [state[0], min(few, state[1])]
        got = check_fork(Q, lens, table, source, keep, pool.extra, ring, state, page, width, in_place=few == 2)
        if few == 0 and not cut:
            assert got["state"][1] >= 0


def test_fork_conserves_pages(Q):  # noqa: F811
    """Twenty rounds of continuing, cutting and ending: every page is free, or held as often as its count says."""
    page, width, P, n = 8, 12, 400, 24
    pool = Pool(P, page, 3)
    r = pool.r
    lens = [r.randint(1, 60) for _ in range(n)]
    table = [pool.request(t, width) for t in lens]
    extra, (ring, state) = pool.extra, pool.ring(P, 5)
    for _ in range(20):
        source = [r.choice([-1, r.randrange(n), r.randrange(n), r.randrange(4)]) for _ in range(n)]
        keep = [r.randint(0, 96) for _ in range(n)]
        got = check_fork(Q, lens, table, source, keep, extra, ring, state, page, width)
        lens, table, extra, ring, state = got["lens"], got["table"], got["extra"], got["ring"], got["state"]
        held = [0] * P
        for row, t in zip(table, lens):
            for p in row[:-(-t // page)]:
                held[p] += 1
        free = [ring[(state[0] + k) % P] for k in range(state[1])]
        assert len(set(free)) == len(free) and all(held[p] == 0 for p in free)
        assert len(free) + sum(h > 0 for h in held) == P and all(extra[p] == max(h - 1, 0) for p, h in enumerate(held))
        # whatever is written next lies on a page of one request alone
        assert all(t % page == 0 or held[row[t // page]] == 1 for row, t in zip(table, lens))


def test_fork_values_out_of_range(Q):  # noqa: F811
    """Lengths, table entries, states, sources and a ring that holds no pages: nothing outside is touched, and the rules hold."""
    table = [[5, 2 ** 31 - 1, 3, -4], [0, 1, 2, 99], [6, 6, 7, 7]]
    for state in ([0, 4], [-3, 9], [100, 2], [5, -1], [2 ** 31 - 1, 2 ** 31 - 1]):
        for lens in ([30, 64, -5], [2 ** 31 - 1, 9, 17]):
            check_fork(Q, lens, table, [0, 0, 1, -2 ** 31, 3, 1], [20, 25, 10 ** 9, 4, 4, 33], [0, 0, 1, 0, 5, 0, 0, -3], [4, -1, 8, 2 ** 31 - 1, 2, 1], state, 8, 4)


def test_fork_without_requests(Q):  # noqa: F811
    got = check_fork(Q, [], [], [], None, [0, 2, 0], [2, 0], [1, 1], 16, 3)
    assert got["state"] == [1, 1]
    got = check_fork(Q, [], [], [0, -1], None, [0, 2, 0], [2, 0], [1, 1], 16, 3)
    assert got["lens"] == [0, 0]
    got = check_fork(Q, [20, 3], [[0, 1, -1], [2, -1, -1]], [], None, [0, 0, 0], [9, 9, 9, 9], [3, 0], 16, 3)
    assert got["ring"] == [1, 2, 9, 0] and got["state"] == [3, 3]


# ---------------------------------------------------------------------------
# Moves
# ---------------------------------------------------------------------------
def held(kv):
    return [x.get() for x in (kv.k, kv.v, kv.k_scale, kv.v_scale) if x is not None]


def moved(kv, before, moves):
    """The contents after single slots were moved one after another."""
    page = kv.k.shape[2]
    after = [x.clone() for x in before]
    for a, b in moves:
        for x in after:
            x[b // page, :, b % page] = x[a // page, :, a % page]
    return after


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("KVH,hd,page,order,layers", [(2, 48, 16, "head", 1), (8, 128, 5, "slot", 3), (1, 8, 1, "head", 70), (3, 24, 64, "slot", 2), (2, 256, 16, "head", 2)])
def test_moves_in_groups(Q, typ, KVH, hd, page, order, layers):  # noqa: F811
    """One after another within a group: chains through a slot, the same slot twice, a move onto itself, padding."""
    r, g = random.Random(hd), torch.Generator().manual_seed(hd)
    n_slots = 6 * 64
    caches = [make_cache(Q, typ, n_slots // page, KVH, page, hd, order, g) for _ in range(layers)]
    n_slots = n_slots // page * page
    ids = list(range(n_slots))
    r.shuffle(ids)
    src, dst, starts, moves = [], [], [0], []
    for size in (0, 1, 9, 30, 8, 17):
        mine = [ids.pop() for _ in range(size + 2)]
        for k in range(size):
            a, b = r.choice([(mine[k + 1], mine[k]), (r.choice(mine), r.choice(mine)), (mine[k], mine[k]), (-1, mine[0]), (mine[0], -5)])
            src.append(a)
            dst.append(b)
            if a >= 0 and b >= 0:
                moves.append((a, b))
        starts.append(len(src))
    before = [held(c) for c in caches]
    Q.paged_move(Q.PagedCaches(caches), dev_i32(src), dev_i32(dst), starts=dev_i32(starts))
    for c, x in zip(caches, before):
        for got, want in zip(held(c), moved(c, x, moves)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("KVH,hd,page,order,n", [(2, 48, 16, "head", 3), (8, 64, 16, "slot", 40), (1, 8, 1, "head", 200), (2, 128, 48, "head", 1)])
def test_moves_of_several_slots(Q, typ, KVH, hd, page, order, n):  # noqa: F811
    """Independent copies of runs of slots, across pages too, with and without counts, and ones that leave the cache."""
    g = torch.Generator().manual_seed(n)
    run = 7
    kv = make_cache(Q, typ, -(-2 * n * run // page) + 1, KVH, page, hd, order, g)
    slots = kv.k.shape[0] * page
    count = [(3 * i) % (run + 1) for i in range(n)] + [5, 2, -1, 2 ** 31 - 1]
    src, dst = [2 * i * run for i in range(n)] + [slots - 2, -1, 0, 0], [(2 * i + 1) * run for i in range(n)] + [0, 0, 0, 0]
    bad, before = dev_i32([10]), held(kv)
    Q.paged_move(kv, dev_i32(src), dev_i32(dst), count=dev_i32(count), bad=bad)
    want = moved(kv, before, [(a + s, b + s) for a, b, c in zip(src[:n], dst[:n], count[:n]) for s in range(c)])
    assert all(torch.equal(x, y) for x, y in zip(held(kv), want)) and bad.get().item() == 12
    before = held(kv)
    Q.paged_move(kv, dev_i32(src[:n]), dev_i32(dst[:n]))
    assert all(torch.equal(x, y) for x, y in zip(held(kv), moved(kv, before, list(zip(src[:n], dst[:n])))))


def test_moves_out_of_range(Q):  # noqa: F811
    kv = make_cache(Q, "bf16", 3, 2, 8, 16)
    before, bad = held(kv), dev_i32([0])
    Q.paged_move(kv, dev_i32([24, 0, 2 ** 31 - 1, 5]), dev_i32([0, 24, 1, 6]), starts=dev_i32([-7, 2, 2 ** 31 - 1]), bad=bad)
    assert all(torch.equal(x, y) for x, y in zip(held(kv), moved(kv, before, [(5, 6)]))) and bad.get().item() == 3
    before = held(kv)
    Q.paged_move(kv, dev_i32([1]), dev_i32([2]), starts=dev_i32([1, 0, -4]))           # falling: no moves
    Q.paged_move(kv, i32(0), i32(0))
    assert all(torch.equal(x, y) for x, y in zip(held(kv), before))


@pytest.mark.parametrize("width", [256, 257, 1100])
@pytest.mark.parametrize("new", [3, 70])
def test_fork_of_long_tables(Q, width, new):  # noqa: F811
    """Tables on both sides of what one block takes, full or nearly, with a shared beginning."""
    pool = Pool(5 * width + 80, 2, width)
    r = pool.r
    lens = [2 * width - 1, 2 * width - 2, 2 * width - 3, 5]
    table = [pool.request(lens[0], width)]
    for t in lens[1:]:
        table.append(pool.request(t, width, table[0], min(t // 2, width - 9)))
    ring, state = pool.ring(len(pool.extra), 3)
    source = [r.choice([0, 0, 1, 2, 3, -1]) for _ in range(new)]
    check_fork(Q, lens, table, source, [r.randint(0, 2 * width) for _ in range(new)], pool.extra, ring, state, 2, width)


def test_fork_of_nothing_over_many_pages(Q):  # noqa: F811
    """No old request, and more counts to carry over than one block copies."""
    extra = [(7 * i) % 5 for i in range(100_003)]
    for in_place in (False, True):
        got = check_fork(Q, [], [], [0, -1, 3], None, extra, [4, 5, 6], [1, 2], 16, 3, in_place=in_place)
        assert got["lens"] == [0, 0, 0] and got["extra"] == extra


@pytest.mark.parametrize("old,new,page,most", [(4, 9, 8, 60), (40, 70, 4, 50), (3, 20, 16, 5000)])
def test_fork_without_free_pages(Q, old, new, page, most):  # noqa: F811
    """Nothing is copied or taken; who would need a copy is refused, the others keep their source's pages, and what is written next
    lies on a page of one request alone."""
    width = -(-most // page) + 1
    pool = Pool(old * width, page, old)
    r = pool.r
    lens = [r.randint(page, most) for _ in range(old)]
    table = [pool.request(lens[0], width)]
    for t in lens[1:]:
        table.append(pool.request(t, width, table[0], r.randint(0, min(t, lens[0]) // page)))
    source, keep = [r.randrange(old) for _ in range(new)], [r.randint(0, 2 * most) for _ in range(new)]
    tokens = [min(keep[i], lens[s]) for i, s in enumerate(source)]
    ring, state = pool.ring(len(pool.extra), 2)
    got = fork_run(Q, lens, table, source, keep, pool.extra, ring, [state[0], 0], page, width)
    assert got["src"] == [-1] * new and got["dst"] == [-1] * new and got["count"] == [0] * new and got["state"][0] == state[0]
    assert got["status"].count(3) > 0 and got["status"].count(0) > 0 and set(got["status"]) == {0, 3}
    held = {}
    for i, (s, t, status, n) in enumerate(zip(source, tokens, got["status"], got["lens"])):
        assert n == (0 if status else t)
        for e in range(-(-n // page)):
            assert got["table"][i][e] == table[s][e]
            held[table[s][e]] = held.get(table[s][e], 0) + 1
        if status:
            assert t % page, "a request that writes to no page that it holds needs no copy"
    assert all(held[table[s][n // page]] == 1 for s, n in zip(source, got["lens"]) if n % page)
    assert all(got["extra"][p] == n - 1 for p, n in held.items())


@pytest.mark.parametrize("new", [9, 70])
def test_a_fork_that_was_refused_is_made_again(Q, new):  # noqa: F811
    """From the same lengths, table, counts and state, and the ring as the refused call has left it."""
    page, width, old = 8, 12, 6
    pool = Pool(old * width, page, new)
    r = pool.r
    lens = [r.randint(18, 90) for _ in range(old)]
    table = [pool.request(t, width) for t in lens]
    ring, state = pool.ring(len(pool.extra) + 5, 4)
    state = [state[0], 3]
    source, keep = [i % 3 for i in range(new)], [r.choice([3, 10, 17]) for _ in range(new)]
    got = check_fork(Q, lens, table, source, keep, pool.extra, ring, state, page, width)
    assert 3 in got["status"] and got["ring"] != ring
    fewer = [i if i < old else -1 for i in range(new)]
    again = check_fork(Q, lens, table, fewer, None, pool.extra, got["ring"], state, page, width)
    assert again["lens"] == lens + [0] * (new - old) and again["status"] == [0] * new and again["state"] == state
    assert [row[:-(-t // page)] for row, t in zip(again["table"], lens)] == [row[:-(-t // page)] for row, t in zip(table, lens)]
    one = check_fork(Q, lens, table, [0, 0, 1, 1, 2, 2], [17] * 6, pool.extra, got["ring"], state, page, width)
    assert one["status"] == [0] * 6 and one["dst"].count(-1) == 3
    assert sorted(d // page for d in one["dst"] if d >= 0) == sorted(pool.free[:3])
