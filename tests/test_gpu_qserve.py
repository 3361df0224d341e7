"""The serving operators (include/qserve.h) on the GPU against plain definitions in whole numbers and 64 bits: pages and
slots, rows into pages, attention of one token over pages, sampled rows, and a run of all four as a server makes it.

Host tensors are torch's, on the CPU; their device copies are the library's own buffers, so the tests do not depend on
whose HIP runtime the process loaded first."""
import ctypes as C
import math
import random

import numpy as np
import pytest

import qlib

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
EPS = 2.0 ** -24                 # half a step of a 32-bit float, relative to the value


@pytest.fixture(scope="module")
def Q():
    q = qlib.load()
    assert q.lib().qllama_device_count() > 0, "no GPU visible to the HIP library"
    q.sample_argmax(np.zeros((1, 4), np.float32))              # the library's first GPU call makes its stream
    return q


class Buffer:
    """Device memory of the library's, freed with its last view."""

    def __init__(self, nbytes):
        self.L, self.nbytes = qlib.load().lib(), nbytes
        self.p = self.L.qllama_dev_alloc(max(nbytes, 16))
        assert self.p

    def __del__(self):
        self.L.qllama_dev_free(self.p)


class Dev:
    """A device tensor as qllama.py takes them: a host tensor's shape and strides over a device copy of its storage.  Views
    (indexing, transpose, split, view) are views of the same device memory."""
    is_cuda = True

    def __init__(self, host, buffer=None, base=None):
        self.host = host
        if buffer is None:
            s = host.untyped_storage()
            buffer, base = Buffer(s.nbytes()), s.data_ptr()
            assert s.nbytes() == 0 or buffer.L.qllama_h2d(buffer.p, s.data_ptr(), s.nbytes()) == 0
        self.buffer, self.base = buffer, base

    dtype = property(lambda self: self.host.dtype)
    shape = property(lambda self: self.host.shape)
    stride = lambda self, *d: self.host.stride(*d)  # noqa: E731
    numel = lambda self: self.host.numel()  # noqa: E731
    element_size = lambda self: self.host.element_size()  # noqa: E731
    is_contiguous = lambda self: self.host.is_contiguous()  # noqa: E731

    def data_ptr(self):
        return self.buffer.p + (self.host.data_ptr() - self.base if self.host.numel() else 0)

    def _of(self, host):
        return Dev(host, self.buffer, self.base)

    def __getitem__(self, i):
        return self._of(self.host[i])

    def transpose(self, a, b):
        return self._of(self.host.transpose(a, b))

    def split(self, sizes, dim):
        return [self._of(x) for x in self.host.split(sizes, dim)]

    def get(self):
        """Its present contents."""
        s = self.host.untyped_storage()
        if s.nbytes():
            assert self.buffer.L.qllama_device_sync() == 0 and self.buffer.L.qllama_d2h(s.data_ptr(), self.buffer.p, s.nbytes()) == 0
        return self.host.clone()

    def set(self, x):
        """New contents (of the whole storage: the host's other values go too)."""
        self.host.copy_(x)
        s = self.host.untyped_storage()
        assert self.buffer.L.qllama_h2d(self.buffer.p, s.data_ptr(), s.nbytes()) == 0
        return self


def dev(x):
    return Dev(x.contiguous())


def i32(*shape):
    return Dev(torch.zeros(shape, dtype=torch.int32))


def dev_i32(x):
    return Dev(torch.tensor(x, dtype=torch.int32))


def same(a, b):
    return torch.equal(a.get() if isinstance(a, Dev) else a, b.get() if isinstance(b, Dev) else b)


# ---------------------------------------------------------------------------
# Plan: a sequential account of the same rules
# ---------------------------------------------------------------------------
def plan_ref(cached, added, table, ring, state, page, max_rows):
    n, width = table.shape
    table, ring = table.copy(), list(ring)
    R = len(ring)
    head, count = state
    head = head if 0 <= head < R else 0
    count = min(max(count, 0), R)
    room = width * page
    asked_pages = asked_rows = taken = back = 0
    lens, status, starts, slots, positions, requests = [], [], [], [], [], []
    returned = []
    for r in range(n):
        c, a = int(cached[r]), int(added[r])
        starts.append(len(slots))
        if not 0 <= c <= room:
            lens.append(0), status.append(2)
            continue
        have = -(-c // page)
        if a < 0:
            returned += [int(x) for x in table[r, :have]]
            lens.append(0), status.append(0)
            continue
        if c + a > room:
            lens.append(c), status.append(1)
            continue
        need = -(-(c + a) // page) - have
        asked_pages += need
        asked_rows += a
        if need and asked_pages > count:
            lens.append(c), status.append(3)
            continue
        if a and asked_rows > max_rows:
            lens.append(c), status.append(4)
            continue
        for j in range(need):
            table[r, have + j] = ring[(head + taken + j) % R]
        taken += need
        lens.append(c + a), status.append(0)
        for t in range(a):
            p = int(table[r, (c + t) // page])
            s = p * page + (c + t) % page
            slots.append(s if p >= 0 and s < 2 ** 31 else -1), positions.append(c + t), requests.append(r)
    starts.append(len(slots))
    for x in returned[:R - count]:
        ring[(head + count + back) % R] = x
        back += 1
    pad = max_rows - len(slots)
    return dict(table=table, ring=np.array(ring), lens=lens, status=status, starts=starts, state=[(head + taken) % R, count - taken + back],
                slots=slots + [-1] * pad, positions=positions + [0] * pad, requests=requests + [-1] * pad)


def plan_run(Q, cached, added, table, ring, state, page, max_rows):
    n = len(cached)
    o = dict(table=dev_i32(table), ring=dev_i32(ring), lens=i32(n), status=i32(n), starts=i32(n + 1), state=i32(2), slots=i32(max_rows),
             positions=i32(max_rows), requests=i32(max_rows))
    Q.paged_plan(dev_i32(cached), dev_i32(added), o["table"], o["ring"], dev_i32(state), page, o["lens"], o["status"], o["starts"],
                 o["state"], o["slots"], o["positions"], o["requests"])
    return {k: v.get().numpy() for k, v in o.items()}


def plan_case(seed, n, width, page, most_add, spare, max_rows):
    r = random.Random(seed)
    room = width * page
    cached = [r.randint(0, room) for _ in range(n)]
    added = [r.choice([0, 1, 1, 1, -1, r.randint(0, most_add)]) for _ in range(n)]
    have = [-(-c // page) for c in cached]
    ids = list(range(sum(have) + spare))
    r.shuffle(ids)
    table = np.full((n, width), -1)
    k = 0
    for i, h in enumerate(have):
        table[i, :h] = ids[k:k + h]
        k += h
    R = len(ids) + r.randint(0, 3) or 1
    ring = np.full(R, -7)
    head, count = r.randint(0, R - 1), len(ids) - k
    for i in range(count):
        ring[(head + i) % R] = ids[k + i]
    return cached, added, table, ring, [head, count], page, max_rows


@pytest.mark.parametrize("seed,n,width,page,most_add,spare,max_rows", [
    (1, 1, 1, 1, 1, 1, 1), (2, 7, 5, 16, 40, 30, 300), (3, 64, 12, 16, 100, 50, 1000), (4, 255, 9, 7, 20, 100, 400), (5, 256, 3, 64, 90, 40, 4000),
    (6, 257, 6, 16, 3, 4, 100), (7, 1000, 4, 8, 9, 2000, 3000), (8, 40, 30, 1, 25, 500, 900), (9, 8192, 2, 16, 5, 3000, 9000), (10, 50, 128, 16, 2000, 6000, 70000),
    (11, 33, 4, 16, 10, 0, 0), (12, 5, 2, 1000003, 1000000, 8, 100000)])
def test_plan_matches_the_account(Q, seed, n, width, page, most_add, spare, max_rows):
    args = plan_case(seed, n, width, page, most_add, spare, max_rows)
    want, got = plan_ref(*args), plan_run(Q, *args)
    for k, v in want.items():
        assert np.array_equal(got[k], np.asarray(v).reshape(got[k].shape)), k


def test_plan_values_out_of_range(Q):
    """Lengths, states and entries no host can refuse: each as documented, nothing outside the buffers written."""
    table = np.array([[3, -5], [4, 2 ** 30], [6, 7], [8, 9], [1, 2]])
    for state in ([0, 4], [-3, 9], [100, 2], [5, -1], [2 ** 31 - 1, 2 ** 31 - 1]):
        args = ([17, 20, -1, 33, 32], [1, 1, 2, 1, 1], table, np.arange(10, 16), state, 16, 8)
        want, got = plan_ref(*args), plan_run(Q, *args)
        for k, v in want.items():
            assert np.array_equal(got[k], np.asarray(v).reshape(got[k].shape)), (k, state)
        assert want["status"] == [0, 0, 2, 2, 1] and want["slots"][:2] == [-1, -1]


def test_plan_without_requests_and_between_sentinels(Q):
    slots, other = Dev(torch.full((12,), 99, dtype=torch.int32)), Dev(torch.full((12,), 99, dtype=torch.int32))
    ring, state, out, starts = dev_i32([5, 6]), dev_i32([1, 2]), i32(2), i32(1)
    e = i32(0)
    Q.paged_plan(e, e, i32(0, 3), ring, state, 16, e, e, starts, out, slots[4:8], other[2:6], other[7:11])
    assert out.get().tolist() == [1, 2] and starts.get().tolist() == [0] and slots.get().tolist() == [99] * 4 + [-1] * 4 + [99] * 4
    assert other.get().tolist() == [99, 99, 0, 0, 0, 0, 99, -1, -1, -1, -1, 99]


def test_plan_a_request_that_needs_no_page_is_not_held_up(Q):
    args = ([16, 3, 16], [1, 1, 1], np.array([[0, -1], [1, -1], [2, -1]]), np.array([9, 9]), [0, 0], 16, 3)
    got = plan_run(Q, *args)
    assert got["status"].tolist() == [3, 0, 3] and got["slots"].tolist() == [1 * 16 + 3, -1, -1] and got["lens"].tolist() == [16, 4, 16]


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
def make_cache(Q, typ, pages, KVH, page, hd, order="head", gen=None):
    """A cache of random contents and its view; order "slot": heads beside each other within a slot."""
    shape = (pages, KVH, page, hd) if order == "head" else (pages, page, KVH, hd)
    turn = (lambda x: x) if order == "head" else (lambda x: x.transpose(1, 2))
    t, s = [], [None, None]
    for _ in range(2):
        x = torch.randint(-127, 128, shape, generator=gen).to(torch.int8) if typ == "i8" else torch.randn(shape, generator=gen).to(DT[typ])
        t.append(turn(Dev(x)))
    if typ == "i8":
        s = [turn(Dev(0.005 + 0.03 * torch.rand(shape[:3], generator=gen))) for _ in range(2)]
    return Q.PagedKV(t[0], t[1], s[0], s[1])


def tables(n, hd):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
    return a.cos().float(), a.sin().float()


def rotate32(x, c, s):
    """Each product and each sum rounded to 32 bits (elementwise torch operations round so)."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def codes(x):
    top = x.abs().amax(-1)
    scale = torch.where(top > 0, top * torch.tensor(np.float32(1) / np.float32(127), device=x.device), torch.ones_like(top))
    return torch.round(x * (1.0 / scale)[..., None]).clamp(-127, 127).to(torch.int8), scale


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("H,KVH,hd,page,rows,order,packed", [
    (6, 2, 48, 16, 1, "head", True), (8, 8, 64, 5, 37, "slot", True), (32, 8, 128, 16, 70, "head", False), (3, 1, 8, 1, 9, "head", True),
    (5, 5, 256, 64, 20, "slot", False), (40, 1, 72, 24, 33, "head", True)])
def test_append_stores_what_the_reference_rounds_to(Q, typ, H, KVH, hd, page, rows, order, packed):
    g = torch.Generator().manual_seed(hd + rows)
    pages = -(-rows // page) + 2
    kv = make_cache(Q, typ, pages, KVH, page, hd, order, g)
    before = [x.get() for x in (kv.k, kv.v)]
    slots = torch.randperm(pages * page, generator=g)[:rows].to(torch.int32)
    if rows > 3:
        slots[-2:] = -1                                        # padding
        slots[0] = -2 ** 31
    pos = torch.randint(0, 50, (rows,), generator=g, dtype=torch.int32)
    cos, sin = tables(50, hd)
    qkv = torch.randn((rows, H + 2 * KVH, hd), generator=g)
    qkv[0, H] = 0.0                                            # a key of zeros
    q, k, v = qkv.split([H, KVH, KVH], 1)
    dq, dk, dv = Dev(qkv).split([H, KVH, KVH], 1) if packed else (dev(q), dev(k), dev(v))
    q_out, bad = Dev(torch.full((rows + 1, H, hd), 7.0)), dev_i32([5])
    Q.paged_append(kv, dk, dv, Dev(slots), q=dq, q_out=q_out[:rows], positions=Dev(pos), cos=Dev(cos), sin=Dev(sin), bad=bad)
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    got = q_out.get()
    assert torch.equal(got[:rows], rotate32(q, c, s)) and bool((got[rows] == 7.0).all())
    assert bad.get().item() == 5
    held = (slots >= 0).nonzero()[:, 0]
    at = slots[held].long()
    for got, want, sc, x in ((kv.k, before[0], kv.k_scale, rotate32(k, c, s)), (kv.v, before[1], kv.v_scale, v)):
        x = x[held]
        if typ == "i8":
            x, scale = codes(x)
            assert torch.equal(sc.get()[at // page, :, at % page], scale)
        want[at // page, :, at % page] = x.to(want.dtype)
        assert torch.equal(got.get(), want)


def test_append_rows_out_of_range_and_unaligned(Q):
    """Positions outside the tables: nothing of the row is written; slots outside the cache: no key and value.  Rows and
    tables on odd addresses give the same values."""
    g = torch.Generator().manual_seed(3)
    H, KVH, hd, page, rows = 4, 2, 64, 16, 6
    kv = make_cache(Q, "f32", 2, KVH, page, hd, gen=g)
    was = kv.k.get()
    raw = torch.randn(rows * (H + 2 * KVH) * hd + 1, generator=g)[1:]
    qkv = raw.view(rows, H + 2 * KVH, hd)
    q, k, v = qkv.split([H, KVH, KVH], 1)
    dq, dk, dv = Dev(qkv).split([H, KVH, KVH], 1)
    assert dq.data_ptr() % 16 == 4
    cos, sin = tables(9, hd)
    slots, pos = [0, 32, 5, 2 ** 31 - 1, 7, -1], torch.tensor([8, 1, 9, 2, -1, 3])
    q_out, bad = Dev(torch.full((rows, H, hd), 7.0)), dev_i32([0])
    Q.paged_append(kv, dk, dv, dev_i32(slots), q=dq, q_out=q_out, positions=dev_i32(pos.tolist()), cos=Dev(cos), sin=Dev(sin), bad=bad)
    assert bad.get().item() == 4
    ok = torch.tensor([0, 1, 3, 5])
    got = q_out.get()
    assert torch.equal(got[ok], rotate32(q[ok], cos[pos[ok]][:, None], sin[pos[ok]][:, None])) and bool((got[[2, 4]] == 7.0).all())
    was[0, :, 0] = rotate32(k[0], cos[8], sin[8])
    assert same(kv.k, was)


def test_append_without_queries_or_rotation_and_in_place(Q):
    g = torch.Generator().manual_seed(8)
    kv = make_cache(Q, "bf16", 3, 2, 8, 64, gen=g)
    k, v = torch.randn(4, 2, 64, generator=g), torch.randn(4, 2, 64, generator=g)
    k[0, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.00390625])          # a tie rounds to even
    slots = torch.tensor([23, 0, 9, 16], dtype=torch.int32)
    Q.paged_append(kv, Dev(k), Dev(v), Dev(slots))
    at = slots.long()
    gk, gv = kv.k.get()[at // 8, :, at % 8], kv.v.get()[at // 8, :, at % 8]
    assert torch.equal(gk.isnan(), k.isnan()) and torch.equal(gk.nan_to_num(1.0), k.bfloat16().nan_to_num(1.0)) and torch.equal(gv, v.bfloat16())
    q = torch.randn(4, 6, 64, generator=g)
    cos, sin = tables(5, 64)
    pos = torch.tensor([4, 0, 2, 2], dtype=torch.int32)
    dq = Dev(q.clone())
    Q.paged_append(kv, Dev(k), Dev(v), Dev(slots), q=dq, q_out=dq, positions=Dev(pos), cos=Dev(cos), sin=Dev(sin))
    assert same(dq, rotate32(q, cos[pos.long()][:, None], sin[pos.long()][:, None]))


def test_append_int8_codes_of_nan(Q):
    """A NaN gets code 0 and does not count for the scale; the other elements keep theirs."""
    kv = make_cache(Q, "i8", 1, 1, 4, 16)
    k = torch.linspace(-1, 1, 16).view(1, 1, 16).clone()
    k[0, 0, 3] = float("nan")
    Q.paged_append(kv, Dev(k), Dev(k), dev_i32([2]))
    want, scale = codes(k.nan_to_num(0.0))
    assert torch.equal(kv.k.get()[0, 0, 2], want[0, 0]) and kv.k_scale.get()[0, 0, 2].item() == scale.item()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def attend_ref(kv, q, table, lens, scale=None, uneven=False):
    """o, lse, and a bound of what 32-bit arithmetic may differ from them, all in 64 bits.

    A score is a sum of 3 hd products at most (three parts of a query), so it is off by (3 hd + 4) EPS sum |q k| scale;
    a weight by that of its score and of the maximum, the exponential's argument (2 EPS |score| each) and the exponential
    (4 EPS); the sums over len tokens, in parts of three, by (3 len + 16) EPS of sum w |v|.

    uneven (int8): a weight times its scale enters as two 16-bit floats of 11 bits, the largest such product between 2^14 and
    2^15 (2^13 after a larger score has come, which halves it at most); the second float's last bit is 2^-24 or the product's
    own 2^-22, so each product is off by 2^-24 / 2^13 = 2^-37 of the largest, and each of len tokens adds that times its code,
    127 at most."""
    n, H, hd = q.shape
    KVH, page = kv.k.shape[1], kv.k.shape[2]
    G = H // KVH
    scale = scale or 1.0 / math.sqrt(hd)
    o, lse, bound, lse_bound = (torch.zeros(s, dtype=torch.float64) for s in ((n, H, hd), (n, H), (n, H, hd), (n, H)))
    lse.fill_(-math.inf)
    k_all, v_all = kv.k.get().double(), kv.v.get().double()
    if kv.k_scale is not None:
        k_all, v_all = k_all * kv.k_scale.get().double()[..., None], v_all * kv.v_scale.get().double()[..., None]
    q = q.double()
    for r, length in enumerate(lens):
        length = min(max(length, 0), table.shape[1] * page)
        t = torch.arange(length)
        p = table[r, t // page].long()
        t = t[(p >= 0) & (p < k_all.shape[0])]
        p = table[r, t // page].long()
        if not len(t):
            continue
        for h in range(H):
            k, v = k_all[p, h // G, t % page], v_all[p, h // G, t % page]
            s = (k @ q[r, h]) * scale
            z = torch.logsumexp(s, 0)
            w = torch.exp(s - z)
            ds = ((3 * hd + 4) * EPS * (k.abs() @ q[r, h].abs()) * scale + 2 * EPS * s.abs()).max()
            dw = 2 * ds + 4 * EPS * s.abs().max() + 8 * EPS
            o[r, h], lse[r, h] = w @ v, z
            bound[r, h] = (2 * dw + (3 * len(t) + 16) * EPS) * (w @ v.abs())
            if uneven:
                bound[r, h] += len(t) * 127 * 2.0 ** -37 * (w * kv.v_scale.get().double()[p, h // G, t % page]).max()
            lse_bound[r, h] = dw + (len(t) + 16) * EPS + 4 * EPS * abs(z)
    return o, lse, bound, lse_bound


def pages_for(lens, page, width, n_pages, seed):
    """A table of distinct pages in random order; entries behind a request's pages point outside the cache."""
    r = random.Random(seed)
    ids = list(range(n_pages))
    r.shuffle(ids)
    table = np.full((len(lens), width), 2 ** 31 - 1)
    for i, x in enumerate(lens):
        for j in range(min(width, -(-max(x, 0) // page))):
            table[i, j] = ids.pop()
    return torch.tensor(table, dtype=torch.int32)


def attend(Q, kv, q, table, lens, **kw):
    n, H, _ = q.shape
    o, lse = Dev(torch.full(q.shape, 7.0)), Dev(torch.full((n, H), 7.0))
    work = Buffer(Q.paged_attention_work(kv, n, H))
    Q.paged_attention(kv, Dev(q), Dev(table), dev_i32(lens), o, Work(work), lse=lse, **kw)
    return o.get(), lse.get()


class Work:
    """A workspace: device bytes."""
    is_cuda = True

    def __init__(self, buffer):
        self.buffer = buffer

    data_ptr = lambda self: self.buffer.p  # noqa: E731
    numel = lambda self: self.buffer.nbytes  # noqa: E731
    element_size = lambda self: 1  # noqa: E731


def widened(table, page):
    """The table with room for 5000 tokens more, in which there are no pages: long tables are served otherwise than short ones."""
    return torch.cat([table, torch.full((len(table), 5000 // page), 2 ** 31 - 1, dtype=torch.int32)], 1)


def check(Q, kv, q, table, lens, uneven=False, **kw):
    wo, wl, bound, lb = attend_ref(kv, q, table, lens, kw.get("scale"), uneven)
    empty = torch.isinf(wl)
    for t in (table, widened(table, kv.k.shape[2])):
        o, lse = attend(Q, kv, q, t, lens, **kw)
        o, lse = o.double(), lse.double()
        assert bool(((o - wo).abs() <= bound).all()), ((o - wo).abs() - bound).max()
        assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all()) and bool((o[empty] == 0).all())
        assert bool(((lse - wl).abs()[~empty] <= lb[~empty]).all())


SHAPES = [(6, 2, 48), (32, 8, 64), (8, 2, 128), (4, 4, 128), (5, 1, 8), (20, 1, 72), (33, 1, 256), (16, 1, 160)]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("H,KVH,hd", SHAPES)
@pytest.mark.parametrize("page,order", [(16, "head"), (5, "slot"), (48, "slot"), (1, "head")])
def test_attention_matches_the_definition(Q, typ, H, KVH, hd, page, order):
    """Lengths of none, one, at and around the steps of 16 and 32 keys and the pages, in one ragged batch."""
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 65, 100, 257, -4]
    g = torch.Generator().manual_seed(H + hd)
    need = sum(-(-max(x, 0) // page) for x in lens)
    kv = make_cache(Q, typ, need + 3, KVH, page, hd, order, g)
    q = torch.randn((len(lens), H, hd), generator=g) * 2.0
    check(Q, kv, q, pages_for(lens, page, -(-257 // page) + 1, need + 3, hd), lens)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("lens,page", [([5000], 16), ([4097, 3], 64), ([1, 6001, 40], 24), ([300] * 70, 16), ([900, 0, 31, 1700] * 9, 128)])
def test_attention_split_and_joined(Q, typ, lens, page):
    """Long and many requests: shares that end inside a tile, begin in another's, and hold several."""
    g = torch.Generator().manual_seed(len(lens))
    need = sum(-(-x // page) for x in lens)
    kv = make_cache(Q, typ, need + 1, 2, page, 64, "head", g)
    q = torch.randn((len(lens), 6, 64), generator=g)
    check(Q, kv, q, pages_for(lens, page, max(-(-x // page) for x in lens), need + 1, 1), lens)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("page", [1, 7, 16, 48])
def test_attention_reads_the_row_that_the_table_names(Q, typ, page):
    """One key stands out by more than a float's range of weights: the output is its value row, as held, and moves with it."""
    KVH, G, hd, n = 2, 3, 64, 9
    g = torch.Generator().manual_seed(page)
    lens = [1, 20, 33, 64, 100, 129, 200, 511, 700]
    need = sum(-(-x // page) for x in lens)
    kv = make_cache(Q, typ, need, KVH, page, hd, "head", g)
    table = pages_for(lens, page, -(-700 // page), need, 5)
    r = random.Random(page)
    at = [r.randrange(x) for x in lens]
    k, values = torch.zeros_like(kv.k.host), kv.v.get()
    for i, t in enumerate(at):
        k[int(table[i, t // page]), :, t % page, 5] = 100
    kv.k.set(k)
    if typ == "i8":
        kv.k_scale.set(torch.ones_like(kv.k_scale.host))
        kv.v_scale.set(torch.full_like(kv.v_scale.host, 0.25))
    q = torch.zeros((n, KVH * G, hd))
    q[:, :, 5] = 64.0                                        # a score of 800 against 0
    o, _ = attend(Q, kv, q, table, lens)
    for i, t in enumerate(at):
        v = values[int(table[i, t // page]), :, t % page].float() * (0.25 if typ == "i8" else 1.0)
        assert torch.equal(o[i], v.repeat_interleave(G, 0)), (i, t)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_leaves_out_what_is_no_token(Q, typ, page):
    """Slots behind the tokens hold NaN and infinities, pages lie outside the cache, lengths exceed the table: none counts."""
    KVH, hd = 2, 64
    g = torch.Generator().manual_seed(9)
    lens = [3, 40, 77, 10 ** 9, 2 ** 31 - 1, 50]
    width = 16
    held = [min(x, width * page) for x in lens]
    need = sum(-(-x // page) for x in held)
    kv = make_cache(Q, typ, need + 2, KVH, page, hd, "head", g)
    table = pages_for(held, page, width, need, 3)
    table[2, 1] = -1
    table[3, 0] = need + 2
    table[5] = -2 ** 31
    used = torch.zeros((need + 2, page), dtype=torch.bool)
    for i, x in enumerate(held):
        for t in range(x):
            p = int(table[i, t // page])
            if 0 <= p < need + 2:
                used[p, t % page] = True
    q = torch.randn((len(lens), 4, hd), generator=g)

    def stale(a, b):                                          # what the slots that hold no token are filled with
        if typ == "i8":
            empty = ~used[:, None, :].expand(kv.k_scale.shape)
            kv.k_scale.set(kv.k_scale.host.masked_fill(empty, a))
            kv.v_scale.set(kv.v_scale.host.masked_fill(empty, b))
        else:
            empty = ~used[:, None, :, None].expand(kv.k.shape)
            kv.k.set(kv.k.host.masked_fill(empty, a))
            kv.v.set(kv.v.host.masked_fill(empty, b))

    for t in (table, widened(table, page)):
        stale(float("nan"), float("inf"))
        o, lse = attend(Q, kv, q, t, lens)
        stale(0.0, 0.0)
        o2, lse2 = attend(Q, kv, q, t, lens)
        assert bool(torch.isfinite(o).all()) and torch.equal(o, o2) and torch.equal(lse, lse2)
        assert bool((o[5] == 0).all()) and bool(torch.isinf(lse[5]).all())
    check(Q, kv, q, table, lens)


@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("order", ["up", "down", "mixed", "one", "zero", "unlikely"])
def test_attention_int8_scales_of_every_size(Q, page, order):
    """Scales of values that run over sixty powers of ten, in rising, falling and mixed order, a single enormous one, ones
    of 0, and an enormous one whose weight is tiny."""
    H, KVH, hd, n = 8, 2, 64, 90
    pages = -(-n // page)
    kv = make_cache(Q, "i8", pages, KVH, page, hd)
    slots = torch.arange(pages * page)
    e = {"up": slots * 0.6 - 27.0, "down": 27.0 - slots * 0.6, "mixed": (slots * 37 % 90) * 0.6 - 27.0, "one": torch.where(slots == 40, 20.0, -5.0),
         "zero": slots * 0.0, "unlikely": torch.where(slots == 3, 18.0, 0.0)}[order].double()
    scale = (10.0 ** e).float().reshape(pages, 1, page).expand(pages, KVH, page).contiguous()
    if order == "zero":
        scale[:, :, ::3] = 0.0
    kv.v_scale.set(scale)
    if order == "unlikely":                                   # the other keys' scores lie far above that one's
        k = kv.k.get()
        k[:] = torch.where(k >= 0, k.clamp(min=20), k.clamp(max=-20))
        k[:, :, 1:] = k[:, :, :1]
        k[0, :, 3] = -k[0, :, 3]
        kv.k.set(k)
        kv.k_scale.set(torch.full_like(scale, 0.05))
    q = torch.randn((2, H, hd), generator=torch.Generator().manual_seed(4))
    if order == "unlikely":
        q = kv.k.get()[0, :, 0].float().repeat_interleave(H // KVH, 0).expand(2, H, hd) * 0.02 * torch.tensor([1.0, 2.0])[:, None, None]
    table = torch.arange(pages, dtype=torch.int32).expand(2, pages).contiguous()
    check(Q, kv, q.contiguous(), table, [n, n - 7], uneven=True)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("H,KVH,hd", [(6, 2, 48), (8, 8, 64), (40, 2, 64), (32, 8, 128), (4, 1, 200)])
@pytest.mark.parametrize("page,n", [(16, 1), (16, 20), (12, 20), (16, 40)])
def test_attention_of_short_and_of_long_tables(Q, typ, H, KVH, hd, page, n):
    """Lengths around those at which the waves of a block that takes a short request have one, two or more steps each."""
    r = random.Random(hd + n)
    lens = ([240] if n == 1 else [0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 240, 255, 256, -1])
    lens += [r.randint(0, 260) for _ in range(n - len(lens))]
    g = torch.Generator().manual_seed(hd)
    need = sum(-(-max(x, 0) // page) for x in lens)
    kv = make_cache(Q, typ, need + 2, KVH, page, hd, "head", g)
    q = torch.randn((n, H, hd), generator=g) * 2.0
    check(Q, kv, q, pages_for(lens, page, -(-260 // page), need + 2, hd), lens)


def test_attention_int8_scores_that_rise_slowly(Q):
    """One enormous scale ahead of scores that rise by less than a factor of 2 a step of 32 keys, until its product is like
    the others': as many equal requests as make every wave take all of a request's 45 steps."""
    n, KVH, hd, page, steps = 1024, 2, 8, 32, 45
    kv = make_cache(Q, "i8", steps, KVH, page, hd, gen=torch.Generator().manual_seed(9))
    k, v = torch.zeros((steps, KVH, page, hd), dtype=torch.int8), kv.v.get()
    k[..., 0] = 127
    v[0, :, 0] = torch.tensor([127, 0, 0, 0, -127, 0, 0, 0], dtype=torch.int8)
    rise = 0.9 * math.log(2.0) * torch.arange(steps)[:, None, None].expand(steps, KVH, page) / 127
    scale = torch.ones((steps, KVH, page))
    scale[0, :, 0] = 2.0 ** 40
    kv.k.set(k), kv.v.set(v), kv.k_scale.set(rise.contiguous()), kv.v_scale.set(scale)
    q = torch.ones((1, KVH, hd))
    table = torch.arange(steps, dtype=torch.int32)[None]
    o, lse = attend(Q, kv, q.expand(n, KVH, hd).contiguous(), table.expand(n, steps).contiguous(), [steps * page] * n, scale=1.0)
    wo, wl, bound, lb = attend_ref(kv, q, table, [steps * page], 1.0, uneven=True)
    assert bool(((o.double() - wo).abs() <= bound).all()) and bool(((lse.double() - wl).abs() <= lb).all())


def test_attention_large_scores_and_nan(Q):
    """Scores of thousands and queries of f16's border; a NaN query spoils its own head only."""
    for typ in ("f32", "f16", "bf16", "i8"):
        g = torch.Generator().manual_seed(4)
        kv = make_cache(Q, typ, 8, 2, 16, 64, "head", g)
        q = torch.randn((2, 4, 64), generator=g)
        q[0] *= 3000.0
        q[1] *= 1e-6
        lens = [60, 33]
        table = pages_for([60, 33], 16, 4, 8, 2)
        check(Q, kv, q, table, lens)
        spoilt = q.clone()
        spoilt[0, 1, 7] = float("nan")
        for t in (table, widened(table, 16)):
            o, _ = attend(Q, kv, q, t, lens)
            o2, _ = attend(Q, kv, spoilt, t, lens)
            assert bool(o2[0, 1].isnan().all())
            assert torch.equal(o2[0, [0, 2, 3]], o[0, [0, 2, 3]]) and torch.equal(o2[1], o[1])


@pytest.mark.parametrize("typ", ["f32", "i8"])
def test_attention_many_requests_most_of_them_empty(Q, typ):
    """700 requests, runs of empty ones among them longer than what a wave looks at at once, the last ones empty too."""
    g = torch.Generator().manual_seed(11)
    r = random.Random(5)
    lens = [r.choice([1, 17, 90]) if r.random() < 0.1 and not 200 < i < 420 and i < 690 else 0 for i in range(700)]
    need = sum(-(-x // 16) for x in lens)
    kv = make_cache(Q, typ, need, 2, 16, 64, "head", g)
    q = torch.randn((700, 2, 64), generator=g)
    check(Q, kv, q, pages_for(lens, 16, 6, need, 1), lens)
    o, lse = attend(Q, kv, q, pages_for([0] * 700, 16, 6, need, 1), [0] * 700)
    assert bool((o == 0).all()) and bool(torch.isinf(lse).all())


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
def test_attention_shared_pages_and_equal_requests(Q, typ):
    """Requests that share a prefix's pages, and the same request twice: equal bits where equal work is asked of equal places
    in a share, and the definition's values anyway."""
    g = torch.Generator().manual_seed(14)
    kv = make_cache(Q, typ, 12, 2, 32, 128, "head", g)
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 2, 3], [7, 7, 7, 7]], dtype=torch.int32)
    q = torch.randn((4, 4, 128), generator=g)
    q[2] = q[0]
    check(Q, kv, q, table, [128, 100, 128, 97])


def test_attention_16_heads_a_group_of_256_in_a_graph(Q):
    """The largest queries in LDS (set as the launch's own size) under capture."""
    g = torch.Generator().manual_seed(15)
    kv = make_cache(Q, "bf16", 30, 1, 16, 256, "head", g)
    lens = [300, 77]
    table = pages_for(lens, 16, 19, 30, 1)
    q = torch.randn((2, 16, 256), generator=g)
    want = attend(Q, kv, q, table, lens)
    dq, dt, dn, o, lse = Dev(q), Dev(table), dev_i32(lens), Dev(torch.zeros_like(q)), Dev(torch.zeros((2, 16)))
    work = Work(Buffer(Q.paged_attention_work(kv, 2, 16)))
    graph = Graph(lambda s: Q.paged_attention(kv, dq, dt, dn, o, work, lse=lse, stream=s))
    for _ in range(3):
        o.set(torch.zeros_like(q))
        graph.replay()
        assert same(o, want[0]) and same(lse, want[1])


def test_attention_scale_strides_and_sentinels(Q):
    """A given scale; queries inside packed rows, outputs with room behind every row, a table inside a larger one."""
    g = torch.Generator().manual_seed(2)
    H, KVH, hd, n = 6, 3, 40, 5
    lens = [50, 1, 0, 33, 64]
    kv = make_cache(Q, "bf16", 20, KVH, 16, hd, "slot", g)
    qkv = torch.randn((n, H + 2 * KVH, hd), generator=g)
    big = torch.full((n, 9), -1, dtype=torch.int32)
    big[:, :4] = pages_for(lens, 16, 4, 20, 8)
    o_all, lse_all = Dev(torch.full((n, H + 2, hd), 7.0)), Dev(torch.full((n, H + 1), 7.0))
    Q.paged_attention(kv, Dev(qkv)[:, :H], Dev(big)[:, :4], dev_i32(lens), o_all[:, :H], Work(Buffer(Q.paged_attention_work(kv, n, H))),
                      lse=lse_all[:, :H], scale=0.3)
    q, table = qkv[:, :H].contiguous(), big[:, :4].contiguous()
    o, lse = attend(Q, kv, q, table, lens, scale=0.3)
    got, got_lse = o_all.get(), lse_all.get()
    assert torch.equal(got[:, :H], o) and torch.equal(got_lse[:, :H], lse)
    assert bool((got[:, H:] == 7.0).all()) and bool((got_lse[:, H:] == 7.0).all())
    check(Q, kv, q, table, lens, scale=0.3)


def test_attention_pages_behind_two_billion_elements(Q):
    """Pages whose offsets pass 32 bits, in elements and in bytes (2.3 G elements; only five pages are filled)."""
    pages, KVH, page, hd = 17600, 8, 16, 1024 // 8
    one = KVH * page * hd
    ids = [17599, 0, 16384, 8200, 17598]
    g = torch.Generator().manual_seed(6)
    host = torch.randn((2, len(ids), KVH, page, hd), generator=g).bfloat16()
    buffers = [Buffer(2 * one * pages) for _ in range(2)]
    for b, x in zip(buffers, host):
        for p, y in zip(ids, x):
            y = y.contiguous()
            assert b.L.qllama_h2d(b.p + 2 * one * p, y.data_ptr(), 2 * one) == 0

    class Far:                                                # a tensor of the whole cache that has no host copy
        is_cuda, dtype, shape = True, torch.bfloat16, (pages, KVH, page, hd)
        stride = lambda self, *d: (one, page * hd, hd, 1) if not d else (one, page * hd, hd, 1)[d[0]]  # noqa: E731
        numel = lambda self: one * pages  # noqa: E731

        def __init__(self, b):
            self.data_ptr = lambda: b.p

    kv = Q.PagedKV(Far(buffers[0]), Far(buffers[1]))
    q = torch.randn((1, 8, hd), generator=g)
    o, lse = attend(Q, kv, q, torch.tensor([ids], dtype=torch.int32), [75])
    small = Q.PagedKV(dev(host[0]), dev(host[1]))
    o2, lse2 = attend(Q, small, q, torch.tensor([[0, 1, 2, 3, 4]], dtype=torch.int32), [75])
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    rows = torch.randn((1, KVH, hd), generator=g)
    Q.paged_append(kv, Dev(rows), Dev(rows), dev_i32([17599 * page + 15]))
    got = torch.empty((KVH, page, hd), dtype=torch.bfloat16)
    for b in buffers:
        assert b.L.qllama_device_sync() == 0 and b.L.qllama_d2h(got.data_ptr(), b.p + 2 * one * 17599, 2 * one) == 0
        assert torch.equal(got[:, 15], rows[0].bfloat16())


# ---------------------------------------------------------------------------
# Sampled rows
# ---------------------------------------------------------------------------
def sample_ref(l, t, k, p, m, u):
    """token, kept, prob of one row in 64 bits (numpy), and whether a border lies so near that rounding decides."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    idx = np.flatnonzero(l > -np.inf)
    if not len(idx):
        return -1, 0, 0.0
    order = idx[np.argsort(-l[idx], kind="stable")]
    if not t > 0:
        return order[0], 1, 1.0
    x = l[order]
    with np.errstate(invalid="ignore"):
        e = np.where(x == x[0], 1.0, np.exp((x - x[0]) / t))
    cum = np.cumsum(e)
    n = len(e)
    if 0 < p < 1:
        n = min(n, int((cum < p * cum[-1]).sum()) + 1)
    if 0 < k:
        n = min(n, k)
    if m > 0:
        n = min(n, int((e >= min(m, 1.0)).sum()))
    u = 0.0 if not u > 0 else min(u, float(np.float32(1) - np.float32(2.0 ** -24)))
    j = min(int((cum[:n] < u * cum[n - 1]).sum()), n - 1)
    return order[j], n, e[j] / cum[n - 1]


def sample_run(Q, logits, u, t=None, k=None, p=None, m=None):
    n, V = logits.shape
    f = lambda x, d: None if x is None else Dev(torch.tensor(x, dtype=d))  # noqa: E731
    token, kept, prob = i32(n), i32(n), Dev(torch.zeros(n))
    Q.sample_rows(logits if isinstance(logits, Dev) else Dev(logits), f(u, torch.float32), token, Work(Buffer(Q.sample_rows_work(n, V))),
                  temperature=f(t, torch.float32), top_k=f(k, torch.int32), top_p=f(p, torch.float32), min_p=f(m, torch.float32), prob=prob,
                  kept=kept)
    return token.get().tolist(), kept.get().tolist(), prob.get().tolist()


def rows_of(kind, n, V, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, V), generator=g) * 2.0
    if kind == "peaked":
        x[:, torch.randperm(V, generator=g)[:max(1, V // 500)]] += 8.0
    elif kind == "flat":
        x *= 0.01
    elif kind == "ties":
        x = torch.round(x * 2.0) / 2.0
    elif kind == "equal":
        x = torch.full((n, V), -3.25)
    elif kind == "masked":
        x[torch.rand((n, V), generator=g) < 0.9] = float("-inf")
        x[:, V // 2] = float("nan")
        x[:, V // 3] = 1.0
    return x


SETTINGS = [(0.8, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 0.5, 0.02), (1.3, 200, 0.99, 0.05), (0.0, 5, 0.5, 0.1),
            (1.0, 1, 1.0, 0.0), (2.0, 0, 0.999, 0.0), (0.05, 0, 0.9, 0.3), (1.0, 3000, 1.0, 0.001), (1.0, 0, 1.0, 1.0)]


@pytest.mark.parametrize("kind", ["normal", "peaked", "flat", "ties", "equal", "masked"])
@pytest.mark.parametrize("V", [1, 2, 63, 1000, 8191, 32000, 151936])
def test_sample_rows_match_the_definition(Q, kind, V):
    """Every setting on rows of each kind: the definition's token, number kept and probability (to 2^-20 of it: its own
    rounding to 32 bits is 2^-24)."""
    n = len(SETTINGS) * 2
    x = rows_of(kind, n, V, V)
    t, k, p, m = (list(c) for c in zip(*(SETTINGS * 2)))
    r = random.Random(V)
    u = [float(np.float32(r.random())) for _ in range(n)]
    u[0], u[1], u[2] = 0.0, float(np.float32(1) - np.float32(2.0 ** -24)), 0.5
    token, kept, prob = sample_run(Q, x, u, t, k, p, m)
    f = lambda y: float(np.float32(y))  # noqa: E731
    for i in range(n):
        want = sample_ref(x[i].numpy(), f(t[i]), k[i], f(p[i]), f(m[i]), u[i])
        assert (token[i], kept[i]) == want[:2], (i, SETTINGS[i % len(SETTINGS)], u[i])
        assert abs(prob[i] - want[2]) <= 2.0 ** -20 * want[2]


@pytest.mark.parametrize("kind", ["normal", "equal", "ties"])
def test_sample_rows_of_the_largest_vocabulary(Q, kind):
    """2^20 tokens: more slices than a mask has bits, and cells of a million equal tokens."""
    x = rows_of(kind, 3, 1 << 20, 2)
    t, k, p, m = [1.0, 0.7, 1.5], [0, 50, 0], [0.9, 1.0, 1.0], [0.0, 0.0, 0.01]
    u = [float(np.float32(y)) for y in (0.77, 0.2, 0.999)]
    token, kept, _ = sample_run(Q, x, u, t, k, p, m)
    f = lambda y: float(np.float32(y))  # noqa: E731
    for i in range(3):
        assert (token[i], kept[i]) == sample_ref(x[i].numpy(), f(t[i]), k[i], f(p[i]), f(m[i]), u[i])[:2], i


@pytest.mark.parametrize("kind", ["normal", "ties", "equal"])
@pytest.mark.parametrize("V", [300, 8193, 40000])
def test_sample_rows_around_64_kept_tokens(Q, kind, V):
    """As many tokens kept as a wave orders at once, and a few more or fewer, by each of the limits; one cell or many."""
    x1 = rows_of(kind, 1, V, 5)
    if kind == "normal":
        x1[0, ::V // 70] = torch.linspace(9.0, 12.0, len(x1[0, ::V // 70]))
    k = list(range(55, 74)) + [0] * 30
    p = [1.0] * 19 + [0.80 + 0.01 * i for i in range(15)] + [1.0] * 15
    m = [0.0] * 34 + [0.001 * 1.6 ** i for i in range(15)]
    r = random.Random(V)
    u = [float(np.float32(r.random())) for _ in k]
    n = len(k)
    token, kept, prob = sample_run(Q, x1.expand(n, V).contiguous(), u, [1.1] * n, k, p, m)
    f = lambda y: float(np.float32(y))  # noqa: E731
    for i in range(n):
        want = sample_ref(x1[0].numpy(), f(1.1), k[i], f(p[i]), f(m[i]), u[i])
        assert (token[i], kept[i]) == want[:2], (i, k[i], p[i], m[i], u[i])
        assert abs(prob[i] - want[2]) <= 2.0 ** -20 * want[2]


def test_sample_rows_of_enormous_logits(Q):
    """Logits and temperatures whose cells are no numbers of their own: the ends of a cell are searched among all floats."""
    x = torch.full((6, 9000), -1e38)
    x[0, 70:80], x[0, 4000:4100] = 3e38, 2.9e38
    x[1, 5:500] = 1e25
    x[2] = torch.linspace(-3e38, 3e38, 9000)
    x[3, ::3] = 1e-3
    x[4, 10], x[4, 8999] = float("inf"), 3e38
    x[5, 100:200] = -1e30
    t = [1.0, 0.5, 1e38, 1e-38, 1.0, float("inf")]
    k, p, m = [0, 30, 100, 0, 0, 0], [0.55, 1.0, 0.9, 0.3, 0.9, 0.5], [0.0, 0.0, 0.0, 0.5, 0.0, 0.0]
    u = [0.77, 0.41, 0.62, 0.37, 0.5, 0.83]
    f = lambda y: float(np.float32(y))  # noqa: E731
    token, kept, _ = sample_run(Q, x, u, t, k, p, m)
    for i in range(6):
        assert (token[i], kept[i]) == sample_ref(x[i].numpy(), f(t[i]), k[i], f(p[i]), f(m[i]), f(u[i]))[:2], i


@pytest.mark.parametrize("n", [1, 31, 33, 300])
def test_sample_rows_batches_of_one_row(Q, n):
    """Every row of a batch of equal rows gets the same token."""
    x = rows_of("peaked", 1, 70001, 3)
    u = float(np.float32(0.61))
    want = sample_ref(x[0].numpy(), float(np.float32(0.9)), 0, float(np.float32(0.97)), 0.0, u)
    token, kept, _ = sample_run(Q, x.expand(n, -1).contiguous(), [u] * n, [0.9] * n, None, [0.97] * n)
    assert token == [want[0]] * n and kept == [want[1]] * n


def test_sample_rows_settings_out_of_range(Q):
    """NaN and out-of-range settings and numbers count as documented; missing arrays as no limit."""
    nan = float("nan")
    x = rows_of("normal", 12, 5000, 8)
    t = [1.0, nan, -1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1e-30, float("inf"), 1.0]
    k = [0, 5, 5, -7, 2 ** 31 - 1, 0, 0, 0, 0, 0, 0, 5000]
    p = [nan, 0.5, 0.5, -0.5, 0.0, 7.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0]
    m = [nan, 0, 0, -1.0, 0, 0, 9.0, 0, 0, 0, 0, 0]
    u = [0.3, 0.3, 0.3, 0.9, 0.99, 0.7, 0.5, nan, -3.0, 0.5, 0.25, 8.0]
    token, kept, prob = sample_run(Q, x, u, t, k, p, m)
    f = lambda y: float(np.float32(y))  # noqa: E731
    for i in range(12):
        assert (token[i], kept[i]) == sample_ref(x[i].numpy(), f(t[i]), k[i], f(p[i]), f(m[i]), f(u[i]))[:2], i
    token, kept, _ = sample_run(Q, x, u)
    for i in range(12):
        assert (token[i], kept[i]) == sample_ref(x[i].numpy(), 1.0, 0, 1.0, 0.0, f(u[i]))[:2], i


def test_sample_rows_masked_infinite_and_signed_zero_rows(Q):
    inf = float("inf")
    x = torch.full((5, 70000), -inf)
    x[1] = float("nan")
    x[2, [9, 500, 69999]] = inf
    x[2, 5] = 3.0
    x[3, 69999] = -1e30
    x[4, 100:300] = 0.0
    x[4, 100:300:2] = -0.0
    token, kept, prob = sample_run(Q, x, [0.5, 0.5, 0.5, 0.9, 0.5], [1.0] * 5)
    assert token == [-1, -1, 500, 69999, 199] and kept[:2] == [0, 0] and kept[2:] == [4, 1, 200] and prob[:2] == [0.0, 0.0]
    assert prob[3] == 1.0 and abs(prob[2] - 1 / 3) < 1e-7 and abs(prob[4] - 1 / 200) < 1e-9
    token, kept, _ = sample_run(Q, x, [0.5] * 5, [0.0] * 5)
    assert token == [-1, -1, 9, 69999, 100] and kept == [0, 0, 1, 1, 1]


def test_sample_rows_frequencies(Q):
    """Numbers on a regular grid fall on the tokens in proportion to the definition's probabilities, to one grid step each."""
    V, n = 200, 4096
    x = rows_of("normal", 1, V, 1)[0]
    u = [(i + 0.5) / n for i in range(n)]
    token, _, _ = sample_run(Q, x.expand(n, V).contiguous(), u, [0.9] * n)
    w = np.exp(x.double().numpy() / float(np.float32(0.9)))
    assert np.abs(np.bincount(token, minlength=V) / n - w / w.sum()).max() <= 1.0 / n


def test_sample_rows_strided_rows_and_agreement_with_sample_token(Q):
    """Rows inside wider ones; and sample_token's draws from the same numbers (its float sums decide otherwise only next
    to a border: 200 draws of this seed have none there)."""
    g = torch.Generator().manual_seed(12)
    wide = torch.randn((200, 1100), generator=g) * 3.0
    x = wide[:, 7:1007]
    rng, us, want = Q.rng_create(5), [], []
    for i in range(200):
        before = Q.Rng(rng.state)
        us.append(Q.lib().rng_uniform(Q.ctypes_byref(before)))
        want.append(Q.sample_token(np.ascontiguousarray(x[i:i + 1].numpy()), 0.8, 40, 0.95, rng))
    token, _, _ = sample_run(Q, Dev(wide)[:, 7:1007], us, [0.8] * 200, [40] * 200, [0.95] * 200)
    assert token == want


# ---------------------------------------------------------------------------
# Streams, graphs, repeatability, and a run of all four
# ---------------------------------------------------------------------------
HIP = C.CDLL("libamdhip64.so.7")                               # the runtime that is loaded already


def hip(name, *args):
    assert getattr(HIP, name)(*args) == 0, name


class Stream:
    def __init__(self):
        self.p = C.c_void_p()
        hip("hipStreamCreateWithFlags", C.byref(self.p), 1)    # not ordered with the default stream

    def sync(self):
        hip("hipStreamSynchronize", self.p)


class Graph:
    """What calls(stream) enqueues, captured once on a stream of its own."""

    def __init__(self, calls):
        self.stream = Stream()
        assert qlib.load().lib().qllama_device_sync() == 0
        hip("hipStreamBeginCapture", self.stream.p, 0)         # global: nothing unsafe for a capture may be called
        calls(self.stream.p.value)
        graph, self.exec = C.c_void_p(), C.c_void_p()
        hip("hipStreamEndCapture", self.stream.p, C.byref(graph))
        hip("hipGraphInstantiate", C.byref(self.exec), graph, None, None, C.c_size_t(0))

    def launch(self):
        hip("hipGraphLaunch", self.exec, self.stream.p)

    def replay(self):
        self.launch()
        self.stream.sync()


class Server:
    """A few requests of one attention layer, as a server keeps them on the device."""

    def __init__(self, Q, typ="bf16", n=5, H=8, KVH=2, hd=64, page=16, pages=40, width=6, rows=64, seed=0):
        self.Q, self.H, self.KVH, self.n, self.page, self.rows = Q, H, KVH, n, page, rows
        g = torch.Generator().manual_seed(seed)
        self.kv = make_cache(Q, typ, pages, KVH, page, hd, gen=g)
        self.table = Dev(torch.full((n, width), -1, dtype=torch.int32))
        self.ring = Dev(torch.randperm(pages, generator=g).to(torch.int32))
        self.state, self.state_out = dev_i32([0, pages]), i32(2)
        self.cached, self.lens, self.added, self.status, self.starts = i32(n), i32(n), i32(n), i32(n), i32(n + 1)
        self.slots, self.positions, self.requests = i32(rows), i32(rows), i32(rows)
        cos, sin = tables(width * page, hd)
        self.cos, self.sin = Dev(cos), Dev(sin)
        self.qkv, self.q = Dev(torch.zeros((rows, H + 2 * KVH, hd))), Dev(torch.zeros((rows, H, hd)))
        self.q_last, self.o, self.lse = Dev(torch.zeros((n, H, hd))), Dev(torch.zeros((n, H, hd))), Dev(torch.zeros((n, H)))
        self.head = torch.randn((H * hd, 500), generator=g) * 0.2
        self.logits, self.u = Dev(torch.zeros((n, 500))), Dev(torch.zeros(n))
        self.settings = dict(temperature=Dev(torch.full((n,), 0.9)), top_k=dev_i32([50] * n), top_p=Dev(torch.full((n,), 0.9)),
                             min_p=Dev(torch.full((n,), 0.01)))
        self.token, self.kept, self.prob = i32(n), i32(n), Dev(torch.zeros(n))
        self.work, self.work2 = Work(Buffer(Q.paged_attention_work(self.kv, n, H))), Work(Buffer(Q.sample_rows_work(n, 500)))

    def store(self, s=None):
        Q = self.Q
        Q.paged_plan(self.cached, self.added, self.table, self.ring, self.state, self.page, self.lens, self.status, self.starts,
                     self.state_out, self.slots, self.positions, self.requests, stream=s)
        q, k, v = self.qkv.split([self.H, self.KVH, self.KVH], 1)
        Q.paged_append(self.kv, k, v, self.slots, q=q, q_out=self.q, positions=self.positions, cos=self.cos, sin=self.sin, stream=s)

    def answer(self, q, s=None):
        self.Q.paged_attention(self.kv, q, self.table, self.lens, self.o, self.work, lse=self.lse, stream=s)

    def sample(self, s=None):
        self.Q.sample_rows(self.logits, self.u, self.token, self.work2, prob=self.prob, kept=self.kept, stream=s, **self.settings)

    def next(self):
        self.cached.set(self.lens.get())
        self.state.set(self.state_out.get())

    def feed(self, step, added, seed=0):
        g = torch.Generator().manual_seed(1000 * seed + step)
        self.added.set(torch.tensor(added, dtype=torch.int32))
        self.qkv.set(torch.randn(self.qkv.shape, generator=g))
        self.u.set(torch.rand(self.n, generator=g))
        self.logits.set(torch.randn((self.n, 500), generator=g) * 2.0)

    def results(self):
        return [x.get() for x in (self.o, self.lse, self.token, self.prob, self.kept, self.lens, self.state_out, self.slots, self.table, self.q)]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
def test_a_run_of_steps_matches_dense_attention(Q, typ):
    """Ten steps, prompts first, then a token each; request 1 ends at step 4 and another takes its place: the paged result
    against attention over each request's own dense rows, kept beside it in 64 bits."""
    s = Server(Q, typ)
    dense = [[] for _ in range(s.n)]
    for step in range(10):
        added = [20, 7, 1, 0, 3] if step == 0 else [1, -1 if step == 4 else 9 if step == 5 else 1, 1, 30 if step == 2 else int(step > 2), 1]
        s.feed(step, added)
        s.store()
        starts = s.starts.get().tolist()
        assert s.status.get().tolist() == [0] * s.n
        q_rows = s.q.get()
        s.q_last.set(q_rows[[max(x - 1, 0) for x in starts[1:]]])
        s.answer(s.q_last)
        o = s.o.get()
        s.logits.set(o.view(s.n, -1) @ s.head)
        s.sample()
        for r, a in enumerate(added):
            if a < 0:
                dense[r] = []
            for i in range(starts[r], starts[r] + max(a, 0)):
                t = len(dense[r])
                k = rotate32(s.qkv.host[i, s.H:s.H + s.KVH], s.cos.host[t], s.sin.host[t])
                held = []
                for x in (k, s.qkv.host[i, s.H + s.KVH:]):
                    if typ == "i8":
                        c, scale = codes(x)
                        held.append(c.double() * scale.double()[:, None])
                    else:
                        held.append(x.to(DT[typ]).double())
                dense[r].append(held)
        assert s.lens.get().tolist() == [len(d) for d in dense]
        for r, d in enumerate(dense):
            if not d:
                assert bool((o[r] == 0).all())
                continue
            k, v = torch.stack([x[0] for x in d]), torch.stack([x[1] for x in d])
            q = s.q_last.host[r].double().view(s.KVH, -1, q_rows.shape[2])
            w = torch.softmax((k.transpose(0, 1)[:, None] * q[:, :, None]).sum(-1) / 8.0, -1)
            want = (w[..., None] * v.transpose(0, 1)[:, None]).sum(2).view(s.H, -1)
            # weights of scores that are off by 200 EPS sum |q k| / 8 at most (64 products in three parts), 64 dims of N(0, 1)
            assert (o[r].double() - want).abs().max() <= 1e-4
        x, u = s.logits.host.numpy(), s.u.host.tolist()
        token, kept = s.token.get().tolist(), s.kept.get().tolist()
        for r in range(s.n):
            want = sample_ref(x[r], float(np.float32(0.9)), 50, float(np.float32(0.9)), float(np.float32(0.01)), u[r])
            assert (token[r], kept[r]) == want[:2]
        s.next()


def one_step(s, stream=None):
    """A decode step of every request: row r of the step is request r's."""
    s.store(stream)
    s.answer(s.q[:s.n], stream)
    s.sample(stream)


def test_graph_replays_equal_eager_steps(Q):
    """The four calls captured once and replayed over changing inputs, with eager work and synchronizations between, beside a
    second server that makes the same steps eagerly; two graphs with workspaces of their own replayed side by side."""
    a, b, c, d = Server(Q, seed=1), Server(Q, seed=1), Server(Q, seed=2), Server(Q, seed=2)
    for s in (a, b, c, d):
        s.feed(0, [20, 7, 1, 12, 3], seed=1 if s in (a, b) else 2)
        s.store()
        s.next()
    graphs = [Graph(lambda stream, s=s: one_step(s, stream)) for s in (a, c)]
    for step in range(1, 9):
        for s in (a, b, c, d):
            s.feed(step, [1] * 5, seed=1 if s in (a, b) else 2)
        for g in graphs:
            g.launch()
        for g in graphs:
            g.stream.sync()
        one_step(b)
        one_step(d)
        for x, y in zip(a.results() + c.results(), b.results() + d.results()):
            assert torch.equal(x, y), step
        for s in (a, b, c, d):
            s.next()


def test_calls_on_other_streams(Q):
    """The library's stream, the default stream and another give the same bits."""
    results = []
    for stream in (None, 0, Stream()):
        s = Server(Q, seed=3)
        s.feed(0, [1] * 5)
        one_step(s, stream.p.value if isinstance(stream, Stream) else stream)
        assert Q.lib().qllama_device_sync() == 0
        results.append(s.results())
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))


def test_host_memory_is_refused(Q, capfd):
    """Addresses that are no device memory are an error of the call, not of the GPU."""
    s = Server(Q)
    host = np.zeros(1 << 16, np.uint8)
    L, at = Q.lib(), host.ctypes.data + 64
    assert L.qllama_sample_rows(Q.SAMPLE_ROWS.pack(1, 10, 10, at, at, 0, 0, 0, 0, at, 0, 0, at & ~15, 1 << 15), None) != 0
    assert "not device memory" in capfd.readouterr().err
    one_step(s)                                                # and the library stays usable
    assert s.status.get().tolist() == [0] * 5


def test_equal_inputs_give_equal_bits(Q):
    g = torch.Generator().manual_seed(1)
    kv = make_cache(Q, "f16", 300, 2, 16, 128, gen=g)
    lens = [1500, 700, 33, 2000]
    q = torch.randn((4, 8, 128), generator=g)
    table = pages_for(lens, 16, 126, 300, 1)
    x = Dev(rows_of("ties", 16, 50000, 3))
    first = None
    for _ in range(5):
        got = attend(Q, kv, q, table, lens) + tuple(torch.tensor(y) for y in sample_run(Q, x, [0.37] * 16, [1.1] * 16, None, [0.97] * 16))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
