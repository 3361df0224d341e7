"""The serving operators (include/qserve.h) on the GPU against plain definitions in whole numbers and 64 bits: pages and
slots, rows into pages, attention of one token over pages, sampled rows, and a run of all four as a server makes it."""
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
    return q


def stream():
    return torch.cuda.current_stream().cuda_stream


def i32(*shape):
    return torch.empty(shape, dtype=torch.int32, device="cuda")


def cuda_i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


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
    o = dict(table=cuda_i32(table), ring=cuda_i32(ring), lens=i32(n), status=i32(n), starts=i32(n + 1), state=i32(2), slots=i32(max_rows),
             positions=i32(max_rows), requests=i32(max_rows))
    Q.paged_plan(cuda_i32(cached), cuda_i32(added), o["table"], o["ring"], cuda_i32(state), page, o["lens"], o["status"], o["starts"],
                 o["state"], o["slots"], o["positions"], o["requests"], stream=stream())
    return {k: v.cpu().numpy() for k, v in o.items()}


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
    slots = torch.full((12,), 99, dtype=torch.int32, device="cuda")
    ring, state, out, starts = cuda_i32([5, 6]), cuda_i32([1, 2]), i32(2), i32(1)
    e = i32(0)
    Q.paged_plan(e, e, i32(0, 3), ring, state, 16, e, e, starts, out, slots[4:8], slots[8:12].clone(), slots[:4].clone(), stream=stream())
    assert out.tolist() == [1, 2] and starts.tolist() == [0] and slots.tolist() == [99] * 4 + [-1] * 4 + [99] * 4


def test_plan_a_request_that_needs_no_page_is_not_held_up(Q):
    args = ([16, 3, 16], [1, 1, 1], np.array([[0, -1], [1, -1], [2, -1]]), np.array([9, 9]), [0, 0], 16, 3)
    got = plan_run(Q, *args)
    assert got["status"].tolist() == [3, 0, 3] and got["slots"].tolist() == [1 * 16 + 3, -1, -1] and got["lens"].tolist() == [16, 4, 16]


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
def make_cache(Q, typ, pages, KVH, page, hd, order="head", gen=None, fill=None):
    """A cache of random contents and its view; order "slot": heads beside each other within a slot."""
    shape = (pages, KVH, page, hd) if order == "head" else (pages, page, KVH, hd)
    t = []
    for _ in range(2):
        x = torch.randn(shape, generator=gen, device="cuda") if fill is None else torch.full(shape, fill, device="cuda")
        x = torch.randint(-127, 128, shape, generator=gen, device="cuda").to(torch.int8) if typ == "i8" else x.to(DT[typ])
        t.append(x if order == "head" else x.transpose(1, 2))
    s = [None, None]
    if typ == "i8":
        sh = shape[:3]
        s = [0.005 + 0.03 * torch.rand(sh, generator=gen, device="cuda") for _ in range(2)]
        s = s if order == "head" else [x.transpose(1, 2) for x in s]
    return Q.PagedKV(t[0], t[1], s[0], s[1])


def tables(n, hd):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
    return a.cos().float().cuda(), a.sin().float().cuda()


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
    g = torch.Generator(device="cuda").manual_seed(hd + rows)
    pages = -(-rows // page) + 2
    kv = make_cache(Q, typ, pages, KVH, page, hd, order, g)
    before = [x.clone() for x in (kv.k, kv.v)]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows].to(torch.int32)
    if rows > 3:
        slots[-2:] = -1                                        # padding
        slots[0] = -2 ** 31
    pos = torch.randint(0, 50, (rows,), generator=g, device="cuda", dtype=torch.int32)
    cos, sin = tables(50, hd)
    qkv = torch.randn((rows, H + 2 * KVH, hd), generator=g, device="cuda")
    qkv[0, H] = 0.0                                            # a key of zeros
    q, k, v = qkv.split([H, KVH, KVH], 1)
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    q_out = torch.full((rows + 1, H, hd), 7.0, device="cuda")
    bad = cuda_i32([5])
    Q.paged_append(kv, k, v, slots, q=q, q_out=q_out[:rows], positions=pos, cos=cos, sin=sin, bad=bad, stream=stream())
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    assert torch.equal(q_out[:rows], rotate32(q, c, s)) and torch.equal(q_out[rows], torch.full_like(q_out[rows], 7.0))
    assert bad.item() == 5
    held = (slots >= 0).nonzero()[:, 0]
    at = slots[held].long()
    for got, was, sc, x in ((kv.k, before[0], kv.k_scale, rotate32(k, c, s)), (kv.v, before[1], kv.v_scale, v)):
        want = was
        x = x[held]
        if typ == "i8":
            x, scale = codes(x)
            assert torch.equal(sc[at // page, :, at % page], scale)
        want[at // page, :, at % page] = x.to(want.dtype)
        assert torch.equal(got, want)


def test_append_rows_out_of_range_and_unaligned(Q):
    """Positions outside the tables: nothing of the row is written; slots outside the cache: no key and value.  Rows and
    tables on odd addresses give the same values."""
    g = torch.Generator(device="cuda").manual_seed(3)
    H, KVH, hd, page, rows = 4, 2, 64, 16, 6
    kv = make_cache(Q, "f32", 2, KVH, page, hd, gen=g)
    was = kv.k.clone()
    raw = torch.randn(rows * (H + 2 * KVH) * hd + 1, generator=g, device="cuda")[1:]
    qkv = raw.view(rows, H + 2 * KVH, hd)
    q, k, v = qkv.split([H, KVH, KVH], 1)
    cos, sin = tables(9, hd)
    slots, pos = cuda_i32([0, 32, 5, 2 ** 31 - 1, 7, -1]), cuda_i32([8, 1, 9, 2, -1, 3])
    q_out, bad = torch.full((rows, H, hd), 7.0, device="cuda"), cuda_i32([0])
    Q.paged_append(kv, k, v, slots, q=q, q_out=q_out, positions=pos, cos=cos, sin=sin, bad=bad, stream=stream())
    assert bad.item() == 4
    ok = torch.tensor([0, 1, 3, 5], device="cuda")
    p = pos[ok].long()
    assert torch.equal(q_out[ok], rotate32(q[ok], cos[p][:, None], sin[p][:, None])) and bool((q_out[[2, 4]] == 7.0).all())
    was[0, :, 0] = rotate32(k[0], cos[8], sin[8])
    assert torch.equal(kv.k, was)


def test_append_without_queries_or_rotation_and_in_place(Q):
    kv = make_cache(Q, "bf16", 3, 2, 8, 64)
    k, v = torch.randn(4, 2, 64, device="cuda"), torch.randn(4, 2, 64, device="cuda")
    k[0, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.00390625], device="cuda")    # a tie rounds to even
    slots = cuda_i32([23, 0, 9, 16])
    Q.paged_append(kv, k, v, slots, stream=stream())
    at = slots.long()
    assert torch.equal(kv.k[at // 8, :, at % 8].isnan(), k.isnan())
    assert torch.equal(kv.k[at // 8, :, at % 8].nan_to_num(1.0), k.bfloat16().nan_to_num(1.0)) and torch.equal(kv.v[at // 8, :, at % 8], v.bfloat16())
    q = torch.randn(4, 6, 64, device="cuda")
    cos, sin = tables(5, 64)
    pos = cuda_i32([4, 0, 2, 2])
    want = rotate32(q, cos[pos.long()][:, None], sin[pos.long()][:, None])
    Q.paged_append(kv, k, v, slots, q=q, q_out=q, positions=pos, cos=cos, sin=sin, stream=stream())
    assert torch.equal(q, want)


def test_append_int8_codes_of_nan_and_infinity(Q):
    """A NaN gets code 0 and does not count for the scale; the finite elements keep theirs."""
    kv = make_cache(Q, "i8", 1, 1, 4, 16)
    k = torch.linspace(-1, 1, 16, device="cuda").view(1, 1, 16).clone()
    k[0, 0, 3] = float("nan")
    Q.paged_append(kv, k, k, cuda_i32([2]), stream=stream())
    want, scale = codes(k.nan_to_num(0.0))
    assert torch.equal(kv.k[0, 0, 2], want[0, 0]) and kv.k_scale[0, 0, 2].item() == scale.item()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def attend_ref(kv, q, table, lens, scale=None):
    """o, lse, and a bound of what 32-bit arithmetic may differ from them, all in 64 bits.

    A score is a sum of 3 hd products at most (three parts of a query), so it is off by (3 hd + 4) EPS sum |q k| scale;
    a weight by that of its score and of the maximum, the exponential's argument (2 EPS |score| each) and the exponential
    (4 EPS); the sums over len tokens, in parts of three, by (3 len + 16) EPS of sum w |v|."""
    n, H, hd = q.shape
    KVH, page = kv.k.shape[1], kv.k.shape[2]
    G = H // KVH
    scale = scale or 1.0 / math.sqrt(hd)
    o, lse, bound, lse_bound = (torch.zeros(s, dtype=torch.float64) for s in ((n, H, hd), (n, H), (n, H, hd), (n, H)))
    lse.fill_(-math.inf)
    k_all, v_all = kv.k.double().cpu(), kv.v.double().cpu()
    if kv.k_scale is not None:
        k_all, v_all = k_all * kv.k_scale.double().cpu()[..., None], v_all * kv.v_scale.double().cpu()[..., None]
    q, table = q.double().cpu(), table.cpu()
    for r, length in enumerate(lens.tolist()):
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
    return cuda_i32(table)


def attend(Q, kv, q, table, lens, **kw):
    n, H, _ = q.shape
    o, lse = torch.full(q.shape, 7.0, device="cuda"), torch.full((n, H), 7.0, device="cuda")
    work = torch.empty(Q.paged_attention_work(kv, n, H), dtype=torch.uint8, device="cuda")
    Q.paged_attention(kv, q, table, lens, o, work, lse=lse, stream=stream(), **kw)
    return o, lse


def check(Q, kv, q, table, lens, **kw):
    o, lse = attend(Q, kv, q, table, lens, **kw)
    wo, wl, bound, lb = attend_ref(kv, q, table, lens, kw.get("scale"))
    o, lse = o.double().cpu(), lse.double().cpu()
    assert bool(((o - wo).abs() <= bound).all()), ((o - wo).abs() - bound).max()
    empty = torch.isinf(wl)
    assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all()) and bool((o[empty] == 0).all())
    assert bool(((lse - wl).abs()[~empty] <= lb[~empty]).all())


SHAPES = [(6, 2, 48), (32, 8, 64), (8, 2, 128), (4, 4, 128), (5, 1, 8), (20, 1, 72), (33, 1, 256), (16, 1, 160)]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("H,KVH,hd", SHAPES)
@pytest.mark.parametrize("page,order", [(16, "head"), (5, "slot"), (48, "slot"), (1, "head")])
def test_attention_matches_the_definition(Q, typ, H, KVH, hd, page, order):
    """Lengths of none, one, at and around the steps of 16 and 32 keys and the pages, in one ragged batch."""
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 65, 100, 257, -4]
    g = torch.Generator(device="cuda").manual_seed(H + hd)
    need = sum(-(-max(x, 0) // page) for x in lens)
    kv = make_cache(Q, typ, need + 3, KVH, page, hd, order, g)
    q = torch.randn((len(lens), H, hd), generator=g, device="cuda") * 2.0
    check(Q, kv, q, pages_for(lens, page, -(-257 // page) + 1, need + 3, hd), cuda_i32(lens))


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("lens,page", [([5000], 16), ([4097, 3], 64), ([1, 6001, 40], 24), ([300] * 70, 16), ([900, 0, 31, 1700] * 9, 128)])
def test_attention_split_and_joined(Q, typ, lens, page):
    """Long and many requests: shares that end inside a tile, begin in another's, and hold several."""
    g = torch.Generator(device="cuda").manual_seed(len(lens))
    need = sum(-(-x // page) for x in lens)
    kv = make_cache(Q, typ, need + 1, 2, page, 64, "head", g)
    q = torch.randn((len(lens), 6, 64), generator=g, device="cuda")
    check(Q, kv, q, pages_for(lens, page, max(-(-x // page) for x in lens), need + 1, 1), cuda_i32(lens))


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("page", [1, 7, 16, 48])
def test_attention_reads_the_row_that_the_table_names(Q, typ, page):
    """One key stands out by more than a float's range of weights: the output is its value row, as held, and moves with it."""
    KVH, G, hd, n = 2, 3, 64, 9
    g = torch.Generator(device="cuda").manual_seed(page)
    lens = [1, 20, 33, 64, 100, 129, 200, 511, 700]
    need = sum(-(-x // page) for x in lens)
    kv = make_cache(Q, typ, need, KVH, page, hd, "head", g)
    kv.k.zero_()
    table = pages_for(lens, page, -(-700 // page), need, 5)
    r = random.Random(page)
    at = [r.randrange(x) for x in lens]
    for i, t in enumerate(at):
        kv.k[int(table[i, t // page]), :, t % page, 5] = 100
    if typ == "i8":
        kv.k_scale.fill_(1.0)
        kv.v_scale.fill_(0.25)
    q = torch.zeros((n, KVH * G, hd), device="cuda")
    q[:, :, 5] = 64.0                                        # a score of 800 against 0
    o, _ = attend(Q, kv, q, table, cuda_i32(lens))
    for i, t in enumerate(at):
        v = kv.v[int(table[i, t // page]), :, t % page].float() * (0.25 if typ == "i8" else 1.0)
        assert torch.equal(o[i], v.repeat_interleave(G, 0)), (i, t)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_leaves_out_what_is_no_token(Q, typ, page):
    """Slots behind the tokens hold NaN and infinities, pages lie outside the cache, lengths exceed the table: none counts."""
    KVH, hd = 2, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    lens = [3, 40, 77, 10 ** 9, 2 ** 31 - 1, 50]
    width = 16
    held = [min(x, width * page) for x in lens]
    need = sum(-(-x // page) for x in held)
    kv = make_cache(Q, typ, need + 2, KVH, page, hd, "head", g)
    table = pages_for(held, page, width, need, 3)
    table[2, 1] = -1
    table[3, 0] = need + 2
    table[5] = -2 ** 31
    used = torch.zeros((need + 2, page), dtype=torch.bool, device="cuda")
    for i, x in enumerate(held):
        for t in range(x):
            p = int(table[i, t // page])
            if 0 <= p < need + 2:
                used[p, t % page] = True
    stale = ~used[:, None, :, None].expand(kv.k.shape)
    if typ == "i8":
        kv.k_scale[~used[:, None, :].expand(kv.k_scale.shape)] = float("nan")
        kv.v_scale[~used[:, None, :].expand(kv.v_scale.shape)] = float("inf")
    else:
        kv.k[stale] = float("nan")
        kv.v[stale] = float("inf")
    q = torch.randn((len(lens), 4, hd), generator=g, device="cuda")
    o, lse = attend(Q, kv, q, table, cuda_i32(lens))
    if typ == "i8":
        kv.k_scale.nan_to_num_(0.0)
        kv.v_scale.nan_to_num_(0.0, posinf=0.0)
    else:
        kv.k[stale] = 0.0
        kv.v[stale] = 0.0
    o2, lse2 = attend(Q, kv, q, table, cuda_i32(lens))
    assert bool(torch.isfinite(o).all()) and torch.equal(o, o2) and torch.equal(lse, lse2)
    assert bool((o[5] == 0).all()) and bool(torch.isinf(lse[5]).all())
    check(Q, kv, q, table, cuda_i32(lens))


def test_attention_large_scores_and_nan(Q):
    """Scores of thousands and queries of f16's border; a NaN query spoils its own head only."""
    for typ in ("f32", "f16", "bf16", "i8"):
        g = torch.Generator(device="cuda").manual_seed(4)
        kv = make_cache(Q, typ, 8, 2, 16, 64, "head", g)
        q = torch.randn((2, 4, 64), generator=g, device="cuda")
        q[0] *= 3000.0
        q[1] *= 1e-6
        lens = cuda_i32([60, 33])
        table = pages_for([60, 33], 16, 4, 8, 2)
        check(Q, kv, q, table, lens)
        o, _ = attend(Q, kv, q, table, lens)
        q[0, 1, 7] = float("nan")
        o2, _ = attend(Q, kv, q, table, lens)
        assert bool(o2[0, 1].isnan().all())
        assert torch.equal(o2[0, [0, 2, 3]], o[0, [0, 2, 3]]) and torch.equal(o2[1], o[1])


@pytest.mark.parametrize("typ", ["f32", "i8"])
def test_attention_many_requests_most_of_them_empty(Q, typ):
    """700 requests, runs of empty ones among them longer than what a wave looks at at once, the last ones empty too."""
    g = torch.Generator(device="cuda").manual_seed(11)
    r = random.Random(5)
    lens = [r.choice([1, 17, 90]) if r.random() < 0.1 and not 200 < i < 420 and i < 690 else 0 for i in range(700)]
    need = sum(-(-x // 16) for x in lens)
    kv = make_cache(Q, typ, need, 2, 16, 64, "head", g)
    q = torch.randn((700, 2, 64), generator=g, device="cuda")
    check(Q, kv, q, pages_for(lens, 16, 6, need, 1), cuda_i32(lens))
    o, lse = attend(Q, kv, q, pages_for([0] * 700, 16, 6, need, 1), cuda_i32([0] * 700))
    assert bool((o == 0).all()) and bool(torch.isinf(lse).all())


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
def test_attention_shared_pages_and_equal_requests(Q, typ):
    """Requests that share a prefix's pages, and the same request twice: equal bits where equal work is asked of equal places
    in a share, and the definition's values anyway."""
    g = torch.Generator(device="cuda").manual_seed(14)
    kv = make_cache(Q, typ, 12, 2, 32, 128, "head", g)
    table = cuda_i32([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 2, 3], [7, 7, 7, 7]])
    q = torch.randn((4, 4, 128), generator=g, device="cuda")
    q[2] = q[0]
    check(Q, kv, q, table, cuda_i32([128, 100, 128, 97]))


def test_attention_16_heads_a_group_of_256_in_a_graph(Q):
    """The largest queries in LDS (set as the launch's own size) under capture."""
    g = torch.Generator(device="cuda").manual_seed(15)
    kv = make_cache(Q, "bf16", 30, 1, 16, 256, "head", g)
    lens = [300, 77]
    table = pages_for(lens, 16, 19, 30, 1)
    q, n = torch.randn((2, 16, 256), generator=g, device="cuda"), cuda_i32(lens)
    want = attend(Q, kv, q, table, n)
    o, lse = torch.zeros_like(q), torch.zeros((2, 16), device="cuda")
    work = torch.empty(Q.paged_attention_work(kv, 2, 16), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Q.paged_attention(kv, q, table, n, o, work, lse=lse, stream=stream())
    for _ in range(3):
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_attention_scale_strides_and_sentinels(Q):
    """A given scale; queries inside packed rows, outputs with room behind every row, a table inside a larger one."""
    g = torch.Generator(device="cuda").manual_seed(2)
    H, KVH, hd, n = 6, 3, 40, 5
    lens = [50, 1, 0, 33, 64]
    kv = make_cache(Q, "bf16", 20, KVH, 16, hd, "slot", g)
    qkv = torch.randn((n, H + 2 * KVH, hd), generator=g, device="cuda")
    q = qkv[:, :H]
    big = torch.full((n, 9), -1, dtype=torch.int32, device="cuda")
    big[:, :4] = pages_for(lens, 16, 4, 20, 8)
    table = big[:, :4]
    o_all, lse_all = torch.full((n, H + 2, hd), 7.0, device="cuda"), torch.full((n, H + 1), 7.0, device="cuda")
    work = torch.empty(Q.paged_attention_work(kv, n, H), dtype=torch.uint8, device="cuda")
    Q.paged_attention(kv, q, table, cuda_i32(lens), o_all[:, :H], work, lse=lse_all[:, :H], scale=0.3, stream=stream())
    o, lse = attend(Q, kv, q.contiguous(), table.contiguous(), cuda_i32(lens), scale=0.3)
    assert torch.equal(o_all[:, :H], o) and torch.equal(lse_all[:, :H], lse)
    assert bool((o_all[:, H:] == 7.0).all()) and bool((lse_all[:, H:] == 7.0).all())
    check(Q, kv, q.contiguous(), table.contiguous(), cuda_i32(lens), scale=0.3)


def test_attention_pages_behind_two_billion_elements(Q):
    """Pages whose offsets pass 32 bits, in elements and in bytes."""
    pages, KVH, page, hd = 2200, 8, 128, 128                     # 288 M elements a 275 pages: 2.3 G in all
    k = torch.empty((pages, KVH, page, hd), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    ids = [2199, 0, 2047, 1025, 2198]
    g = torch.Generator(device="cuda").manual_seed(6)
    for p in ids:
        k[p] = torch.randn((KVH, page, hd), generator=g, device="cuda").bfloat16()
        v[p] = torch.randn((KVH, page, hd), generator=g, device="cuda").bfloat16()
    kv = Q.PagedKV(k, v)
    q = torch.randn((1, 8, hd), generator=g, device="cuda")
    o, lse = attend(Q, kv, q, cuda_i32([ids]), cuda_i32([600]))
    small = Q.PagedKV(k[ids].contiguous(), v[ids].contiguous())
    o2, lse2 = attend(Q, small, q, cuda_i32([[0, 1, 2, 3, 4]]), cuda_i32([600]))
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    rows = torch.randn((1, KVH, hd), generator=g, device="cuda")
    Q.paged_append(kv, rows, rows, cuda_i32([2199 * page + 127]), stream=stream())
    assert torch.equal(k[2199, :, 127], rows[0].bfloat16()) and torch.equal(v[2199, :, 127], rows[0].bfloat16())


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
    f = lambda x, d: None if x is None else torch.tensor(x, dtype=d, device="cuda")  # noqa: E731
    token, kept, prob = i32(n), i32(n), torch.empty(n, device="cuda")
    work = torch.empty(Q.sample_rows_work(n, V), dtype=torch.uint8, device="cuda")
    Q.sample_rows(logits, f(u, torch.float32), token, work, temperature=f(t, torch.float32), top_k=f(k, torch.int32), top_p=f(p, torch.float32),
                  min_p=f(m, torch.float32), prob=prob, kept=kept, stream=stream())
    return token.tolist(), kept.tolist(), prob.tolist()


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
    token, kept, prob = sample_run(Q, x.cuda(), u, t, k, p, m)
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
    token, kept, _ = sample_run(Q, x.cuda(), u, t, k, p, m)
    f = lambda y: float(np.float32(y))  # noqa: E731
    for i in range(3):
        assert (token[i], kept[i]) == sample_ref(x[i].numpy(), f(t[i]), k[i], f(p[i]), f(m[i]), u[i])[:2], i


@pytest.mark.parametrize("n", [1, 31, 33, 300])
def test_sample_rows_batches_around_the_slice_rule(Q, n):
    """Numbers of rows that take slices of either length give the same tokens for the same row."""
    x = rows_of("peaked", 1, 70001, 3)
    u = float(np.float32(0.61))
    want = sample_ref(x[0].numpy(), float(np.float32(0.9)), 0, float(np.float32(0.97)), 0.0, u)
    token, kept, _ = sample_run(Q, x.expand(n, -1).contiguous().cuda(), [u] * n, [0.9] * n, None, [0.97] * n)
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
    token, kept, prob = sample_run(Q, x.cuda(), u, t, k, p, m)
    f = lambda y: float(np.float32(y))  # noqa: E731
    for i in range(12):
        assert (token[i], kept[i]) == sample_ref(x[i].numpy(), f(t[i]), k[i], f(p[i]), f(m[i]), f(u[i]))[:2], i
    token, kept, _ = sample_run(Q, x.cuda(), u)
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
    token, kept, prob = sample_run(Q, x.cuda(), [0.5, 0.5, 0.5, 0.9, 0.5], [1.0] * 5)
    assert token == [-1, -1, 500, 69999, 199] and kept[:2] == [0, 0] and kept[2:] == [4, 1, 200] and prob[:2] == [0.0, 0.0]
    assert prob[3] == 1.0 and abs(prob[2] - 1 / 3) < 1e-7 and abs(prob[4] - 1 / 200) < 1e-9
    token, kept, _ = sample_run(Q, x.cuda(), [0.5] * 5, [0.0] * 5)
    assert token == [-1, -1, 9, 69999, 100] and kept == [0, 0, 1, 1, 1]


def test_sample_rows_frequencies(Q):
    """Numbers on a regular grid fall on the tokens in proportion to the definition's probabilities, to one grid step each."""
    V, n = 200, 4096
    x = rows_of("normal", 1, V, 1)[0]
    u = [(i + 0.5) / n for i in range(n)]
    token, _, _ = sample_run(Q, x.expand(n, V).contiguous().cuda(), u, [0.9] * n)
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
    token, _, _ = sample_run(Q, wide.cuda()[:, 7:1007], us, [0.8] * 200, [40] * 200, [0.95] * 200)
    assert token == want


# ---------------------------------------------------------------------------
# Streams, graphs, repeatability, and a run of all four
# ---------------------------------------------------------------------------
class Server:
    """A few requests of one attention layer, as a server keeps them on the device."""

    def __init__(self, Q, typ="bf16", n=5, H=8, KVH=2, hd=64, page=16, pages=40, width=6, rows=64, seed=0):
        self.Q, self.H, self.page, self.rows = Q, H, page, rows
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.kv = make_cache(Q, typ, pages, KVH, page, hd, gen=g)
        self.table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
        self.ring = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.state = [cuda_i32([0, pages]), i32(2)]
        self.lens = [torch.zeros(n, dtype=torch.int32, device="cuda"), i32(n)]
        self.added, self.status, self.starts = cuda_i32([0] * n), i32(n), i32(n + 1)
        self.slots, self.positions, self.requests = i32(rows), i32(rows), i32(rows)
        self.cos, self.sin = tables(width * page, hd)
        self.qkv = torch.zeros((rows, H + 2 * KVH, hd), device="cuda")
        self.q = torch.zeros((rows, H, hd), device="cuda")
        self.q_last, self.o, self.lse = torch.zeros((n, H, hd), device="cuda"), torch.zeros((n, H, hd), device="cuda"), torch.zeros((n, H), device="cuda")
        self.head = torch.randn((H * hd, 500), generator=g, device="cuda") * 0.2
        self.logits, self.u = torch.zeros((n, 500), device="cuda"), torch.zeros(n, device="cuda")
        self.settings = dict(temperature=torch.full((n,), 0.9, device="cuda"), top_k=cuda_i32([50] * n), top_p=torch.full((n,), 0.9, device="cuda"),
                             min_p=torch.full((n,), 0.01, device="cuda"))
        self.token, self.kept, self.prob = i32(n), i32(n), torch.zeros(n, device="cuda")
        self.work = torch.zeros(Q.paged_attention_work(self.kv, n, H), dtype=torch.uint8, device="cuda")
        self.work2 = torch.zeros(Q.sample_rows_work(n, 500), dtype=torch.uint8, device="cuda")
        self.KVH, self.n = KVH, n

    def step(self):
        Q, s = self.Q, stream()
        Q.paged_plan(self.lens[0], self.added, self.table, self.ring, self.state[0], self.page, self.lens[1], self.status, self.starts,
                     self.state[1], self.slots, self.positions, self.requests, stream=s)
        q, k, v = self.qkv.split([self.H, self.KVH, self.KVH], 1)
        Q.paged_append(self.kv, k, v, self.slots, q=q, q_out=self.q, positions=self.positions, cos=self.cos, sin=self.sin, stream=s)
        last = (self.starts[1:] - 1).clamp(min=0).long()
        self.q_last.copy_(self.q[last])
        Q.paged_attention(self.kv, self.q_last, self.table, self.lens[1], self.o, self.work, lse=self.lse, stream=s)
        torch.matmul(self.o.view(self.n, -1), self.head, out=self.logits)
        Q.sample_rows(self.logits, self.u, self.token, self.work2, prob=self.prob, kept=self.kept, stream=s, **self.settings)
        self.lens[0].copy_(self.lens[1])
        self.state[0].copy_(self.state[1])

    def feed(self, step, seed=0):
        """Inputs of a step: prompts first, then a token each; request 1 ends at step 4 and another takes its place."""
        g = torch.Generator(device="cuda").manual_seed(1000 * seed + step)
        added = [20, 7, 1, 0, 3] if step == 0 else [1, -1 if step == 4 else 9 if step == 5 else 1, 1, 30 if step == 2 else int(step > 2), 1]
        self.added.copy_(cuda_i32(added[:self.n]))
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g, device="cuda"))
        self.u.copy_(torch.rand(self.n, generator=g, device="cuda"))
        return added

    def results(self):
        return [x.clone() for x in (self.o, self.lse, self.token, self.prob, self.kept, self.lens[1], self.state[1], self.slots)]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
def test_a_run_of_steps_matches_dense_attention(Q, typ):
    """Ten steps: the paged result against attention over each request's own dense rows, kept beside it in 64 bits."""
    s = Server(Q, typ)
    dense = [[] for _ in range(s.n)]
    for step in range(10):
        added = s.feed(step)
        s.step()
        starts = s.starts.tolist()
        assert s.status.tolist() == [0] * s.n
        for r, a in enumerate(added):
            if a < 0:
                dense[r] = []
            for i in range(starts[r], starts[r] + max(a, 0)):
                t = len(dense[r])
                k = rotate32(s.qkv[i, s.H:s.H + s.KVH], s.cos[t], s.sin[t])
                v = s.qkv[i, s.H + s.KVH:]
                held = []
                for x in (k, v):
                    if typ == "i8":
                        c, scale = codes(x)
                        held.append(c.double() * scale.double()[:, None])
                    else:
                        held.append(x.to(DT[typ]).double())
                dense[r].append(held)
        assert s.lens[1].tolist() == [len(d) for d in dense]
        for r, d in enumerate(dense):
            if not d:
                assert bool((s.o[r] == 0).all())
                continue
            k, v = torch.stack([x[0] for x in d]), torch.stack([x[1] for x in d])
            q = s.q_last[r].double().view(s.KVH, -1, s.q.shape[2])
            w = torch.softmax((k.transpose(0, 1)[:, None] * q[:, :, None]).sum(-1) / 8.0, -1)
            want = (w[..., None] * v.transpose(0, 1)[:, None]).sum(2).view(s.H, -1)
            # weights of scores that are off by 200 EPS sum |q k| / 8 at most (64 products in three parts), 64 dims of N(0, 1)
            assert (s.o[r].double() - want).abs().max() <= 1e-4
        x = s.logits.cpu().numpy()
        for r in range(s.n):
            want = sample_ref(x[r], float(np.float32(0.9)), 50, float(np.float32(0.9)), float(np.float32(0.01)), s.u[r].item())
            assert (s.token[r].item(), s.kept[r].item()) == want[:2]


def test_graph_replays_equal_eager_steps(Q):
    """The four calls captured once and replayed over changing inputs, with eager work and synchronizations between, beside a
    second server that makes the same steps eagerly; two graphs with workspaces of their own replayed side by side."""
    a, b, c = Server(Q, seed=1), Server(Q, seed=1), Server(Q, seed=2)
    d = Server(Q, seed=2)
    for s in (a, b, c, d):                                     # every kernel has run before a capture
        s.feed(0)
        s.step()
    side = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for s in (a, c):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.step()
        graphs.append(g)
    for step in range(1, 8):
        for s in (a, b, c, d):
            s.feed(step, seed=1 if s in (a, b) else 2)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        b.step()
        d.step()
        torch.cuda.synchronize()
        for x, y in zip(a.results() + c.results(), b.results() + d.results()):
            assert torch.equal(x, y), step


def test_calls_on_another_stream_and_on_the_librarys(Q):
    """Work ordered on a stream that is not the current one, and on qllama_stream()."""
    s = Server(Q, seed=3)
    s.feed(0)
    s.step()
    want = s.results()
    for other in (torch.cuda.Stream(), torch.cuda.ExternalStream(Q.lib().qllama_stream() or _library_stream(Q))):
        t = Server(Q, seed=3)
        t.feed(0)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            t.step()
        other.synchronize()
        for x, y in zip(t.results(), want):
            assert torch.equal(x, y)


def _library_stream(Q):
    Q.sample_argmax(np.zeros((1, 4), np.float32))              # the library's first GPU call makes its stream
    return Q.lib().qllama_stream()


def test_equal_inputs_give_equal_bits(Q):
    kv = make_cache(Q, "f16", 300, 2, 16, 128, gen=torch.Generator(device="cuda").manual_seed(1))
    lens = [1500, 700, 33, 2000]
    q = torch.randn((4, 8, 128), device="cuda")
    table = pages_for(lens, 16, 126, 300, 1)
    x = rows_of("ties", 16, 50000, 3).cuda()
    first = None
    for _ in range(5):
        got = attend(Q, kv, q, table, cuda_i32(lens)) + tuple(torch.tensor(y) for y in sample_run(Q, x, [0.37] * 16, [1.1] * 16, None, [0.97] * 16))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
