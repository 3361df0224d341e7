"""The serving operators (include/qserve.h) on the GPU where a caller's program meets them at an edge: an error that an
earlier call of the program has left behind, negative scales of an int8 cache, what float arithmetic may lose, equal
requests, the model's own products between the calls, and torch's GPU tensors."""
import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest

import qlib
from test_gpu_qserve import (EPS, HIP, Buffer, Dev, Server, Work, attend, attend_ref, dev_i32, i32, make_cache, one_step, pages_for,  # noqa: F401
                             sample_ref, sample_run, widened, Q)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_an_error_left_by_another_call_is_not_the_operators(Q):
    """An unrelated HIP call of the caller's has failed and nobody has asked for its error: the four calls do their work and
    return 0, and the error is still there for the caller to find."""
    HIP.hipGetLastError()
    a, b = Server(Q, seed=6), Server(Q, seed=6)
    for s in (a, b):
        s.feed(0, [3, 1, 40, 0, 9])
    one_step(a)
    want = a.results()
    assert HIP.hipSetDevice(1 << 20) != 0                      # no such device; the current one stays
    left = HIP.hipPeekAtLastError()
    assert left != 0, "the runtime keeps no error here: this test shows nothing"
    b.store()
    assert HIP.hipPeekAtLastError() == left
    b.answer(b.q[:b.n])
    assert HIP.hipPeekAtLastError() == left
    b.sample()
    assert HIP.hipPeekAtLastError() == left
    wide = attend_two_launches(Q)                              # its join is a launch of its own
    assert HIP.hipGetLastError() == left
    assert all(torch.equal(x, y) for x, y in zip(want, b.results()))
    assert all(torch.equal(x, y) for x, y in zip(wide, attend_two_launches(Q)))


def attend_two_launches(Q):
    """A request long enough to be split and joined."""
    g = torch.Generator().manual_seed(2)
    kv = make_cache(Q, "f16", 130, 2, 16, 64, gen=g)
    return attend(Q, kv, torch.randn((1, 4, 64), generator=g), pages_for([2000], 16, 125, 130, 1), [2000])


@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("order", ["all", "mixed", "one", "up", "down"])
def test_attention_int8_negative_scales(Q, page, order):
    """A scale is the caller's number, of either sign: all of them negative, signs in turn, one enormous negative one among
    small positive ones, and negative ones that run over sixty powers of ten.  The bound is the one of positive scales of
    these sizes."""
    H, KVH, hd, n = 8, 2, 64, 90
    pages = -(-n // page)
    kv = make_cache(Q, "i8", pages, KVH, page, hd, gen=torch.Generator().manual_seed(page))
    slots = torch.arange(pages * page)
    e = {"up": slots * 0.6 - 27.0, "down": 27.0 - slots * 0.6, "one": torch.where(slots == 40, 20.0, -5.0)}.get(order, slots * 0.0 - 1.5).double()
    sign = {"mixed": 1.0 - 2.0 * (slots % 3 != 0), "one": torch.where(slots == 40, -1.0, 1.0)}.get(order, -torch.ones(len(slots)))
    size = (10.0 ** e).float()
    shape = lambda x: x.float().reshape(pages, 1, page).expand(pages, KVH, page).contiguous()  # noqa: E731
    kv.v_scale.set(shape(size * sign))
    kv.k_scale.set(kv.k_scale.get() * shape(sign))
    sizes = Q.PagedKV(kv.k, kv.v, kv.k_scale, Dev(shape(size)))
    q = torch.randn((2, H, hd), generator=torch.Generator().manual_seed(4))
    table, lens = torch.arange(pages, dtype=torch.int32).expand(2, pages).contiguous(), [n, n - 7]
    wo, wl, _, lb = attend_ref(kv, q, table, lens)
    bound = attend_ref(sizes, q, table, lens, uneven=True)[2]
    for t in (table, widened(table, page)):
        o, lse = attend(Q, kv, q, t, lens)
        assert bool(((o.double() - wo).abs() <= bound).all()), ((o.double() - wo).abs() - bound).max()
        assert bool(((lse.double() - wl).abs() <= lb).all())


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
def test_attention_lse_of_small_scores(Q, typ):
    """One token whose score is small: its log-sum-exp is the score.  q and k are powers of two, so that the score is exact but
    for its way through base two: log2 e as a float (EPS), that in two 16-bit floats (2 EPS: off by 2^-23), and back (the
    constant and the product, 2 EPS).  The logarithm of a sum of one weight is 0."""
    H, KVH, hd = 4, 2, 64
    kv = make_cache(Q, typ, 2, KVH, 16, hd)
    kv.k.set(torch.zeros_like(kv.k.host))
    k = kv.k.host.clone()
    k[:, :, 0, 3] = 1
    kv.k.set(k)
    if typ == "i8":
        kv.k_scale.set(torch.ones_like(kv.k_scale.host))
    q = torch.zeros((6, H, hd))
    score = torch.tensor([2.0 ** -3, 2.0 ** -6, -2.0 ** -6, 2.0 ** -9, 2.0 ** -12, -2.0 ** -15])
    q[:, :, 3] = score[:, None]
    table = torch.zeros((6, 1), dtype=torch.int32)
    for t in (table, widened(table, 16)):
        _, lse = attend(Q, kv, q, t, [1] * 6, scale=1.0)
        assert bool(((lse.double() - score.double()[:, None]).abs() <= 5 * EPS * score.abs().double()[:, None]).all()), lse


def test_attention_int8_keeps_a_scale_to_23_bits(Q):
    """One token: the output is its code times its scale.  The scale enters the product as two 16-bit floats, each rounded to
    nearest: the first is off by half a step of 11 bits, 2^-11 of the scale's power of two, the second by half a step of 11
    bits of that, 2^-23; the products' sum is rounded once (2^-23 if that is cut off).  Scales whose last bits make two floats
    that are cut off differ by 3 x 2^-23 are among them."""
    KVH, hd, n = 2, 64, 64
    g = torch.Generator().manual_seed(3)
    kv = make_cache(Q, "i8", n, KVH, 16, hd, gen=g)
    r = np.random.default_rng(1)
    m = r.integers(0, 1 << 23, (n, KVH)).astype(np.uint32)
    m[:8] = (1 << 12) * np.arange(1, 9)[:, None] + 3
    m[8:16] = 0x7fffff
    scale = torch.zeros((n, KVH, 16))
    scale[:, :, 0] = torch.from_numpy((m + np.uint32(0x3f800000)).view(np.float32).copy()) * torch.tensor([0.5, 0.03125] * (n // 2))[:, None]
    kv.v_scale.set(scale)
    table = torch.arange(n, dtype=torch.int32)[:, None].contiguous()
    want = (kv.v.get()[:, :, 0].double() * scale[:, :, 0, None].double())
    for t in (table, widened(table, 16)):
        o, _ = attend(Q, kv, torch.randn((n, KVH, hd), generator=g), t, [1] * n)
        assert bool(((o.double() - want).abs() <= 2.0 ** -22 * want.abs()).all()), ((o.double() - want).abs() / want.abs().clamp(min=1e-30)).max()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "i8"])
def test_attention_equal_requests_give_equal_bits(Q, typ):
    """Short tables: a block takes a tile, so equal requests are equal work, and give equal bits."""
    g = torch.Generator().manual_seed(14)
    kv = make_cache(Q, typ, 12, 2, 32, 128, "head", g)
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 2, 3], [7, 7, 7, 7]], dtype=torch.int32)
    q = torch.randn((4, 4, 128), generator=g)
    q[2] = q[0]
    o, lse = attend(Q, kv, q, table, [128, 100, 128, 97])
    assert torch.equal(o[0], o[2]) and torch.equal(lse[0], lse[2])
    assert not torch.equal(o[0], o[1])


def test_a_step_with_the_models_products_between(Q):
    """The step as a model's layer makes it, with nothing waited for: rows of q, k and v from an int8 product, plan, append,
    attention, the output's product, logits, sampling.  The products run on the library's stream, so the calls do too."""
    L = Q.lib()
    L.qmatmul_device_noalloc.argtypes = [C.c_void_p, C.c_int, C.POINTER(Q.QTensor), C.c_void_p]
    H, KVH, hd, n, D, V = 8, 2, 64, 5, 256, 500
    r = np.random.default_rng(8)
    weights = [(r.standard_normal(s) * 0.05).astype(np.float32) for s in ((D, (H + 2 * KVH) * hd), (H * hd, D), (D, V))]
    W = [Q.QWeight(w) for w in weights]
    x = r.standard_normal((n, D)).astype(np.float32)
    s = Server(Q, rows=n, seed=2)
    dx, dy = Dev(torch.from_numpy(x)), Dev(torch.zeros((n, D)))

    def product(a, w, out):
        assert L.qmatmul_device_noalloc(a.data_ptr(), n, C.byref(w.t), out.data_ptr()) == 0

    try:
        for step in range(6):
            s.feed(step, [1] * n)
            assert L.qllama_device_sync() == 0
            product(dx, W[0], s.qkv)
            s.store()
            s.answer(s.q)
            product(s.o, W[1], dy)
            product(dy, W[2], s.logits)
            s.sample()
            assert L.qllama_sync() == 0
            # each product on the values that the call before it left, through the host entry point
            assert np.array_equal(s.qkv.get().numpy().reshape(n, -1), Q.qmatmul(x, W[0]))
            y = Q.qmatmul(s.o.get().numpy().reshape(n, -1), W[1])
            assert np.array_equal(dy.get().numpy(), y) and np.array_equal(s.logits.get().numpy(), Q.qmatmul(y, W[2]))
            lens = s.lens.get().tolist()
            assert lens == [step + 1] * n and s.slots.get().min() >= 0
            wo, _, bound, _ = attend_ref(s.kv, s.q.get(), s.table.get(), lens)
            assert bool(((s.o.get().double() - wo).abs() <= bound).all())
            token, u = s.token.get().tolist(), s.u.get().tolist()
            for i in range(n):
                want = sample_ref(s.logits.host.numpy()[i], float(np.float32(0.9)), 50, float(np.float32(0.9)), float(np.float32(0.01)), u[i])
                assert token[i] == want[0]
            s.next()
    finally:
        for w in W:
            w.close()


PRODUCTS_CHILD = """
import ctypes as C, sys
import numpy as np, torch
sys.path.insert(0, "tests")
import qlib
Q = qlib.load()
L = Q.lib()
L.qmatmul_device_noalloc.argtypes = [C.c_void_p, C.c_int, C.POINTER(Q.QTensor), C.c_void_p]
n, D, H, KVH, hd, page = 7, 256, 8, 2, 64, 16
r = np.random.default_rng(3)
W = [Q.QWeight((r.standard_normal(s) * 0.05).astype(np.float32)) for s in ((D, (H + 2 * KVH) * hd), (H * hd, D))]
product = lambda a, w, out: L.qmatmul_device_noalloc(a.data_ptr(), n, C.byref(w.t), out.data_ptr())
stream = torch.cuda.ExternalStream(L.qllama_stream())
stream.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(stream):
    s = torch.cuda.current_stream().cuda_stream
    i32 = lambda *d: torch.zeros(d, dtype=torch.int32, device="cuda")
    kv = Q.PagedKV(*(torch.zeros((9, KVH, page, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    table, ring, state, cached, added = i32(n, 2), torch.arange(9, dtype=torch.int32, device="cuda"), i32(2), i32(n), i32(n) + 1
    state[1] = 9
    lens, status, starts, state_out, slots, positions, requests = i32(n), i32(n), i32(n + 1), i32(2), i32(n), i32(n), i32(n)
    cos, sin = torch.ones((32, hd // 2), device="cuda"), torch.zeros((32, hd // 2), device="cuda")
    work = torch.empty(Q.paged_attention_work(kv, n, H), dtype=torch.uint8, device="cuda")
    seen = []
    for step in range(4):                    # nothing is waited for: torch's work, the products and the calls follow each other
        x = torch.full((n, D), 0.001 * (step + 1), device="cuda") * torch.arange(D, device="cuda")
        qkv, o, y = torch.empty((n, H + 2 * KVH, hd), device="cuda"), torch.empty((n, H, hd), device="cuda"), torch.empty((n, D), device="cuda")
        assert product(x, W[0], qkv) == 0
        Q.paged_plan(cached, added, table, ring, state, page, lens, status, starts, state_out, slots, positions, requests, stream=s)
        q, k, v = qkv.split([H, KVH, KVH], 1)
        Q.paged_append(kv, k, v, slots, q=q, q_out=q, positions=positions, cos=cos, sin=sin, stream=s)
        Q.paged_attention(kv, q, table, lens, o, work, stream=s)
        assert product(o, W[1], y) == 0
        cached, state = lens.clone(), state_out.clone()
        seen.append((x, qkv, o, y * 1.0))
stream.synchronize()
values = []
for x, qkv, o, y in seen:
    x, qkv, o, y = (t.cpu().numpy() for t in (x, qkv, o, y))
    assert np.array_equal(qkv.reshape(n, -1), Q.qmatmul(x, W[0])) and np.array_equal(y, Q.qmatmul(o.reshape(n, -1), W[1]))
    values.append(torch.from_numpy(qkv).bfloat16().double().numpy()[:, H + KVH:])
    k = torch.from_numpy(np.stack([t[1].cpu().numpy() for t in seen[:len(values)]])).bfloat16().double()[:, :, H:H + KVH]
    for h in range(H):                       # the rotation is none here; a weight is off by 200 EPS sum |q k| / 8 = 5e-5 at most
        w = torch.softmax(torch.from_numpy(qkv).double()[None, :, h].mul(k[:, :, h // 4]).sum(-1) / 8.0, 0)
        want = (w[..., None] * torch.from_numpy(np.stack(values))[:, :, h // 4]).sum(0)
        assert (torch.from_numpy(o).double()[:, h] - want).abs().max() <= 1e-4 * max(1.0, want.abs().max().item())
print("steps", len(seen))
"""


def in_torch(code):
    """What a process prints that has loaded torch's HIP runtime first."""
    done = subprocess.run([sys.executable, "-u", "-c", code], cwd=qlib.ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout + done.stderr[-2000:]
    return done.stdout


def test_torch_tensors_and_products_on_the_librarys_stream():
    """A step as documented: torch's work, the products and the calls all on the library's stream, none waited for."""
    assert "steps 4" in in_torch(PRODUCTS_CHILD)


TORCH_CHILD = """
import random, sys
import torch
sys.path.insert(0, "perf")
import operators as P
rng = random.Random(5)
cases = [c for c in P.listed() if c["name"] in ("plan_step", "append_step", "attend_tiny", "attend_one", "sample_few")]
cases += [dict(kind="append", shape="1b", type="i8", page=20, rows=33, mix=4),
          dict(kind="attend", shape="1b", type="i8", page=20, requests=9, most=300, mix=5),
          dict(kind="sample", rows=20, vocab=5001, settings="mixed", mix=6)]
for c in cases:
    out = []
    for P.own in (False, True):
        o = P.run(P.prepare(c, 3))
        torch.cuda.synchronize()
        out.append({k: v.cpu() for k, v in o.items()})
    for k, want in out[0].items():
        got = out[1][k]
        if want.dtype.is_floating_point:
            torch.testing.assert_close(got.float(), want.float(), rtol=2e-5, atol=2e-5)
        else:
            assert torch.equal(got, want), (c, k)
    print("same", c.get("name", c["kind"]), flush=True)
print("all", len(cases))
"""


def test_torch_tensors_on_the_gpu():
    """The Python mirror on torch's own GPU tensors, on torch's stream, in a process that has loaded torch's HIP runtime first:
    whole outputs against elementary torch operations."""
    assert "all 8" in in_torch(TORCH_CHILD)

# ---------------------------------------------------------------------------
# The documented limits
# ---------------------------------------------------------------------------
def attend_dense(kv, q, table, lens):
    """attend_ref for many short requests at once: tables of few pages inside the cache, one KV head a query head."""
    page, hd = kv.k.shape[2], q.shape[2]
    n, room = len(lens), table.shape[1] * page
    rows = lambda x: x.get().double()[table.long()].transpose(1, 2).reshape(n, -1, room, hd)  # noqa: E731
    k, v, q = rows(kv.k), rows(kv.v), q.double()[:, :, None]
    scale, there = 1.0 / math.sqrt(hd), (torch.arange(room) < torch.tensor(lens)[:, None])[:, None]
    s = ((k * q).sum(-1) * scale).masked_fill(~there, -math.inf)
    z = torch.logsumexp(s, 2, keepdim=True)
    w = torch.where(there, torch.exp(s - z), 0.0)
    size = torch.where(there, ((3 * hd + 4) * EPS * (k * q).abs().sum(-1)) * scale + 2 * EPS * s.abs(), 0.0).amax(2, keepdim=True)
    dw = 2 * size + 4 * EPS * torch.where(there, s.abs(), 0.0).amax(2, keepdim=True) + 8 * EPS
    tokens = torch.tensor(lens).double()[:, None]
    wide = lambda x: (x[..., None] * v).sum(2)  # noqa: E731
    bound = (2 * dw + (3 * tokens[..., None] + 16) * EPS) * (w[..., None] * v.abs()).sum(2)
    return wide(w), z[..., 0], bound, dw[..., 0] + (tokens + 16) * EPS + 4 * EPS * z[..., 0].abs()


@pytest.mark.parametrize("typ", ["f32", "i8"])
def test_attention_of_seventy_thousand_requests(Q, typ):
    """More requests than a grid's second dimension takes."""
    n, page, hd, pages = 70000, 16, 8, 500
    g = torch.Generator().manual_seed(1)
    kv = make_cache(Q, typ, pages, 1, page, hd, "head", g)
    if typ == "i8":
        values = kv.k.get().double() * kv.k_scale.get().double()[..., None], kv.v.get().double() * kv.v_scale.get().double()[..., None]
    else:
        values = kv.k.get().double(), kv.v.get().double()
    q = torch.randn((n, 1, hd), generator=g)
    table = torch.randint(0, pages, (n, 2), generator=g, dtype=torch.int32)
    lens = torch.randint(1, 33, (n,), generator=g).tolist()
    o, lse = attend(Q, kv, q, table, lens)

    class Held:
        k, v = (type("T", (), {"shape": x.shape, "get": lambda self, x=x: x})() for x in values)

    wo, wl, bound, lb = attend_dense(Held, q, table, lens)
    if typ == "i8":                                        # 2^-37 of the largest product a token, times its code
        bound = bound + torch.tensor(lens)[:, None, None] * 127 * 2.0 ** -37 * 0.035
    assert bool(((o.double() - wo).abs() <= bound).all()) and bool(((lse.double() - wl).abs() <= lb).all())


@pytest.mark.parametrize("H,KVH", [(65535, 1), (65535, 65535), (65534, 32767)])
def test_attention_of_the_most_heads(Q, H, KVH):
    page, hd, lens = 16, 8, [20]
    g = torch.Generator().manual_seed(2)
    kv = make_cache(Q, "bf16", 2, KVH, page, hd, "head", g)
    q = torch.randn((1, H, hd), generator=g)
    o, lse = attend(Q, kv, q, torch.tensor([[1, 0]], dtype=torch.int32), lens)

    class Held:
        k, v = (type("T", (), {"shape": x.shape, "get": lambda self, x=x: x.get().repeat_interleave(H // KVH, 1)})() for x in (kv.k, kv.v))

    wo, wl, bound, lb = attend_dense(Held, q, torch.tensor([[1, 0]]), lens)
    assert bool(((o.double() - wo).abs() <= bound).all()) and bool(((lse.double() - wl).abs() <= lb).all())


def test_append_of_the_most_rows(Q):
    """2^23 rows, in a random order of their slots."""
    rows, page, hd = 1 << 23, 64, 8
    g = torch.Generator().manual_seed(3)
    kv = Q.PagedKV(*(Dev(torch.zeros((rows // page, 1, page, hd), dtype=torch.bfloat16)) for _ in range(2)))
    k = torch.randn((rows, 1, hd), generator=g)
    slots = torch.randperm(rows, generator=g).to(torch.int32)
    dk = Dev(k)
    Q.paged_append(kv, dk, dk, Dev(slots))
    want = torch.zeros((rows, hd), dtype=torch.bfloat16)
    want[slots.long()] = k[:, 0].bfloat16()
    for x in (kv.k, kv.v):
        assert torch.equal(x.get().view(rows, hd), want)


def test_sample_rows_of_the_most_rows(Q):
    """65535 rows of 7 tokens, every setting in turn."""
    n, V = 65535, 7
    g = torch.Generator().manual_seed(4)
    x = torch.randn((n, V), generator=g) * 2.0
    u = torch.rand(n, generator=g).tolist()
    t, k, p, m = ([y[i % len(y)] for i in range(n)] for y in ([0.8, 1.0, 0.0], [0, 3, 5, 0, 1], [1.0, 0.9, 0.5, 0.97], [0.0, 0.05, 0.0, 0.0, 0.3, 0.0, 0.0]))
    token, kept, prob = sample_run(Q, x, u, t, k, p, m)
    f = lambda y: float(np.float32(y))  # noqa: E731
    for i in list(range(0, n, 61)) + [n - 2, n - 1]:
        want = sample_ref(x[i].numpy(), f(t[i]), k[i], f(p[i]), f(m[i]), u[i])
        assert (token[i], kept[i]) == want[:2] and abs(prob[i] - want[2]) <= 2.0 ** -20 * want[2], i
