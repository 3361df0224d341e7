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
                             sample_ref, widened, Q)

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
