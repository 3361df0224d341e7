"""Drafted trees, shared pages and rules on logits (include/qserve.h) on the GPU at their documented limits: offsets past 32
bits, the most requests and rows, long histories; and two calls side by side on streams of their own."""
import math
import random

import numpy as np
import pytest
from test_gpu_qserve import Buffer, Dev, Q, Stream, Work, dev_i32, i32, make_cache  # noqa: F401
from test_gpu_qserve_pages import fork_ref, fork_run
from test_gpu_qserve_tree import attend, case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class Raw:
    """A device tensor of which only some pages have a host copy."""
    is_cuda, dtype = True, torch.bfloat16

    def __init__(self, buffer, shape):
        self.buffer, self.shape = buffer, torch.Size(shape)

    def stride(self):
        st, n = [], 1
        for s in reversed(self.shape):
            st.insert(0, n)
            n *= s
        return tuple(st)

    data_ptr = lambda self: self.buffer.p  # noqa: E731
    numel = lambda self: math.prod(self.shape)  # noqa: E731
    element_size = lambda self: 2  # noqa: E731
    is_contiguous = lambda self: True  # noqa: E731


def test_pages_behind_two_billion_elements(Q):  # noqa: F811
    """Attention and moves where offsets pass 32 bits, in elements and in bytes (2.3 G elements; only six pages are filled):
    what the same rows give in a small cache."""
    pages, KVH, page, hd = 17600, 8, 16, 128
    one = KVH * page * hd
    ids = [17599, 0, 16384, 8200, 17598, 12000]
    g = torch.Generator().manual_seed(6)
    host = [torch.randn((len(ids), KVH, page, hd), generator=g).bfloat16() for _ in range(2)]
    buffers = [Buffer(2 * one * pages) for _ in range(2)]
    put = lambda b, p, y: b.L.qllama_h2d(b.p + 2 * one * p, y.contiguous().data_ptr(), 2 * one)  # noqa: E731
    for b, x in zip(buffers, host):
        for p, y in zip(ids, x):
            assert put(b, p, y) == 0
    big = Q.PagedKV(*(Raw(b, (pages, KVH, page, hd)) for b in buffers))
    small = Q.PagedKV(*(Dev(x) for x in host))
    q = torch.randn((7, 16, hd), generator=g)
    table = torch.tensor([[0, 1, 2, 3, 4]], dtype=torch.int32)
    for kv, t in ((small, table), (big, torch.tensor([ids[:5]], dtype=torch.int32))):
        o, lse = attend(Q, kv, q, [0, 7], t, [75], None, nodes=7)
        if kv is small:
            want = o, lse
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    at = lambda i: ids[i] * page  # noqa: E731
    Q.paged_move(big, dev_i32([at(0) + 3]), dev_i32([at(5) + 1]), count=dev_i32([9]))
    Q.paged_move(big, dev_i32([at(4) + 2, at(2)]), dev_i32([at(5), at(3) + 15]), starts=dev_i32([0, 2]))
    for b, x in zip(buffers, host):
        y = x.clone()
        y[5, :, 1:10] = x[0, :, 3:12]
        y[5, :, 0] = x[4, :, 2]
        y[3, :, 15] = x[2, :, 0]
        got = torch.empty_like(x)
        assert b.L.qllama_device_sync() == 0
        for i, p in enumerate(ids):
            z = torch.empty((KVH, page, hd), dtype=torch.bfloat16)
            assert b.L.qllama_d2h(z.data_ptr(), b.p + 2 * one * p, 2 * one) == 0
            got[i] = z
        assert torch.equal(got, y)


def test_the_most_requests(Q):  # noqa: F811
    """8192 requests of 0 to 3 rows: plan and acceptance; a fork of 8192 into 8192."""
    n, r = 8192, random.Random(1)
    m = [r.randint(0, 3) for _ in range(n)]
    starts = np.concatenate([[0], np.cumsum(m)])
    rows = int(starts[-1])
    lens = np.array(m) + 100
    parents = torch.tensor([[-1, 0, r.randint(0, 1)] for _ in range(n)], dtype=torch.int32)
    pos, mask = i32(rows), Dev(torch.zeros((rows, 1), dtype=torch.int64))
    ds, dn, dp = dev_i32(starts.tolist()), dev_i32(lens.tolist()), Dev(parents)
    Q.tree_plan(ds, dn, dp, pos, mask)
    deep = lambda i, j: 0 if j == 0 else 1 if j == 1 else 1 + int(parents[i, 2])  # noqa: E731
    assert np.array_equal(pos.get(), [100 + deep(i, j) for i in range(n) for j in range(m[i])])
    assert np.array_equal(mask.get().flatten(), [[1, 3, 5 + 2 * int(parents[i, 2])][j] for i in range(n) for j in range(m[i])])
    zero = dev_i32([0] * rows)
    acc, last, lens2, path, src, dst = i32(n), i32(n), i32(n), i32(rows), i32(rows), i32(rows)
    Q.tree_accept(ds, dn, dp, zero, zero, dev_i32(list(range(rows))), acc, last, lens2, path, src, dst)
    # all tokens are alike: the path goes to the first child each time
    want = [min(k, 2) + (k == 3 and int(parents[i, 2]) == 1) for i, k in enumerate(m)]
    assert np.array_equal(acc.get(), want) and np.array_equal(last.get(), [0 if k else -1 for k in m])
    table = np.arange(2 * n).reshape(n, 2)
    source = [r.randrange(n) for _ in range(n)]
    ring = list(range(2 * n, 3 * n)) + [-1] * (2 * n)
    args = ([r.randint(0, 8) for _ in range(n)], table.tolist(), source, [r.randint(0, 9) for _ in range(n)], [0] * (3 * n), ring, [0, n], 4)
    want, got = fork_ref(*args, [[-77] * 2 for _ in source], 2), fork_run(Q, *args, 2)
    assert [k for k in want if not np.array_equal(got[k], want[k])] == []


def test_the_most_rows_of_logits(Q):  # noqa: F811
    rows, V = 65535, 40
    x = torch.randn(rows, V)
    req = torch.arange(rows, dtype=torch.int32) % 7
    tokens = torch.arange(7 * 3, dtype=torch.int32).view(7, 3)
    out = Dev(torch.zeros(rows, V))
    Q.logit_rules(Dev(x), out, requests=Dev(req), tokens=Dev(tokens), n_tokens=dev_i32([3] * 7), presence=Dev(torch.full((7,), 0.5)))
    want = x.double()
    want[torch.arange(rows)[:, None], tokens.long()[req.long()]] -= 0.5
    assert torch.equal(out.get(), want.float())
    big = torch.zeros(2, 1 << 20)
    out = Dev(big.clone())
    Q.logit_rules(Dev(big), out, bias_tokens=dev_i32([[(1 << 20) - 1, 0], [7, 1 << 20]]), bias=Dev(torch.tensor([[1.0, 2.0], [3.0, 4.0]])))
    got = out.get()
    assert got[0, -1] == 1 and got[0, 0] == 2 and got[1, 7] == 3 and got.count_nonzero() == 3


def test_two_calls_side_by_side(Q):  # noqa: F811
    """Calls on two streams, with workspaces of their own, many times: each gives what it gives alone."""
    a = case("bf16", 8, 2, 128, 16, "head", [3000, 500], [20, 3], 1, 1, Q, "tree")
    b = case("f32", 6, 2, 64, 16, "head", [2100, 900, 40], [40, 9, 5], 0, 2, Q)
    sides = []
    for kv, q, starts, table, lens, seen, mask in (a, b):
        want = attend(Q, kv, q, starts, table, lens, mask, spare=0)
        H = q.shape[1]
        args = [Dev(q), dev_i32(starts), Dev(table), dev_i32(lens), Dev(torch.zeros_like(q)), Work(Buffer(Q.tree_attention_work(kv, len(q), len(lens), H)))]
        sides.append((kv, args, None if mask is None else Dev(mask), Dev(torch.zeros(q.shape[:2])), want, Stream()))
    for _ in range(20):
        for kv, args, mask, lse, _, s in sides:
            Q.tree_attention(kv, *args, mask=mask, lse=lse, stream=s.p.value)
    for kv, args, mask, lse, want, s in sides:
        s.sync()
        assert torch.equal(args[4].get(), want[0]) and torch.equal(lse.get(), want[1])
