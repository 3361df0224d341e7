"""Rules on logits (include/qserve.h) on the GPU: every output is the definition's, evaluated in 64 bits and rounded once."""
import random

import numpy as np
import pytest
from test_gpu_qserve import Dev, Q, dev_i32  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
INF = float("inf")


def rules_ref(x, req, n_req, hist, rep, pres, freq, drafted, bias, allowed):
    """hist: per request (tokens, prompt); drafted: per row, tokens above it; bias: per request [(token, value)]; allowed: per row a
    truth value a token, or None.  64-bit arithmetic, rounded once."""
    out = x.copy()
    rows, V = x.shape
    with np.errstate(all="ignore"):
        for i in range(rows):
            r = req[i]
            if not 0 <= r < n_req:
                out[i] = 7.0
                continue
            y = x[i].astype(np.float64)
            tokens, prompt = hist[r] if hist else ([], 0)
            made = [t for t in list(tokens[prompt:]) + drafted[i] if 0 <= t < V]
            known = {t for t in list(tokens[:prompt]) if 0 <= t < V} | set(made)
            f = lambda a, none: none if a is None or np.isnan(a[r]) else np.float64(np.float32(a[r]))  # noqa: E731
            p, q, s = f(rep, 1.0), f(pres, 0.0), f(freq, 0.0)
            p = p if p > 0 else np.float64(1.0)
            for t in known:
                y[t] = y[t] / p if y[t] > 0 else y[t] * p
            for t in set(made):
                y[t] -= s * made.count(t) + q
            seen = set()
            for t, b in bias[r] if bias else []:
                if 0 <= t < V and t not in seen:
                    seen.add(t)
                    if not np.isnan(b):
                        y[t] += np.float64(np.float32(b))
            out[i] = y.astype(np.float32)
            if allowed[i] is not None:
                out[i][~allowed[i]] = -INF
    return out


def build(seed, rows, V, n_req, history, n_bias, masks, tree):
    r, g = random.Random(seed), np.random.default_rng(seed)
    x = (g.standard_normal((rows, V)) * 5).astype(np.float32)
    x[:, ::17] = [-INF, INF, np.nan, 0.0][seed % 4]
    req = [i % n_req for i in range(rows)] if not tree else sorted(i % n_req for i in range(rows))
    hot = [r.randrange(V) for _ in range(9)]
    pick = lambda: r.choice([r.choice(hot), r.randrange(V), -3, V, 2 ** 31 - 1]) if r.random() < 0.5 else r.randrange(V)  # noqa: E731
    cap = max(1, history)
    tokens = np.array([[pick() for _ in range(cap)] for _ in range(n_req)], np.int64)
    lens = [r.choice([0, history, r.randint(0, history)]) for _ in range(n_req)]
    prompt = [r.choice([0, x0, r.randint(0, x0)]) for x0 in lens]
    hist = [(list(tokens[i, :lens[i]]), prompt[i]) for i in range(n_req)]
    s = {"rep": [r.choice([1.0, 1.3, 0.7, float("nan"), -2.0, 0.0]) for _ in range(n_req)], "pres": [r.choice([0.0, 0.7, float("nan")]) for _ in range(n_req)],
         "freq": [r.choice([0.0, 0.3, -0.1]) for _ in range(n_req)]}
    bias = [[(pick(), r.choice([-INF, 2.5, float("nan"), -1.0])) for _ in range(n_bias)] for _ in range(n_req)] if n_bias else None
    words = -(-V // 32) + 1
    bits = g.random((max(masks, 1), words * 32)) < g.random((max(masks, 1), 1))
    which = [r.choice([-1, masks, r.randrange(masks)]) if masks else -1 for _ in range(rows)]
    packed = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    starts, drafted, mask, above = None, None, None, [[] for _ in range(rows)]
    if tree:
        starts = [sum(q < k for q in req) for k in range(n_req + 1)]
        drafted = [pick() for _ in range(rows)]
        mask = np.zeros((rows, 2), np.uint64)
        for i in range(rows):
            m = starts[req[i] + 1] - starts[req[i]]
            for b in range(128):
                if r.random() < 0.3:
                    mask[i, b // 64] |= np.uint64(1) << np.uint64(b % 64)
                    if b < m:
                        above[i].append(drafted[starts[req[i]] + b])
    return x, req, tokens, lens, prompt, hist, s, bias, bits[:, :V], which, packed, starts, drafted, mask, above


def run(Q, x, out, req, tokens, lens, prompt, s, bias, which, packed, masks, starts, drafted, mask):  # noqa: F811
    f32 = lambda a: Dev(torch.tensor(a, dtype=torch.float32))  # noqa: E731
    kw = {}
    if bias is not None:
        kw.update(bias_tokens=dev_i32([[t for t, _ in b] for b in bias]), bias=f32([[v for _, v in b] for b in bias]))
    if masks:
        kw.update(allowed=Dev(torch.from_numpy(packed)), allowed_rows=dev_i32(which))
    if mask is not None:
        kw.update(starts=dev_i32(starts), drafted=dev_i32(drafted), mask=Dev(torch.from_numpy(mask.view(np.int64))))
    Q.logit_rules(x, out, requests=dev_i32(req), tokens=Dev(torch.from_numpy(tokens.astype(np.int32))), n_tokens=dev_i32(lens), n_prompt=dev_i32(prompt),
                  repetition=f32(s["rep"]), presence=f32(s["pres"]), frequency=f32(s["freq"]), **kw)


def same(a, b):
    return np.array_equal(a.view(np.int32)[~np.isnan(b)], b.view(np.int32)[~np.isnan(b)]) and np.array_equal(np.isnan(a), np.isnan(b))


@pytest.mark.parametrize("seed,rows,V,n_req,history,n_bias,masks,tree", [
    (1, 1, 1, 1, 3, 1, 1, False), (2, 3, 100, 3, 20, 4, 2, False), (3, 7, 2047, 3, 50, 0, 0, False), (4, 5, 2049, 5, 0, 3, 1, False), (5, 20, 5001, 4, 200, 70, 3, True),
    (6, 130, 1000, 2, 30, 0, 2, True), (7, 2, 128256, 2, 3000, 300, 2, False), (8, 70, 32000, 70, 40, 2, 5, False), (9, 300, 32001, 30, 10, 1, 4, True),
    (10, 140, 128256, 12, 100, 4, 3, True), (11, 9, 4100, 1, 1000, 200, 1, True)])
def test_rules(Q, seed, rows, V, n_req, history, n_bias, masks, tree):  # noqa: F811
    """Odd vocabularies, slices of every size, tokens out of range, settings that are none, infinities and NaN among the logits;
    into another buffer (its stride odd or not) and in place."""
    x, req, tokens, lens, prompt, hist, s, bias, bits, which, packed, starts, drafted, mask, above = build(seed, rows, V, n_req, history, n_bias, masks, tree)
    if rows > 2 and not tree:
        req[1], req[2] = -1, n_req                     # rows of no request
    allowed = [bits[w] if masks and 0 <= w < masks else None for w in which]
    want = rules_ref(x, req, n_req, hist, s["rep"], s["pres"], s["freq"], above, bias, allowed)
    pad = [0, 1, 4][seed % 3]
    dx = Dev(torch.from_numpy(np.concatenate([x, np.zeros((rows, pad), np.float32)], 1)))[:, :V]
    out = Dev(torch.full((rows, V + 4 * (seed % 2)), 7.0))[:, :V]
    args = (req, tokens, lens, prompt, s, bias, which, packed, masks, starts, drafted, mask)
    run(Q, dx, out, *args)
    assert same(out.get().contiguous().numpy(), want)
    run(Q, dx, dx, *args)
    want[[i for i in range(rows) if not 0 <= req[i] < n_req]] = x[[i for i in range(rows) if not 0 <= req[i] < n_req]]
    assert same(dx.get().contiguous().numpy(), want)


def test_no_rules_and_a_mask_alone(Q):  # noqa: F811
    x = torch.randn(4, 333)
    out = Dev(torch.zeros(4, 333))
    Q.logit_rules(Dev(x), out)
    assert torch.equal(out.get(), x)
    words = torch.zeros((1, 11), dtype=torch.int32)
    words[0, 3] = -2 ** 31 + 5
    Q.logit_rules(Dev(x), out, allowed=Dev(words), allowed_rows=dev_i32([0, -1, 0, 1]))
    got = out.get()
    want = torch.full((333,), -INF)
    for t in (96, 98, 127):
        want[t] = x[0, t]
    assert torch.equal(got[0], want) and torch.equal(got[1], x[1]) and torch.equal(got[3], x[3])
    empty = Dev(torch.zeros((1, 11), dtype=torch.int32))
    Q.logit_rules(Dev(x), out, allowed=empty, allowed_rows=dev_i32([0, 0, 0, 0]))
    assert bool((out.get() == -INF).all())


def test_a_token_used_a_million_times(Q):  # noqa: F811
    """Counts pass 16 bits and are exact."""
    n = 1_000_003
    tokens = torch.zeros((1, n + 5), dtype=torch.int32)
    tokens[0, :10] = 1
    out = Dev(torch.zeros(1, 8))
    Q.logit_rules(Dev(torch.ones(1, 8)), out, tokens=Dev(tokens), n_tokens=dev_i32([n]), frequency=Dev(torch.tensor([0.25])))
    assert out.get().tolist() == [[1 - 0.25 * (n - 10), 1 - 2.5] + [1.0] * 6]


def test_lengths_out_of_range(Q):  # noqa: F811
    """A length above the capacity counts as the capacity, a prompt longer than the history as the history."""
    tokens = dev_i32([[1, 2, 2, 3], [1, 1, 1, 1], [4, 4, 4, 4]])
    out = Dev(torch.zeros(3, 6))
    Q.logit_rules(Dev(torch.ones(3, 6)), out, tokens=tokens, n_tokens=dev_i32([2 ** 31 - 1, -5, 2]), n_prompt=dev_i32([-1, 3, 9]),
                  presence=Dev(torch.tensor([1.0, 1.0, 1.0])), repetition=Dev(torch.tensor([1.0, 2.0, 2.0])))
    assert out.get().tolist() == [[1, 0, 0, 0, 1, 1], [1] * 6, [1, 1, 1, 1, 0.5, 1]]


def test_masks_of_requests_beyond_the_rows(Q):  # noqa: F811
    """Without settings nothing is looked up by request, and any number but a negative one names a row that takes part: a grammar
    alone, one active request of many; a drafted tree's rows with no penalties."""
    x = torch.randn(3, 70)
    words = torch.tensor([[5, 0, 1], [-1, -1, -1]], dtype=torch.int32)
    want = torch.full((3, 70), -INF)
    want[0, [0, 2, 64]] = x[0, [0, 2, 64]]
    want[1] = x[1]
    for req in ([3, 900, 2 ** 31 - 2], [3, 3, -1]):
        want[2] = x[2] if req[2] < 0 else torch.where(want[0] > -INF, x[2], -INF)
        same_row = Dev(x.clone())
        Q.logit_rules(same_row, same_row, requests=dev_i32(req), allowed=Dev(words), allowed_rows=dev_i32([0, 1, 0]))
        assert torch.equal(same_row.get(), want)
        out = Dev(torch.full((3, 70), 7.0))
        Q.logit_rules(Dev(x), out, requests=dev_i32(req), allowed=Dev(words), allowed_rows=dev_i32([0, 1, 0]))
        if req[2] < 0:
            want[2] = 7.0
        assert torch.equal(out.get(), want)
    out = Dev(torch.full((3, 70), 7.0))
    Q.logit_rules(Dev(x), out, requests=dev_i32([0, 0, 0]), starts=dev_i32([0, 3]), drafted=dev_i32([1, 2, 3]), mask=Dev(torch.ones((3, 1), dtype=torch.int64)),
                  allowed=Dev(words), allowed_rows=dev_i32([0, 1, 1]))
    want[0], want[2] = torch.full((70,), -INF), x[2]
    want[0, [0, 2, 64]] = x[0, [0, 2, 64]]
    assert torch.equal(out.get(), want)
