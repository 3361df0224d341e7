"""A server that verifies drafted trees, as a user's program runs the calls of include/qserve.h together: pages, positions and
masks, rows into their slots, attention, rules, tokens, acceptance, moves and the rejected rows' pages back; eagerly and
as a captured step.  What it answers is what one token a step answers."""
import random

import numpy as np
import pytest
from test_gpu_qserve import HIP, Dev, Graph, Q, Buffer, Work, dev_i32, i32, same  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
H, KVH, HD, PAGE, VOCAB, LAYERS = 4, 2, 64, 8, 50, 2


class Model:
    """Layers of attention over fixed projections of a token's embedding; the products are the host's, in 32 bits a row."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.w = [torch.randn((VOCAB, (H + 2 * KVH) * HD), generator=g) * 0.7 for _ in range(LAYERS)]
        self.out = torch.randn((H * HD, VOCAB), generator=g) * 2.0
        a = torch.arange(512, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(HD // 2, dtype=torch.float64) / HD)
        self.cos, self.sin = Dev(a.cos().float()), Dev(a.sin().float())

    def rows(self, layer, tokens):
        return self.w[layer][torch.as_tensor(tokens).long().clamp(min=0)].view(len(tokens), H + 2 * KVH, HD)

    def logits(self, o):
        return sum(o).double().reshape(-1, H * HD).matmul(self.out.double()).float()


class Server:
    """n requests; `width` rows a step at most."""

    def __init__(self, Q, model, n, typ, width=64):  # noqa: F811
        self.Q, self.model, self.n, self.R = Q, model, n, width
        self.P, self.W, self.nodes = 40 * n, 40, 16
        shape = (self.P, KVH, PAGE, HD)
        dt = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}[typ]
        mk = lambda: Q.PagedKV(Dev(torch.zeros(shape, dtype=dt)), Dev(torch.zeros(shape, dtype=dt)),  # noqa: E731
                               *([Dev(torch.zeros(shape[:3])), Dev(torch.zeros(shape[:3]))] if typ == "i8" else []))
        self.caches = Q.PagedCaches([mk() for _ in range(LAYERS)])
        ids = list(range(self.P))
        random.Random(1).shuffle(ids)
        self.table, self.ring, self.state = Dev(torch.full((n, self.W), -1, dtype=torch.int32)), dev_i32(ids), dev_i32([0, self.P])
        self.cached, self.extra = dev_i32([0] * n), dev_i32([0] * self.P)
        R = self.R
        self.added, self.lens, self.status, self.starts, self.state2 = i32(n), i32(n), i32(n), i32(n + 1), i32(2)
        self.slots, self.pos, self.req = i32(R), i32(R), i32(R)
        self.parents, self.mask, self.tokens = i32(n, self.nodes), Dev(torch.zeros((R, 1), dtype=torch.int64)), i32(R)
        self.qkv = [Dev(torch.zeros((R, H + 2 * KVH, HD))) for _ in range(LAYERS)]
        self.q, self.o = [Dev(torch.zeros((R, H, HD))) for _ in range(LAYERS)], [Dev(torch.zeros((R, H, HD))) for _ in range(LAYERS)]
        self.work = [Work(Buffer(Q.tree_attention_work(self.caches.caches[0], R, n, H, self.nodes))) for _ in range(LAYERS)]
        self.logits, self.history, self.n_tokens = Dev(torch.zeros((R, VOCAB))), i32(n, 400), dev_i32([0] * n)
        self.rep, self.freq = Dev(torch.full((n,), 1.2)), Dev(torch.full((n,), 0.3))
        self.u, self.choice, self.sample_work = Dev(torch.zeros(R)), i32(R), Work(Buffer(Q.sample_rows_work(R, VOCAB)))
        self.zero = Dev(torch.zeros(R))
        self.accepted, self.last, self.lens2, self.path, self.src, self.dst = i32(n), i32(n), i32(n), i32(R), i32(R), i32(R)
        self.ident, self.table2, self.lens3, self.status2 = dev_i32(list(range(n))), Dev(torch.full((n, self.W), -1, dtype=torch.int32)), i32(n), i32(n)
        self.extra2, self.state3, self.fsrc, self.fdst, self.fcount = i32(self.P), i32(2), i32(n), i32(n), i32(n)
        self.fork_work = Work(Buffer(Q.paged_fork_work(n, n, self.P)))
        self.known = [[] for _ in range(n)]

    def feed(self, trees):
        """trees: per request (tokens, parents), the rows packed one request behind another."""
        tokens = [t for tree in trees for t in tree[0]]
        self.added.set(torch.tensor([len(t[0]) for t in trees], dtype=torch.int32))
        par = torch.full((self.n, self.nodes), -1, dtype=torch.int32)
        for r, (_, p) in enumerate(trees):
            par[r, :len(p)] = torch.tensor(p, dtype=torch.int32)
        self.parents.set(par)
        tokens += [0] * (self.R - len(tokens))
        self.tokens.set(torch.tensor(tokens, dtype=torch.int32))
        for layer, x in enumerate(self.qkv):
            x.set(self.model.rows(layer, tokens))
        h = torch.zeros((self.n, 400), dtype=torch.int32)
        for r, k in enumerate(self.known):
            h[r, :len(k)] = torch.tensor(k, dtype=torch.int32)
        self.history.set(h)
        self.n_tokens.set(torch.tensor([len(k) for k in self.known], dtype=torch.int32))

    def first(self, stream):
        """Up to the attention's outputs."""
        Q = self.Q
        Q.paged_plan(self.cached, self.added, self.table, self.ring, self.state, PAGE, self.lens, self.status, self.starts, self.state2, self.slots,
                     self.pos, self.req, stream=stream)
        Q.tree_plan(self.starts, self.lens, self.parents, self.pos, self.mask, stream=stream)
        for kv, x, q, o, w in zip(self.caches.caches, self.qkv, self.q, self.o, self.work):
            Q.paged_append(kv, x[:, H:H + KVH], x[:, H + KVH:], self.slots, q=x[:, :H], q_out=q, positions=self.pos, cos=self.model.cos,
                           sin=self.model.sin, stream=stream)
            Q.tree_attention(kv, q, self.starts, self.table, self.lens, o, w, mask=self.mask, nodes=self.nodes, stream=stream)

    def second(self, stream):
        """From the logits on."""
        Q = self.Q
        Q.logit_rules(self.logits, self.logits, requests=self.req, tokens=self.history, n_tokens=self.n_tokens, repetition=self.rep, frequency=self.freq,
                      starts=self.starts, drafted=self.tokens, mask=self.mask, stream=stream)
        Q.sample_rows(self.logits, self.u, self.choice, self.sample_work, temperature=self.zero, stream=stream)
        Q.tree_accept(self.starts, self.lens, self.parents, self.tokens, self.choice, self.slots, self.accepted, self.last, self.lens2, self.path,
                      self.src, self.dst, stream=stream)
        Q.paged_move(self.caches, self.src, self.dst, starts=self.starts, stream=stream)
        Q.paged_fork(self.lens, self.table, self.ident, self.extra, self.ring, self.state2, PAGE, self.table2, self.lens3, self.status2, self.extra2,
                     self.state3, self.fsrc, self.fdst, self.fcount, self.fork_work, keep=self.lens2, stream=stream)
        Q.paged_move(self.caches, self.fsrc, self.fdst, count=self.fcount, stream=stream)

    def close(self):
        """The next step begins where this one has ended; the accepted tokens, and what was chosen behind them."""
        self.logits.get()
        got, path, tokens, choice = [], self.path.get().tolist(), self.tokens.get().tolist(), self.choice.get().tolist()
        starts, acc = self.starts.get().tolist(), self.accepted.get().tolist()
        for r in range(self.n):
            rows = path[starts[r]:starts[r] + acc[r]]
            self.known[r] += [tokens[i] for i in rows]
            got.append([tokens[i] for i in rows[1:]] + ([choice[rows[-1]]] if rows else []))
        self.cached.set(self.lens3.get())
        self.table.set(self.table2.get())
        self.state.set(self.state3.get())
        self.extra.set(self.extra2.get())
        return got

    def step(self, trees, stream=None):
        self.feed(trees)
        self.first(stream)
        self.logits.set(self.model.logits([o.get() for o in self.o]))
        self.second(stream)
        return self.close()


def plain(Q, typ, prompts, steps):  # noqa: F811
    """One token a request and step."""
    model = Model(3)
    s = Server(Q, model, len(prompts), typ)
    out = [[] for _ in prompts]
    for k in range(max(len(p) for p in prompts) - 1 + steps):
        trees = [([p[k]] if k < len(p) else [out[r][-1]], [-1]) for r, p in enumerate(prompts)]
        for r, x in enumerate(s.step(trees)):
            if k >= len(prompts[r]) - 1:
                out[r] += x
    return out


PROMPTS = [[3, 9, 30], [7], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [40, 41]]


@pytest.mark.parametrize("typ", ["f32", "bf16", "i8"])
def test_drafted_steps_answer_as_single_tokens_do(Q, typ):  # noqa: F811
    """Drafts that are right, wrong and half right, over many steps: the same tokens in fewer steps, and no page is lost."""
    want = plain(Q, typ, PROMPTS, 40)
    r, model = random.Random(5), Model(3)
    s = Server(Q, model, len(PROMPTS), typ)
    out, first = [[] for _ in PROMPTS], True
    for step in range(60):
        trees = []
        for i, p in enumerate(PROMPTS):
            if first:
                trees.append((p, list(range(-1, len(p) - 1))))            # a prompt is a chain whose tokens are certain
                continue
            ahead = want[i][len(out[i]):]
            tokens, parents, at = [out[i][-1]], [-1], 0
            for d in range(r.randint(0, 5)):
                others = [x for x in (r.randrange(VOCAB), r.randrange(VOCAB)) if not ahead[d:] or x != ahead[d]]
                for x in others[:r.randint(0, 2)]:
                    tokens.append(x)
                    parents.append(at)
                if not ahead[d:] or r.random() < 0.2:
                    break
                tokens.append(ahead[d])
                parents.append(at)
                at = len(tokens) - 1
            trees.append((tokens, parents))
        if first:
            # prompts: every row's token is certain, so only the choice behind the last one counts
            s.feed(trees)
            s.first(None)
            s.logits.set(model.logits([o.get() for o in s.o]))
            s.Q.logit_rules(s.logits, s.logits, requests=s.req, tokens=s.history, n_tokens=s.n_tokens, repetition=s.rep, frequency=s.freq, starts=s.starts,
                            drafted=s.tokens, mask=s.mask)
            s.Q.sample_rows(s.logits, s.u, s.choice, s.sample_work, temperature=s.zero)
            choice, starts = s.choice.get().tolist(), s.starts.get().tolist()
            for i, p in enumerate(PROMPTS):
                s.known[i] = list(p)
                out[i] = [choice[starts[i + 1] - 1]]
            s.cached.set(s.lens.get())
            s.state.set(s.state2.get())
            first = False
        else:
            for o, x in zip(out, s.step(trees)):
                o += x
        if all(len(o) >= 40 for o in out):
            break
    assert [o[:40] for o in out] == [w[:40] for w in want] and step < 38
    used = sum(-(-x // PAGE) for x in s.cached.get().tolist())
    assert s.state.get().tolist()[1] == s.P - used and not any(s.extra.get().tolist())


def test_a_captured_step_equals_an_eager_one(Q):  # noqa: F811
    """Both halves of a step in graphs of their own, replayed between eager steps of a second server with the same inputs."""
    model = Model(4)
    a, b = Server(Q, model, 4, "bf16"), Server(Q, model, 4, "bf16")
    halves = [Graph(lambda stream: b.first(stream)), Graph(lambda stream: b.second(stream))]
    r = random.Random(2)
    for step in range(5):
        trees = []
        for i in range(4):
            m = r.randint(1, 12)
            trees.append(([r.randrange(VOCAB) for _ in range(m)], [-1] + [r.randrange(j) for j in range(1, m)]))
        got = a.step(trees)
        b.feed(trees)
        halves[0].replay()
        logits = model.logits([o.get() for o in b.o])
        b.logits.set(logits)
        halves[1].replay()
        assert b.close() == got
        for x, y in zip(a.o + [a.choice, a.path, a.cached, a.table, a.state, a.ring], b.o + [b.choice, b.path, b.cached, b.table, b.state, b.ring]):
            assert same(x, y.get())
        for x, y in zip(a.caches.caches, b.caches.caches):
            assert same(x.k, y.k.get()) and same(x.v, y.v.get())


def test_forked_requests_continue_apart(Q):  # noqa: F811
    """A request continued by three: each goes on as a server that was fed its tokens alone."""
    model = Model(6)
    s = Server(Q, model, 4, "f32")
    beginning, ends = [5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15], [[20, 21, 22], [30, 31, 32], [40, 41, 42]]
    for t in beginning:
        s.step([([t], [-1])] + [([], [])] * 3)
    src = dev_i32([0, 0, 0, -1])
    Q.paged_fork(s.cached, s.table, src, s.extra, s.ring, s.state, PAGE, s.table2, s.lens3, s.status2, s.extra2, s.state3, s.fsrc, s.fdst, s.fcount, s.fork_work)
    Q.paged_move(s.caches, s.fsrc, s.fdst, count=s.fcount)
    assert s.lens3.get().tolist() == [11, 11, 11, 0] and s.fcount.get().tolist() == [0, 3, 3, 0]
    for x, y in ((s.cached, s.lens3), (s.table, s.table2), (s.extra, s.extra2), (s.state, s.state3)):
        x.set(y.get())
    s.known[1], s.known[2] = list(s.known[0]), list(s.known[0])
    got = [[], [], []]
    for k in range(3):
        s.step([([e[k]], [-1]) for e in ends] + [([], [])])
        for i in range(3):
            got[i].append(s.o[0].get()[i].clone())
    for i, e in enumerate(ends):
        alone = Server(Q, model, 4, "f32")
        for t in beginning:
            alone.step([([t], [-1])] + [([], [])] * 3)
        for k in range(3):
            alone.step([([e[k]], [-1])] + [([], [])] * 3)
            assert torch.equal(alone.o[0].get()[0], got[i][k]), (i, k)


def test_an_error_left_by_another_call_is_not_the_operators(Q):  # noqa: F811
    """An unrelated HIP call of the caller's has failed: the calls do their work, and its error is there to be found."""
    HIP.hipGetLastError()
    model = Model(4)
    a, b = Server(Q, model, 2, "bf16"), Server(Q, model, 2, "bf16")
    trees = [([1, 2, 3], [-1, 0, 0]), ([4, 5], [-1, 0])]
    want = a.step(trees)
    assert HIP.hipSetDevice(1 << 20) != 0                      # no such device; the current one stays
    left = HIP.hipPeekAtLastError()
    assert left != 0, "the runtime keeps no error here: this test shows nothing"
    b.feed(trees)
    b.first(None)
    assert HIP.hipPeekAtLastError() == left
    b.logits.set(model.logits([o.get() for o in b.o]))
    b.second(None)
    assert HIP.hipGetLastError() == left
    assert b.close() == want
