"""The C ABI of the serving operators for drafted trees, shared pages and rules on logits (include/qserve.h) and their Python
mirror without a GPU: structure layouts and the refusals (all made before any device work)."""
import ctypes as C
import os
import struct
import subprocess

import pytest

import qlib

Q = qlib.load()
L = Q.lib()
A = 0x7000000000                 # addresses that are never dereferenced
B = A + (1 << 20)

FIELDS = {
    "tree_plan": ("QTreePlan", Q.TREE_PLAN, "n_req nodes max_rows words parent_stride starts lens parents positions mask"),
    "tree_accept": ("QTreeAccept", Q.TREE_ACCEPT, "n_req nodes max_rows parent_stride starts lens parents tokens chosen slots accepted last lens_out path src dst"),
    "query": ("QTreeQuery", Q.TREE_QUERY, "rows n_req n_heads width words nodes q_stride o_stride lse_stride table_stride q o lse mask starts table lens scale work work_bytes"),
    "fork": ("QPagedFork", Q.PAGED_FORK, "n_old n_new width page_size n_pages ring_size table_stride table_out_stride lens table from keep extra state ring table_out "
             "lens_out status extra_out state_out src dst count work work_bytes"),
    "moves": ("QPagedMoves", Q.PAGED_MOVES, "n_moves n_groups src dst count starts bad"),
    "rules": ("QLogitRules", Q.LOGIT_RULES, "rows vocab n_req stride out_stride logits out requests capacity token_stride tokens n_tokens n_prompt repetition presence "
              "frequency words starts drafted mask n_bias bias_stride bias_tokens bias n_masks allowed_stride allowed allowed_rows"),
}
GOOD = {
    "tree_plan": dict(n_req=3, nodes=8, max_rows=20, words=1, parent_stride=8, starts=A, lens=A, parents=A, positions=B, mask=B),
    "tree_accept": dict(n_req=3, nodes=8, max_rows=20, parent_stride=8, starts=A, lens=A, parents=A, tokens=A, chosen=A + 64, slots=A + 128, accepted=B,
                        last=B, lens_out=B, path=B, src=B + 64, dst=B + 128),
    "query": dict(rows=9, n_req=2, n_heads=4, width=5, words=1, nodes=0, q_stride=256, o_stride=256, lse_stride=4, table_stride=5, q=A, o=B, lse=0, mask=A,
                  starts=A, table=A, lens=A, scale=0.0, work=A, work_bytes=1 << 40),
    "fork": {**dict(n_old=2, n_new=3, width=4, page_size=16, n_pages=50, ring_size=50, table_stride=4, table_out_stride=4),
             **{k: A + 4096 * i for i, k in enumerate("lens table from keep extra state ring table_out lens_out status extra_out state_out src dst count work".split())},
             "work_bytes": 1 << 40},
    "moves": dict(n_moves=4, n_groups=0, src=A, dst=A, count=0, starts=0, bad=0),
    "rules": dict(rows=2, vocab=100, n_req=2, stride=100, out_stride=100, logits=A, out=B, requests=0, capacity=5, token_stride=5, tokens=A, n_tokens=A, n_prompt=0,
                  repetition=0, presence=0, frequency=0, words=0, starts=0, drafted=0, mask=0, n_bias=0, bias_stride=0, bias_tokens=0, bias=0, n_masks=0,
                  allowed_stride=0, allowed=0, allowed_rows=0),
}


def pack(name, change):
    _, fmt, fields = FIELDS[name]
    v = {**GOOD[name], **change}
    assert set(v) == set(fields.split())
    return fmt.pack(*(v[f] for f in fields.split()))


def cache(**kw):
    c = Q.QPagedKV(Q.KV_F32, 10, 16, 2, 64, 2 * 16 * 64, 16 * 64, 64, A, A + (1 << 20), 0, 0, 0, None, None)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def caches(*changes):
    return (Q.QPagedKV * len(changes))(*[cache(**c) for c in changes])


def test_structures_match_the_header(tmp_path):
    """Size, and offset of every member, as a C compiler lays them out: a number packed at a member lands there."""
    src = tmp_path / "s.c"
    lines = ['#include <stdio.h>', '#include "qserve.h"', 'int main(void) {']
    for kind, _, fields in FIELDS.values():
        lines.append(f'printf("%zu", sizeof({kind}));')
        lines += [f'printf(" %zu", offsetof({kind}, {f}));' for f in fields.split()] + ['printf("\\n");']
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(qlib.ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    for (kind, fmt, fields), line in zip(FIELDS.values(), out):
        size, *offsets = [int(x) for x in line.split()]
        assert fmt.size <= size <= fmt.size + 7, kind        # struct leaves out the padding at the end
        codes = [c for c in fmt.format.lstrip("@")]
        assert len(codes) == len(offsets), kind
        for i, (f, at) in enumerate(zip(fields.split(), offsets)):
            v = [0] * len(codes)
            v[i] = 1.0 if codes[i] == "f" else 0x11223344
            mark = struct.pack("@" + codes[i], v[i])
            assert fmt.pack(*v)[at:at + len(mark)] == mark, (kind, f)


CALLS = {"tree_plan": lambda kw: L.qllama_tree_plan(pack("tree_plan", kw), None),
         "tree_accept": lambda kw: L.qllama_tree_accept(pack("tree_accept", kw), None),
         "query": lambda kw: L.qllama_tree_attention(C.byref(cache()), pack("query", kw), None),
         "cache": lambda kw: L.qllama_tree_attention(C.byref(cache(**kw)), pack("query", {}), None),
         "cache_move": lambda kw: L.qllama_paged_move(C.byref(cache(**kw)), 1, pack("moves", {}), None),
         "second": lambda kw: L.qllama_paged_move(caches({}, kw), 2, pack("moves", {}), None),
         "fork": lambda kw: L.qllama_paged_fork(pack("fork", kw), None),
         "moves": lambda kw: L.qllama_paged_move(caches({}), 1, pack("moves", kw), None),
         "rules": lambda kw: L.qllama_logit_rules(pack("rules", kw), None)}

REFUSED = [("tree_plan", kw, w) for kw, w in [
    ({"n_req": -1}, "n_req"), ({"n_req": 8193}, "n_req"), ({"nodes": 0}, "nodes"), ({"nodes": 1025, "parent_stride": 1025}, "nodes"), ({"parent_stride": 7}, "nodes"),
    ({"words": 0}, "words"), ({"words": 5}, "words"), ({"max_rows": -1}, "max_rows"), ({"starts": 0}, "null"), ({"lens": 0}, "null"), ({"parents": 0}, "null"),
    ({"positions": 0}, "null"), ({"mask": 0}, "null"), ({"mask": B + 4}, "aligned"), ({"lens": A + 2}, "aligned")]]
REFUSED += [("tree_accept", kw, w) for kw, w in [
    ({"n_req": 8193}, "n_req"), ({"nodes": 0}, "nodes"), ({"parent_stride": -1}, "nodes"), ({"max_rows": -1}, "max_rows"), ({"max_rows": (1 << 30) + 1}, "max_rows"),
    ({"path": A}, "output"), ({"src": A + 64}, "output"), ({"dst": A + 128}, "output"), ({"slots": A + 1}, "aligned"), ({"last": B + 2}, "aligned")]
    + [({f: 0}, "null") for f in "starts lens parents tokens chosen slots accepted last lens_out path src dst".split()]]
REFUSED += [("query", kw, w) for kw, w in [
    ({"n_req": -1}, "n_req"), ({"rows": -1}, "rows"), ({"rows": (1 << 23) + 1}, "rows"), ({"nodes": -1}, "nodes"), ({"n_heads": 3}, "multiple"), ({"n_heads": 0}, "multiple"),
    ({"q": 0}, "null"), ({"o": 0}, "null"), ({"table": 0}, "null"), ({"lens": 0}, "null"), ({"starts": 0}, "null"), ({"words": 0}, "words"), ({"words": 5}, "words"),
    ({"mask": 0}, "words"), ({"mask": A + 4}, "aligned"), ({"q_stride": 255}, "stride"), ({"o_stride": 0}, "stride"), ({"lse": A, "lse_stride": 3}, "stride"),
    ({"width": 0}, "width"), ({"table_stride": 4}, "width"), ({"width": (1 << 27) - 60, "table_stride": 1 << 27}, "2^31 - 1024"), ({"scale": -1.0}, "scale"),
    ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"o": A}, "o must not"), ({"work": 0}, "work"), ({"work": A + 8}, "work"),
    ({"work_bytes": 100}, "work"), ({"q": A + 1}, "aligned"), ({"rows": 1 << 23, "n_heads": 256, "q_stride": 1 << 20, "o_stride": 1 << 20}, "2^31 - 1024"),
    ({"n_req": 1 << 30, "rows": 1 << 22, "n_heads": 256, "q_stride": 1 << 20, "o_stride": 1 << 20, "width": 1 << 26, "table_stride": 1 << 26}, "too large")]]
REFUSED += [("fork", kw, w) for kw, w in [
    ({"n_old": -1}, "n_old"), ({"n_new": 8193}, "n_old"), ({"width": 0}, "width"), ({"page_size": 0}, "page size"),
    ({"width": 1 << 20, "page_size": 1 << 11, "table_stride": 1 << 20, "table_out_stride": 1 << 20}, "31 bits"), ({"n_pages": 0}, "pages"), ({"n_pages": 1 << 28}, "31 bits"),
    ({"ring_size": 0}, "ring"), ({"ring_size": (1 << 30) + 1}, "ring"), ({"table_stride": 3}, "stride"), ({"table_out_stride": 3}, "stride"),
    ({"state_out": A + 4096 * 5}, "output"), ({"table_out": A + 4096}, "output"), ({"lens_out": A}, "output"), ({"count": A + 4096 * 3}, "output"),
    ({"work": 0}, "work"), ({"work": A + 8}, "work"), ({"work_bytes": 16}, "work"), ({"keep": A + 1}, "aligned")]
    + [({f: 0}, "null") for f in "lens table from extra state ring table_out lens_out status extra_out state_out src dst count".split()]]
REFUSED += [("moves", kw, w) for kw, w in [
    ({"n_moves": -1}, "n_moves"), ({"n_moves": (1 << 23) + 1}, "n_moves"), ({"starts": A, "n_groups": -1}, "n_groups"), ({"starts": A, "n_groups": 2, "count": A}, "count"),
    ({"src": 0}, "null"), ({"dst": 0}, "null"), ({"count": A + 2}, "aligned"), ({"bad": A + 1}, "aligned"), ({"starts": A + 1, "n_groups": 2}, "aligned")]]
REFUSED += [("second", kw, "alike") for kw in [{"type": 1}, {"n_pages": 9}, {"page_size": 8}, {"n_kv": 1}, {"head_dim": 56}, {"page_stride": 4096}, {"head_stride": 2048},
                                               {"slot_stride": 72}]]
REFUSED += [("rules", kw, w) for kw, w in [
    ({"rows": -1}, "rows"), ({"rows": 65536}, "rows"), ({"vocab": 0}, "vocab"), ({"vocab": (1 << 20) + 1, "stride": 1 << 21, "out_stride": 1 << 21}, "vocab"), ({"n_req": -1}, "n_req"),
    ({"logits": 0}, "null"), ({"out": 0}, "null"), ({"stride": 99}, "vocab"), ({"out_stride": 99}, "vocab"), ({"out": A, "out_stride": 104}, "same stride"),
    ({"n_tokens": 0}, "history"), ({"capacity": -1}, "history"), ({"token_stride": 4}, "history"), ({"mask": A, "words": 1, "starts": A}, "mask"),
    ({"mask": A, "words": 1, "drafted": A}, "mask"), ({"mask": A, "words": 5, "starts": A, "drafted": A}, "mask"), ({"mask": A + 4, "words": 1, "starts": A, "drafted": A}, "aligned"),
    ({"n_bias": 4097, "bias": A, "bias_tokens": A, "bias_stride": 5000}, "n_bias"), ({"n_bias": 2, "bias": A, "bias_stride": 2}, "n_bias"),
    ({"n_bias": 2, "bias": A, "bias_tokens": A, "bias_stride": 1}, "n_bias"), ({"allowed": A, "allowed_stride": 4}, "masks"),
    ({"allowed": A, "allowed_rows": A, "allowed_stride": 3}, "masks"), ({"logits": A + 2}, "aligned"), ({"frequency": A + 1}, "aligned")]]
REFUSED += [(n, kw, w) for n in ("cache", "cache_move") for kw, w in [({"k": None}, "null"), ({"type": 4}, "type"), ({"head_dim": 60}, "head_dim"), ({"slot_stride": 56}, "strides"),
                                                                    ({"k": A + 8}, "aligned"), ({"type": 3}, "scales")]]


@pytest.mark.parametrize("call,change,word", REFUSED, ids=lambda x: str(x) if not isinstance(x, dict) else "-".join(x))
def test_refusals(call, change, word, capfd):
    assert CALLS[call](change) != 0
    err = capfd.readouterr().err
    assert err.startswith("Error: qllama_") and word in err, err


@pytest.mark.skipif(qlib.gpu_available(), reason="checks the no-GPU error path")
@pytest.mark.parametrize("call", ["tree_plan", "tree_accept", "query", "fork", "moves", "rules"])
def test_without_a_gpu_the_calls_fail_cleanly(call, capfd):
    assert CALLS[call]({}) != 0
    assert "no GPU" in capfd.readouterr().err


def test_nothing_to_do_is_no_error():
    assert CALLS["tree_plan"]({"n_req": 0}) == 0 and CALLS["tree_accept"]({"n_req": 0}) == 0
    assert CALLS["query"]({"n_req": 0}) == 0 and CALLS["query"]({"rows": 0}) == 0
    assert CALLS["moves"]({"n_moves": 0}) == 0 and CALLS["moves"]({"starts": A, "n_groups": 0}) == 0 and CALLS["rules"]({"rows": 0}) == 0
    assert L.qllama_paged_move(caches({}), 0, pack("moves", {}), None) == 0


def test_workspace_sizes():
    w = L.qllama_tree_attention_work
    assert w(C.byref(cache()), 8, 2, 4, 0) > 0 and w(C.byref(cache()), 0, 0, 4, 0) > 0
    assert w(C.byref(cache()), 8, 2, 5, 0) == 0 and w(C.byref(cache(type=9)), 8, 2, 4, 0) == 0 and w(C.byref(cache()), -1, 2, 4, 0) == 0
    assert L.qllama_paged_fork_work(0, 0, 1) > 0 and L.qllama_paged_fork_work(1, 1, 0) == 0 and L.qllama_paged_fork_work(8193, 1, 5) == 0


def test_python_mirror_refuses_what_does_not_fit():
    torch = pytest.importorskip("torch")
    i, f = torch.zeros(8, dtype=torch.int32), torch.zeros(2, 9)
    with pytest.raises(ValueError, match="not on the GPU"):
        Q.tree_plan(i, i, i.view(2, 4), i, i.long().view(8, 1), stream=0)
    with pytest.raises(ValueError, match="not on the GPU"):
        Q.tree_accept(i, i, i.view(2, 4), i, i, i, i, i, i, i, i, i, stream=0)
    with pytest.raises(ValueError, match="a row for every request"):
        Q.paged_fork(i, i.view(2, 4), i, i, i, i, 16, i.view(2, 4), i, i, i, i, i, i, i, i, stream=0)
    with pytest.raises(ValueError, match="not on the GPU"):
        Q.logit_rules(f, f, stream=0)
    with pytest.raises(ValueError, match="no such requests"):
        Q.paged_fork_work(1, 1, 0)


class Tensor:
    """A host tensor that passes for one on the GPU: the mirror only reads its address, type, shape and strides."""
    is_cuda = True

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)


class Calls:
    """In the library's place: keeps the structures that it is handed."""

    def __getattr__(self, name):
        return lambda a, stream: self.__dict__.__setitem__("got", a) or 0


def packed(monkeypatch, kind, call):
    monkeypatch.setattr(Q, "_lib", Calls())
    call()
    _, fmt, fields = FIELDS[kind]
    return dict(zip(fields.split(), fmt.unpack(Q._lib.__dict__["got"])))


def test_logit_rules_counts_requests_where_something_is_looked_up_by_them(monkeypatch):
    """The number of requests is that of the settings' rows; without any, all numbers but negative ones are requests."""
    torch = pytest.importorskip("torch")
    i = lambda *s: Tensor(torch.zeros(s, dtype=torch.int32))  # noqa: E731
    f = lambda *s: Tensor(torch.zeros(s))  # noqa: E731
    x, masks, tree = f(2, 40), dict(allowed=i(1, 2), allowed_rows=i(2)), dict(mask=Tensor(torch.zeros((2, 1), dtype=torch.int64)), drafted=i(2))
    n_req = lambda **kw: packed(monkeypatch, "rules", lambda: Q.logit_rules(x, x, stream=0, **kw))["n_req"]  # noqa: E731
    assert n_req(**masks) == 2
    assert n_req(requests=i(2), **masks) == 2 ** 31 - 1
    assert n_req(requests=i(2)) == 2 ** 31 - 1
    assert n_req(requests=i(2), starts=i(6), **tree, **masks) == 5
    assert n_req(requests=i(2), starts=i(2), **tree) == 1
    assert n_req(requests=i(2), tokens=i(5, 3), n_tokens=i(5)) == 5
    for name, t in (("repetition", f(7)), ("presence", f(7)), ("frequency", f(7))):
        assert n_req(requests=i(2), **{name: t}, **masks) == 7
    assert n_req(requests=i(2), bias=f(4, 2), bias_tokens=i(4, 2)) == 4
    with pytest.raises(ValueError, match="frequency has 3 elements"):
        n_req(requests=i(2), presence=f(4), frequency=f(3))
    with pytest.raises(ValueError, match="bias_tokens"):
        n_req(bias=f(2, 2))


def test_tree_accept_leaves_out_rows_that_the_mask_has_no_bit_for(monkeypatch):
    torch = pytest.importorskip("torch")
    i = lambda *s: Tensor(torch.zeros(s, dtype=torch.int32))  # noqa: E731
    args = (i(3), i(2), i(2, 100), *(i(200) for _ in range(3)), *(i(2) for _ in range(3)), *(i(200) for _ in range(3)))
    call = lambda *m: packed(monkeypatch, "tree_accept", lambda: Q.tree_accept(*args, stream=0, **(dict(mask=Tensor(torch.zeros((200, m[0]), dtype=torch.int64))) if m else {})))  # noqa: E731
    for got, nodes in ((call(), 100), (call(1), 64), (call(2), 100), (call(4), 100)):
        assert got["nodes"] == nodes and got["parent_stride"] == 100


@pytest.mark.parametrize("n_req", [2 ** 31 - 1, 2 ** 31 - 4096])
def test_loops_over_requests_stay_in_32_bits(n_req, capfd):
    """As many requests as a step of 64 or 2048 past them would leave 32 bits: both attentions refuse them."""
    assert CALLS["query"]({"n_req": n_req, "rows": 1, "n_heads": 2, "width": 1, "table_stride": 1}) != 0
    assert "n_req" in capfd.readouterr().err
    c = cache(page_size=1, page_stride=2 * 64, head_stride=64)
    assert L.qllama_paged_attention(C.byref(c), Q.PAGED_QUERY.pack(n_req, 2, 1, 128, 128, 2, 1, A, B, 0, A, A, 0.0, A, 1 << 40), None) != 0
    assert "too large" in capfd.readouterr().err
