"""The serving operators' C ABI (include/qserve.h) and their Python mirror without a GPU: symbols, structure layouts,
the refusals (all made before any device work), and where the attention looks for a token."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import qlib

Q = qlib.load()
HEADER = os.path.join(qlib.ROOT, "include", "qserve.h")


def declared():
    text = re.sub(r"//.*", "", open(HEADER).read())
    text = re.sub(r"(?m)^\s*#.*$", "", text)
    return sorted(set(re.findall(r"\b(qllama_[a-z_]+)\s*\([^;{}]*\)\s*;", text)))


def test_every_declared_function_is_exported():
    names = declared()
    assert {"qllama_paged_plan", "qllama_paged_append", "qllama_paged_attention", "qllama_sample_rows"} <= set(names)
    out = subprocess.run(["nm", "-D", "--defined-only", Q.LIB_PATH], capture_output=True, text=True, check=True).stdout
    exported = set(line.split()[-1] for line in out.splitlines() if line.strip())
    assert not [n for n in names if n not in exported]


def test_structures_match_the_header(tmp_path):
    """Sizes and the offset of every last member as a C compiler lays them out."""
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "qserve.h"\nint main(void) {\n'
                   'printf("%zu %zu %zu %zu %zu\\n", sizeof(QPagedKV), sizeof(QPagedPlan), sizeof(QPagedRows), sizeof(QPagedQuery), sizeof(QSampleRows));\n'
                   'printf("%zu %zu %zu %zu %zu\\n", offsetof(QPagedKV, v_scale), offsetof(QPagedPlan, table_stride), offsetof(QPagedRows, bad), offsetof(QPagedQuery, work), offsetof(QSampleRows, work));\n'
                   'return 0; }\n')
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(qlib.ROOT, "include"), str(src), "-o", str(exe)], check=True)
    sizes, offsets = ([int(x) for x in line.split()] for line in
                      subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert sizes == [C.sizeof(Q.QPagedKV), Q.PAGED_PLAN.size, Q.PAGED_ROWS.size, Q.PAGED_QUERY.size, Q.SAMPLE_ROWS.size]
    at = lambda s, mark: s.index(np.uint64(mark).tobytes())  # noqa: E731
    M = 0x1122334455667788
    plan = Q.PAGED_PLAN.pack(1, 2, 3, 4, 5, M, *([0] * 12))
    rows = Q.PAGED_ROWS.pack(*([0] * 15), M)
    query = Q.PAGED_QUERY.pack(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0.0, M, 0)
    sample = Q.SAMPLE_ROWS.pack(0, 0, 0, *([0] * 9), M, 0)
    assert offsets == [Q.QPagedKV.v_scale.offset, at(plan, M), at(rows, M), at(query, M), at(sample, M)]


# Addresses that are never dereferenced: every refusal below comes before device work.
A = 0x7000000000


def cache(**kw):
    c = Q.QPagedKV(Q.KV_F32, 10, 16, 2, 64, 2 * 16 * 64, 16 * 64, 64, A, A + (1 << 20), 0, 0, 0, None, None)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def plan(**kw):
    names = ("n_req", "width", "page_size", "ring_size", "max_rows", "table_stride", "cached", "added", "state", "table", "ring", "lens",
             "status", "starts", "state_out", "slots", "positions", "requests")
    v = dict(zip(names, [3, 4, 16, 20, 8, 4] + [A + 4096 * i for i in range(12)]))
    v.update(kw)
    return Q.PAGED_PLAN.pack(*(v[n] for n in names))


def rows(**kw):
    names = ("rows", "n_heads", "q", "k", "v", "q_out", "q_stride", "k_stride", "v_stride", "q_out_stride", "slots", "positions", "cos_t",
             "sin_t", "n_pos", "bad")
    v = dict(rows=5, n_heads=4, q=A, k=A, v=A, q_out=A, q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, slots=A, positions=A,
             cos_t=A, sin_t=A, n_pos=7, bad=0)
    v.update(kw)
    return Q.PAGED_ROWS.pack(*(v[n] for n in names))


def query(**kw):
    names = ("n_req", "n_heads", "width", "q_stride", "o_stride", "lse_stride", "table_stride", "q", "o", "lse", "table", "lens", "scale",
             "work", "work_bytes")
    v = dict(n_req=2, n_heads=4, width=5, q_stride=256, o_stride=256, lse_stride=4, table_stride=5, q=A, o=A + 4096, lse=0, table=A, lens=A,
             scale=0.0, work=A, work_bytes=1 << 40)
    v.update(kw)
    return Q.PAGED_QUERY.pack(*(v[n] for n in names))


def sample(**kw):
    names = ("rows", "vocab", "stride", "logits", "u", "temperature", "top_k", "top_p", "min_p", "token", "kept", "prob", "work", "work_bytes")
    v = dict(rows=2, vocab=100, stride=100, logits=A, u=A, temperature=0, top_k=0, top_p=0, min_p=0, token=A, kept=0, prob=0, work=A,
             work_bytes=1 << 40)
    v.update(kw)
    return Q.SAMPLE_ROWS.pack(*(v[n] for n in names))


L = Q.lib()
CALLS = {"plan": lambda kw: L.qllama_paged_plan(plan(**kw), None),
         "rows": lambda kw: L.qllama_paged_append(C.byref(cache()), rows(**kw), None),
         "query": lambda kw: L.qllama_paged_attention(C.byref(cache()), query(**kw), None),
         "cache": lambda kw: L.qllama_paged_attention(C.byref(cache(**kw)), query(), None),
         "cache_append": lambda kw: L.qllama_paged_append(C.byref(cache(**kw)), rows(), None),
         "sample": lambda kw: L.qllama_sample_rows(sample(**kw), None)}

BAD_CACHE = [({"k": None}, "null"), ({"v": None}, "null"), ({"type": 4}, "type"), ({"type": -1}, "type"), ({"n_pages": 0}, "pages"),
             ({"page_size": 0}, "pages"), ({"n_pages": 1 << 20, "page_size": 1 << 12}, "pages"), ({"n_kv": 0}, "KV heads"),
             ({"head_dim": 60}, "head_dim"), ({"head_dim": 264, "slot_stride": 264}, "head_dim"), ({"head_dim": 0}, "head_dim"),
             ({"slot_stride": 56}, "strides"), ({"slot_stride": 68}, "strides"), ({"head_stride": 1028}, "strides"), ({"page_stride": 0}, "strides"),
             ({"page_stride": -2048}, "strides"), ({"k": A + 8}, "aligned"), ({"v": A + 4}, "aligned"), ({"type": 3}, "scales"),
             ({"type": 3, "k_scale": A, "v_scale": A}, "strides of the scales")]
REFUSED = [("plan", kw, w) for kw, w in [
    ({"n_req": -1}, "n_req"), ({"n_req": 8193}, "n_req"), ({"width": 0}, "width"), ({"page_size": 0}, "page size"),
    ({"width": 1 << 20, "page_size": 1 << 11, "table_stride": 1 << 20}, "31 bits"), ({"ring_size": 0}, "ring"), ({"max_rows": -1}, "max_rows"),
    ({"ring_size": (1 << 30) + 1}, "ring"), ({"max_rows": (1 << 30) + 1}, "max_rows"),
    ({"table_stride": 3}, "stride"), ({"state": 0}, "null"), ({"ring": 0}, "null"), ({"cached": 0}, "null"), ({"added": 0}, "null"),
    ({"table": 0}, "null"), ({"lens": 0}, "null"), ({"starts": 0}, "null"), ({"state_out": 0}, "null"), ({"slots": 0}, "null"),
    ({"positions": 0}, "null"), ({"requests": 0}, "null"), ({"state_out": A + 4096 * 2}, "output"), ({"lens": A}, "output"),
    ({"status": A + 4096}, "output")]]
REFUSED += [("rows", kw, w) for kw, w in [
    ({"rows": -1}, "rows"), ({"rows": (1 << 23) + 1}, "rows"), ({"k": 0}, "null"), ({"v": 0}, "null"), ({"slots": 0}, "null"),
    ({"q_out": 0}, "q_out"), ({"n_heads": 0}, "q_out"),
    ({"sin_t": 0}, "rotation"), ({"positions": 0}, "rotation"), ({"n_pos": 0}, "rotation"), ({"k_stride": 127}, "stride"),
    ({"v_stride": 0}, "stride"), ({"q_stride": 255}, "stride"), ({"q_out_stride": 255}, "stride"), ({"k": A + 2}, "aligned")]]
REFUSED += [("query", kw, w) for kw, w in [
    ({"n_req": -1}, "n_req"), ({"n_heads": 3}, "multiple"), ({"n_heads": 0}, "multiple"), ({"q": 0}, "null"), ({"o": 0}, "null"), ({"table": 0}, "null"),
    ({"lens": 0}, "null"), ({"q_stride": 255}, "stride"), ({"o_stride": 0}, "stride"), ({"lse": A, "lse_stride": 3}, "stride"), ({"width": 0}, "width"),
    ({"table_stride": 4}, "width"), ({"width": 1 << 28, "table_stride": 1 << 28}, "2^31 - 64"),
    ({"width": (1 << 27) - 4, "table_stride": 1 << 27, "n_req": 1}, "2^31 - 64"), ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"),
    ({"scale": float("inf")}, "scale"), ({"o": A}, "o must not"), ({"work": 0}, "work"), ({"work": A + 8}, "work"), ({"work_bytes": 100}, "work"),
    ({"q": A + 1}, "aligned")]]
REFUSED += [("sample", kw, w) for kw, w in [
    ({"rows": -1}, "rows"), ({"vocab": 0}, "vocab"), ({"vocab": (1 << 20) + 1, "stride": 1 << 21}, "vocab"), ({"stride": 99}, "vocab"),
    ({"logits": 0}, "null"), ({"u": 0}, "null"), ({"token": 0}, "null"), ({"work": 0}, "work"), ({"work": A + 4}, "work"), ({"work_bytes": 0}, "work"),
    ({"logits": A + 2}, "aligned")]]
REFUSED += [(n, kw, w) for kw, w in BAD_CACHE for n in ("cache", "cache_append")]


@pytest.mark.parametrize("call,change,word", REFUSED, ids=lambda x: str(x) if not isinstance(x, dict) else "-".join(x))
def test_refusals(call, change, word, capfd):
    assert CALLS[call](change) != 0
    err = capfd.readouterr().err
    assert err.startswith("Error: qllama_") and word in err, err


@pytest.mark.skipif(qlib.gpu_available(), reason="checks the no-GPU error path")
@pytest.mark.parametrize("call", ["plan", "rows", "query", "sample"])
def test_without_a_gpu_the_calls_fail_cleanly(call, capfd):
    assert CALLS[call]({}) != 0
    assert "no GPU" in capfd.readouterr().err


def test_nothing_to_do_is_no_error():
    assert CALLS["rows"]({"rows": 0}) == 0 and CALLS["query"]({"n_req": 0}) == 0 and CALLS["sample"]({"rows": 0}) == 0


def test_workspace_sizes():
    assert L.qllama_paged_attention_work(C.byref(cache()), 3, 4) > 0
    assert L.qllama_paged_attention_work(C.byref(cache()), 3, 5) == 0 and L.qllama_paged_attention_work(C.byref(cache(type=9)), 3, 4) == 0
    assert L.qllama_sample_rows_work(5, 1000) > 0 and L.qllama_sample_rows_work(5, 0) == 0 and L.qllama_sample_rows_work(-1, 10) == 0


@pytest.mark.parametrize("page_size", [1, 3, 16, 48])
def test_page_of_a_token(page_size):
    """Every token of a table with holes: the page and place of the definition, -1 for pages outside the cache, for
    tokens behind the request and for lengths above the table's room."""
    rng = np.random.default_rng(page_size)
    width, n_pages = 5, 11
    table = rng.integers(-2, n_pages + 2, width).astype(np.int32)
    table[0], table[1] = n_pages, -1
    place = C.c_int(0)
    f = L.qllama_test_page_of
    f.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_longlong, C.POINTER(C.c_int)]
    for length in (-3, 0, 1, page_size, 2 * page_size + 1, width * page_size, width * page_size + 9, 2 ** 31 - 1):
        held = min(max(length, 0), width * page_size)
        for key in list(range(-1, width * page_size + 3)) + [2 ** 31, 2 ** 40]:
            page = f(table.ctypes.data, width, page_size, n_pages, length, key, C.byref(place))
            want = int(table[key // page_size]) if 0 <= key < held else -1
            if want >= n_pages or want < 0:
                assert page == -1 and place.value == 0
            else:
                assert page == want and place.value == key % page_size


def test_python_mirror_refuses_what_does_not_fit():
    torch = pytest.importorskip("torch")
    f = torch.zeros(4, 2, 16, 64)
    with pytest.raises(ValueError, match="not on the GPU"):
        Q.PagedKV(f, f)
    with pytest.raises(ValueError, match="no cache of"):
        Q.PagedKV(f.double(), f.double())
    with pytest.raises(ValueError, match="scales"):
        Q.PagedKV(f.to(torch.int8), f.to(torch.int8))
    with pytest.raises(ValueError, match="alike"):
        Q.PagedKV(f, f.transpose(1, 2))
    i = torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError, match="not on the GPU"):
        Q.paged_plan(i, i, i.view(8, 1), i, i, 16, i, i, i, i, i, i, i, stream=0)
    with pytest.raises(ValueError, match="not on the GPU"):
        Q.sample_rows(torch.zeros(2, 9), torch.zeros(2), i, i, stream=0)
    with pytest.raises(ValueError, match="no such rows"):
        Q.sample_rows_work(1, 0)
