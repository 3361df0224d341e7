"""Calls of the serving operators' Python mirror and C ABI that must be refused before any device work, without a GPU."""
import ctypes as C
import decimal

import numpy as np
import pytest

import qlib
from test_qserve import A, CALLS

torch = pytest.importorskip("torch")
Q = qlib.load()


class OnGpu:
    """A host tensor that says it lies on a GPU, at an address that is never used."""
    is_cuda = True

    def __init__(self, host):
        self.host = host

    dtype = property(lambda self: self.host.dtype)
    shape = property(lambda self: self.host.shape)
    stride = lambda self, *d: self.host.stride(*d)  # noqa: E731
    numel = lambda self: self.host.numel()  # noqa: E731
    element_size = lambda self: self.host.element_size()  # noqa: E731
    is_contiguous = lambda self: self.host.is_contiguous()  # noqa: E731
    data_ptr = lambda self: A  # noqa: E731


def on_gpu(*shape, dtype=torch.float32):
    return OnGpu(torch.zeros(shape, dtype=dtype))


def paged_kv():
    return Q.PagedKV(on_gpu(4, 2, 16, 64), on_gpu(4, 2, 16, 64))


@pytest.mark.parametrize("cos,sin", [((9, 64), (9, 64)), ((9, 32), (9, 64)), ((9, 64), (9, 32)), ((18, 32), (9, 32)), ((9, 32), (18, 32)),
                                     ((288,), (288,)), ((9, 2, 16), (9, 2, 16))])
def test_tables_of_another_shape_are_refused(cos, sin):
    """A table as wide as a head, with every angle twice, has enough elements, and another position's angles in every row."""
    i = on_gpu(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="positions, head_dim / 2"):
        Q.paged_append(paged_kv(), on_gpu(3, 2, 64), on_gpu(3, 2, 64), i, positions=i, cos=on_gpu(*cos), sin=on_gpu(*sin), stream=0)


@pytest.mark.parametrize("call", ["attention", "sample"])
def test_a_workspace_that_is_larger_than_its_memory_is_refused(call):
    """An expanded tensor has more elements than bytes behind it."""
    work = OnGpu(torch.zeros(1, dtype=torch.uint8).expand(1 << 28))
    i = on_gpu(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="work is not contiguous"):
        if call == "sample":
            Q.sample_rows(on_gpu(2, 100), on_gpu(2), i, work, stream=0)
        else:
            Q.paged_attention(paged_kv(), on_gpu(2, 4, 64), on_gpu(2, 3, dtype=torch.int32), i, on_gpu(2, 4, 64), work, stream=0)


@pytest.mark.skipif(qlib.gpu_available(), reason="the calls that are not refused would run")
def test_scales_up_to_the_last_one_whose_base_two_form_is_finite(capfd):
    """Scores are formed in base two: a scale times log2 e above a float's range would make a score of 0 a NaN."""
    for scale in (2.4e38, 2.9e38, 3e38):
        assert CALLS["query"]({"scale": scale}) != 0
        assert "scale must" in capfd.readouterr().err
    assert CALLS["query"]({"scale": 2.3e38}) != 0
    assert "no GPU" in capfd.readouterr().err


@pytest.mark.parametrize("top", [0.0, 0.7, 20.0, -20.0, 333.25, 1e6, -1e6, 1e9, 2.0 ** 40])
@pytest.mark.parametrize("temperature", [0.001, 0.7, 1.0, 3.0, 64.0, 1e6])
def test_weights_of_sampled_tokens(top, temperature):
    """e of a token against 60 digits: off by 2^-37 + 2^-52 |top| / temperature of the largest at most, as documented.

    The first part: both tokens' fractions of a cell are rounded to 2^-38 (2^-39 each), their series ends behind 2^-44, and
    each is rounded to 2^-43; 2 (2^-39 + 2^-43) in all.  The second: the grid's place of a logit, 16 log2(e) l / T, is a product
    rounded to 2^-53 of itself, and an error of it counts ln 2 / 16 times; for the top and a token near it 2 x 2^-53 |top| / T, and a
    token far from it weighs little.  The factor's own rounding counts (l_0 - l) / T 2^-52 e^-((l_0 - l) / T) < 2^-53."""
    t = np.float32(temperature)
    rng, l0 = np.random.default_rng(int(temperature * 1000)), np.float32(top)
    x = np.float32(np.float64(l0) - float(t) * np.concatenate([rng.random(150) * 3.0, rng.random(150) * 30.0]))
    f = Q.lib().qllama_test_sample_weight
    f.argtypes, f.restype = [C.c_float] * 3, C.c_ulonglong
    whole = f(l0, l0, t)
    assert 2 ** 43 <= whole < 1.045 * 2 ** 43
    with decimal.localcontext(decimal.Context(prec=60)):
        bound = decimal.Decimal(2) ** -37 + decimal.Decimal(2) ** -52 * abs(decimal.Decimal(float(l0))) / decimal.Decimal(float(t))
        for l in x:
            e = ((decimal.Decimal(float(l)) - decimal.Decimal(float(l0))) / decimal.Decimal(float(t))).exp()
            off = abs(decimal.Decimal(f(l, l0, t)) / whole - e)
            assert off <= bound, (l, off / bound)
