"""Calls of the serving operators' Python mirror and C ABI that must be refused before any device work, without a GPU."""
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
