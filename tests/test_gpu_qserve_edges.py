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
