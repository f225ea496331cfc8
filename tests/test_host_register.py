"""host_register / host_unregister of the Python codec, on the CPU with a stand-in for the
library: a refusal of the runtime leaves the buffer pageable and is not an error."""
import numpy as np
import pytest

from bitalosdb_amd import _lib as B
from bitalosdb_amd.codec import BithashCodec


class Library:
    def __init__(self):
        self.rc, self.calls = B.BHG_OK, []

    def bhg_host_register(self, ctx, p, n):
        self.calls.append(("register", p, n))
        return self.rc

    def bhg_host_unregister(self, ctx, p):
        self.calls.append(("unregister", p))
        return B.BHG_OK

    def bhg_last_error(self, ctx):
        return b"refused"


@pytest.fixture
def codec(monkeypatch):
    L = Library()
    monkeypatch.setattr(B, "lib", lambda: L)
    c = BithashCodec.__new__(BithashCodec)      # no GPU here: __init__ would raise
    c.L, c.ctx, c._unpinned = L, None, set()
    return c


def test_refused_registration_leaves_the_buffer_pageable(codec):
    a, b = np.zeros(64, np.uint8), np.zeros(64, np.uint8)
    codec.L.rc = B.BHG_EHIP
    assert codec.host_register(a) is False
    codec.L.rc = B.BHG_OK
    assert codec.host_register(b) is True
    codec.host_unregister(a)                    # was never pinned: the library is not called
    codec.host_unregister(b)
    assert codec.L.calls == [("register", a.ctypes.data, 64), ("register", b.ctypes.data, 64),
                             ("unregister", b.ctypes.data)]


def test_registered_after_a_refusal(codec):
    a = np.zeros(64, np.uint8)
    codec.L.rc = B.BHG_EHIP
    assert codec.host_register(a) is False
    codec.L.rc = B.BHG_OK
    assert codec.host_register(a) is True       # no unregister in between: the pin counts
    codec.host_unregister(a)
    assert codec.L.calls[-1] == ("unregister", a.ctypes.data)


@pytest.mark.parametrize("rc", [B.BHG_EINVAL, B.BHG_ENOMEM, B.BHG_ENODEV])
def test_other_failures_raise(codec, rc):
    codec.L.rc = rc
    a = np.zeros(64, np.uint8)
    with pytest.raises(B.BhgError, match="bhg_host_register"):
        codec.host_register(a)
    codec.host_unregister(a)                    # not noted as refused
    assert codec.L.calls[-1] == ("unregister", a.ctypes.data)
