"""A call that the HIP runtime refuses reports its error once: the calls after it, the
library's and torch's, work and do not report it again."""
import random

import numpy as np
import pytest
import torch

from oracle import oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def codec():
    from bitalosdb_amd.codec import BithashCodec
    c = BithashCodec(0)
    yield c
    c.close()


def records(n, seed):
    rng = random.Random(seed)
    buf, hs = bytearray(), []
    for i in range(n):
        rec = O.record_set(rng.randbytes(32), (i + 1) << 8 | 1, rng.randbytes(rng.choice([1, 64, 1024])), 3)
        hs.append((len(buf), len(rec), 0))
        buf += rec
    return np.frombuffer(bytes(buf), np.uint8).copy(), np.array(hs, dtype=O.HANDLE_DT)


def assert_same(got, exp):
    for f in O.DESC_DT.names:
        assert np.array_equal(got[f], exp[f]), f


def test_refused_allocation_is_reported_once(codec):
    """An allocation of 2^60 bytes, more than any card has: NULL and a text, nothing more."""
    src, h = records(300, 5)
    exp, _, _ = O.decode_batch(src, h)
    for _ in range(2):
        assert not codec.L.bhg_malloc_device(codec.ctx, 1 << 60)
        assert b"hipMalloc" in codec.L.bhg_last_error(codec.ctx)
        got, _, _ = codec.decode_host(src, h)   # the library's launch first: no torch call in between
        assert_same(got, exp)
    assert not codec.L.bhg_malloc_device(codec.ctx, 1 << 60)
    assert int((torch.arange(1000, device=codec.device) + 1).sum()) == 500500
