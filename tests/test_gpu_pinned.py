"""bhg_decode_batch_host on memory that was allocated page-locked and mapped (bhg_malloc_host,
torch's pin_memory): the in-place decode of unsorted handles, the chunked pipelines and the copy
kernel into a mapped value buffer, against the restatement, bit for bit.  Buffers also start
inside their allocation, at addresses of every kind mod 16 that the types allow."""
import ctypes
import random

import numpy as np
import pytest
import torch

from bitalosdb_amd.codec import DESC_DT, BithashCodec
from oracle import oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture
def alloc(request, monkeypatch):
    """alloc(nbytes, offset) -> uint8 array in page-locked memory, offset bytes into it."""
    monkeypatch.setenv("BHG_HOST_CHUNK_BYTES", str(1 << 16))
    c = BithashCodec(0)
    held, ptrs = [], []

    def make(nbytes, offset=0):
        if request.param == "torch":
            t = torch.empty(nbytes + offset, dtype=torch.uint8, pin_memory=True)
            held.append(t)
            return t.numpy()[offset:]
        p = c.L.bhg_malloc_host(c.ctx, nbytes + offset)
        assert p
        ptrs.append(p)
        return np.frombuffer((ctypes.c_uint8 * (nbytes + offset)).from_address(p), np.uint8)[offset:]

    make.codec = c
    yield make
    c.sync()
    for p in ptrs:
        assert c.L.bhg_free_host(c.ctx, p) == 0
    c.close()


both = pytest.mark.parametrize("alloc", ["library", "torch"], indirect=True)


def records(n, codec, seed):
    """Records with gaps, a zero-length handle and one that runs past src; CRCs, some wrong."""
    rng = random.Random(seed)
    buf, hs = bytearray(), []
    for i in range(n):
        buf += rng.randbytes(rng.randrange(4))
        v = rng.choice([rng.randbytes, lambda k: (b"value-%d-" % i * k)[:k]])(rng.choice([0, 1, 64, 1024, 3000]))
        rec = O.record_set(rng.randbytes(rng.choice([0, 7, 32])), (i + 1) << 8 | 1,
                           O.snappy_encode(v) if codec else v, 4)
        hs.append((len(buf), len(rec), 0))
        buf += rec
    h = np.array(hs, dtype=O.HANDLE_DT)
    h["length"][n // 3] = 0
    h["length"][n - 1] += 9
    crc = O.decode_batch(bytes(buf), h, codec=codec)[0]["crc"].copy()
    crc[5::97] ^= 1
    return np.frombuffer(bytes(buf), np.uint8), h, crc


def place(alloc, a, offset=0):
    out = alloc(max(a.nbytes, 1), offset)[:a.nbytes]
    out[:] = a.view(np.uint8).reshape(-1)
    return out.view(a.dtype)


def assert_same(got, exp):
    for f in O.DESC_DT.names:
        bad = np.nonzero(got[f] != exp[f])[0]
        assert bad.size == 0, (f, bad[:8])


@both
@pytest.mark.parametrize("unsorted,n,offset", [(False, 1, 0), (False, 3000, 0), (False, 3000, 5), (True, 2, 0),
                                               (True, 3000, 0), (True, 3000, 13)])
def test_uncompressed(alloc, unsorted, n, offset):
    src, h, crc = records(n, 0, 11 + n)
    if unsorted:
        perm = np.random.default_rng(3).permutation(n) if n > 2 else np.arange(n)[::-1]
        h, crc = h[perm].copy(), crc[perm].copy()
    exp, _, _ = O.decode_batch(src, h, expected_crc=crc)
    for pin_rest in (False, True):              # handles, CRCs and descriptors pageable, then pinned
        hp, cp, out = h, crc, np.zeros(n + 1, DESC_DT)
        if pin_rest:
            hp, cp, out = place(alloc, h, 16), place(alloc, crc, 4), place(alloc, out, 40)
        out.view(np.uint8)[:] = 0xEE
        got, _, _ = alloc.codec.decode_host(place(alloc, src, offset), hp, expected_crc=cp, out_desc=out)
        assert_same(got, exp)
        assert (out[n:].view(np.uint8) == 0xEE).all()


@both
@pytest.mark.parametrize("unsorted", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 8, 15])
def test_snappy(alloc, unsorted, offset):
    src, h, crc = records(2500, 1, 29)
    if unsorted:
        perm = np.random.default_rng(17).permutation(len(h))
        h, crc = h[perm].copy(), crc[perm].copy()
    exp, ev, eo = O.decode_batch(src, h, codec=1, expected_crc=crc)
    total = int(eo[-1])
    vals = alloc(total + 100, offset)
    vals[:] = 0xEE
    got, gv, go = alloc.codec.decode_host(place(alloc, src, offset), h, compressor=1, expected_crc=crc,
                                          out_desc=place(alloc, np.zeros(len(h), DESC_DT)), out_vals=vals)
    assert_same(got, exp)
    assert np.array_equal(go, eo) and gv.tobytes() == ev[:total].tobytes()
    assert (vals[total:] == 0xEE).all()
