"""bench.py's end-to-end leg (host buffers) is optional: whatever the host refuses there, the
measured line is kept, with the reason in the leg's own field."""
import sys

import pytest
import torch

import bench
from bitalosdb_amd import _lib as B


def test_a_refusal_is_recorded():
    def refused():
        raise B.BhgError("bhg_decode_batch_host failed (-2): invalid argument")
    out = {"value": 4355.1, "valid": True}
    bench.host_leg(out, refused)
    assert out["value"] == 4355.1 and out["valid"] is True
    assert out["e2e_host"]["value"] is None and "invalid argument" in out["e2e_host"]["error"]
    bench.host_leg(out, lambda: {"value": 50.0})
    assert out["e2e_host"] == {"value": 50.0}


def test_a_mistake_in_the_leg_is_not_hidden():
    with pytest.raises(TypeError):
        bench.host_leg({}, lambda: None + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("measure", ["c2", "c3"])
@pytest.mark.parametrize("refuse", [False, True])
def test_measured_line(measure, refuse, monkeypatch):
    from bitalosdb_amd.codec import BithashCodec
    monkeypatch.setattr(sys, "argv", ["bench.py", "--blocks", "20000", "--steps", "3", "--warmup", "1", "--ramp-ms", "0",
                                      "--no-cpu", "--no-traffic"])
    a = bench.parse()
    dev = torch.device("cuda", 0)
    codec = BithashCodec(0)
    if refuse:
        def page_lock(arr):
            raise B.BhgError("bhg_host_register failed (-2): invalid argument")

        def decode_host(*args, **kw):
            raise B.BhgError("bhg_decode_batch_host failed (-2): invalid argument")
        monkeypatch.setattr(codec, "host_register", page_lock)
        monkeypatch.setattr(codec, "decode_host", decode_host)
    with torch.cuda.stream(codec.stream):
        if measure == "c2":
            out = bench.c2_measure(a, 1, 0, 0, dev, codec, with_extras=True)
        else:
            out = bench.c3_measure(a, 1, 0, 0, dev, codec, "dict", extras=True)
    codec.close()
    assert out["value"] > 0 and out["valid"] is True and out["status_ok_blocks"] == 20000
    e = out["e2e_host"]
    if refuse:
        assert e["value"] is None and "invalid argument" in e["error"]
    else:
        assert e["value"] > 0 and e["pageable"] > 0 and e["matches_device_path"] is True
