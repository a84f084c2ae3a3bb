"""Page-locking of existing host memory: a refusal answers False and leaves no HIP error for the next call to report."""
import pytest
import torch


def test_host_register_refuses_nonsense(hiplib):
    assert hiplib.pg_host_register(None, 64) == -1
    buf = torch.zeros(16)
    assert hiplib.pg_host_register(buf.data_ptr(), 0) == -1


@pytest.mark.gpu
def test_host_register_leaves_no_error_behind(dev, hiplib):
    from pagraph_amd import _lib as L
    from pagraph_amd.storage.storage import huge_page_tensor
    t, ok = huge_page_tensor((4096, 64))                      # registered, or refused by the machine: both are fine
    assert isinstance(ok, bool)
    out = torch.full((128,), 7, dtype=torch.int32, device=dev)
    # the library's launches check the runtime's last error
    L.check(hiplib.pg_slot_map_reset(L.ptr(out), out.numel(), L.stream_ptr()), "pg_slot_map_reset")
    assert (out == -1).all()
