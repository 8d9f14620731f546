"""Host side of the calls, on a machine without a GPU: what they refuse before any
launch, what they keep alive until one is made, and what importing needs."""
import pytest
import torch

from parakeet_b200 import ops
from parakeet_b200.modules.subsample import ConvSubsampling


class NoLaunch:
    """A library whose calls fail the test."""

    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(f"{name} was called")
        return call


@pytest.fixture
def no_launch(monkeypatch):
    """A machine with a GPU, as far as torch's host calls tell."""
    import parakeet_b200.modules.subsample as sub
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    for module in (ops, sub):
        monkeypatch.setattr(module, "lib", NoLaunch)


def test_host_tensors_are_refused_before_a_launch(no_launch):
    """A kernel given host pointers would fault."""
    a, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, 64, dtype=torch.bfloat16)
    ops._gemm_error.pop(a.device, None)
    with pytest.raises(ValueError, match="cuda device"):
        ops.gemm(a, w)
    sub = ConvSubsampling(64, 64, 80, 8)
    with pytest.raises(ValueError, match="cuda device"):
        sub.forward_stream(torch.zeros(1, 80, 16))
    ops._gemm_error.pop(a.device, None)
