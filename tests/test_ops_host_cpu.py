"""Host side of the calls, on a machine without a GPU: what they refuse before any
launch, what they keep alive until one is made, and what importing needs."""
import subprocess
import sys
import weakref

import pytest
import torch

from conftest import REPO
from parakeet_b200 import adapters, ops, tokens
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


def test_imports_where_torch_has_no_cuda_bindings():
    code = ("import sys, torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            f"sys.path[:0] = [{REPO!r}, {REPO + '/parakeet-streaming_b200'!r}]\n"
            "import parakeet_b200\n"
            "from parakeet_b200.ops import gemm_supported, layer_norm\n"
            "a = torch.zeros(4, 64)\n"
            "assert not gemm_supported(a, a)\n"
            "layer_norm(a, torch.nn.LayerNorm(64))\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_attention_keeps_its_workspace_until_it_has_launched(monkeypatch):
    """The call's two launches share it.  Given back before them, it could go to a call
    that another thread makes on the same stream, between the two."""
    made = []

    class Block:
        """A step's block that remembers what was allocated beside it."""

        def new_empty(self, n):
            t = torch.empty(n)
            made.append((weakref.ref(t), t.data_ptr()))
            return t

        def data_ptr(self):
            return 64

    launches = []

    def launch(device, fn, *args):
        ref, ptr = made[-1]
        assert ref() is not None and ptr in args
        launches.append(fn)

    monkeypatch.setattr(tokens, "_launch", launch)
    monkeypatch.setattr(tokens, "_stream", lambda device: 0)
    pool = object.__new__(tokens.TokenKVPool)
    pool.dtype, pool.device, pool._index = torch.float32, torch.device("cpu"), -1
    pool.num_heads, pool.num_kv_heads, pool.head_dim, pool._h = 2, 1, 64, None
    pool._lib = NoLaunch()
    step = tokens.TokenStep(pool, Block(), 1, 3, False, (0,) * 6, 4096)
    pool.attention(0, torch.zeros(3, 2, 64), step)
    assert len(launches) == 1 and len(made) == 1


@pytest.mark.parametrize("who", ["gemm", "adapters"])
def test_a_devices_error_word_is_one_whoever_makes_it_first(monkeypatch, who):
    """Two threads' first calls: the word that one of them gives to its kernel is the one
    that stays, not a tensor that is freed under the kernel."""
    device = torch.device("cpu")
    monkeypatch.setattr(ops, "_gemm_error", {})
    monkeypatch.setattr(adapters, "_gemm_error", ops._gemm_error)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    zeros, others = torch.zeros, []

    def zeros_while_another_thread_is_faster(*shape, **kw):
        if not others:
            others.append(zeros(1, dtype=torch.int32))
            ops._gemm_error[device] = others[0]
        return zeros(*shape, **kw)

    monkeypatch.setattr(torch, "zeros", zeros_while_another_thread_is_faster)
    if who == "adapters":
        given = adapters._error_word(device)
    else:
        calls = []
        monkeypatch.setattr(ops, "_stream", lambda device: 0)
        monkeypatch.setattr(ops, "lib", lambda: type("L", (), {
            "pk_gemm_bf16": staticmethod(lambda *args: calls.append(args) or 0)}))
        a = torch.ones(4, 64, dtype=torch.bfloat16)
        ops.gemm(a, torch.ones(64, 64, dtype=torch.bfloat16))
        given = calls[0][-2]
    assert ops._gemm_error[device] is others[0] and given == others[0].data_ptr()
