"""Learned codes on the CPU: calls of the Python entry points that have to be refused, or have to be safe, whatever the
tensors hold (nothing launches)."""
import pytest
import torch

import yanerf_boot  # noqa: F401
from yanerf_amd import _C


def recorders():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def fake(f):
        def run(x):
            with FakeTensorMode(allow_non_fake_inputs=True):
                return f(x)
        return run

    return {"jit": lambda f: lambda x: torch.jit.trace(f, (x,)), "make_fx": make_fx,
            "pre-dispatch": lambda f: make_fx(f, pre_dispatch=True), "fake": fake}


@pytest.mark.parametrize("how", ["jit", "make_fx", "pre-dispatch", "fake"])
def test_recording_is_refused(how):
    """A recorder sees the allocation of the output and not the kernel, so its replay would return unwritten memory."""
    m, i = _C.torch_ops(), torch.zeros(3, dtype=torch.int64)
    for f in (lambda t: m.dropout(t, 0.5, 0, 0, None), lambda t: m.embedding(t, i, 1.0, None, 0.0, 0, 0, None, -1, 0)):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            recorders()[how](f)(torch.zeros(6, 4))
