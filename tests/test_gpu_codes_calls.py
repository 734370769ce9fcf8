"""Learned codes on the GPU: calls that the operators allow or refuse whatever their sizes are."""
import numpy as np
import pytest
import torch

import codes_reference as R
import yanerf_boot  # noqa: F401
from test_gpu_codes import BF16, DEV, F16, F32, NAME, TYPES, ops, rand, some_ids  # noqa: F401

pytestmark = pytest.mark.gpu


def captured(f, before=None):
    """(graph, f()) of a capture of f on a side stream; `before` runs eagerly first."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    if before is not None:
        with torch.cuda.stream(s):
            before()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = f()
    return g, out


# ------------------------------------------------------------------------------------------- recorders
def test_recording_is_refused(ops):
    """A recorder sees the allocation of the output and not the kernel, so its replay would return unwritten memory."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, t, i = rand(64, 16), rand(64, 16), some_ids(50, 64)
    for f in (lambda t: ops.dropout(t, 0.5, rng=(1, 2)), lambda t: ops.embedding(t, i, check=False)):
        for record in (lambda f: torch.jit.trace(f, (x,)), lambda f: make_fx(f)(x), lambda f: make_fx(f, pre_dispatch=True)(x),
                       lambda f: make_fx(f, tracing_mode="fake")(x)):
            with pytest.raises(RuntimeError, match="cannot be recorded"):
                record(f)
        leaf = t.clone().requires_grad_()
        y = f(leaf)
        with pytest.raises(RuntimeError, match="cannot be recorded"):  # the backward of a graph made before
            make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True)[0])(torch.ones_like(y))


def test_watching_is_allowed(ops):
    """A dispatch mode that only watches gets the eager results."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    t, i = rand(64, 16).requires_grad_(), some_ids(50, 64)
    f = lambda: ops.dropout(ops.embedding(t, i, dropout=0.25, rng=(1, 2), check=False), 0.5, rng=(1, 3))
    want = f()
    (gw,) = torch.autograd.grad(want.sum(), t)
    with Watch():
        y = f()
        (gt,) = torch.autograd.grad(y.sum(), t)
    assert torch.equal(y, want) and torch.equal(gt, gw)
