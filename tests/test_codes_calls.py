"""Learned codes on the CPU: calls of the Python entry points that have to be refused, or have to be safe, whatever the
tensors hold (nothing launches)."""
import ctypes
import subprocess
import weakref

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


def test_first_use_of_an_id_flag_by_two_threads(monkeypatch):
    """Two threads that make their first lookup at once: each address that a lookup gets belongs to memory that stays (here to a
    tensor that its thread still holds while another thread makes its own)."""
    import threading
    from types import SimpleNamespace
    from yanerf_amd import ops
    made, meet = [], threading.Barrier(2)

    def zeros(*shape, **kw):
        t = torch.full(shape, 0, dtype=kw["dtype"])
        made.append(weakref.ref(t))
        meet.wait(10)  # both threads have found none
        return t

    fake = SimpleNamespace(**{k: getattr(torch, k) for k in ("int32", "empty")}, zeros=zeros,
                           cuda=SimpleNamespace(current_stream=lambda dev: SimpleNamespace(synchronize=lambda: None)))
    monkeypatch.setattr(ops, "torch", fake)
    held, done, got = [], threading.Barrier(3), []

    def work():
        got.append(ops._id_flag(0, own=True))
        got.append(ops._id_flag(0, own=True))
        done.wait(10)
        done.wait(10)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    done.wait(10)
    held = [r().data_ptr() for r in made if r() is not None]
    done.wait(10)
    for t in threads:
        t.join()
    assert len(got) == 4 and len(set(got)) == 2 and set(got) == set(held)


def test_flag_c_refusals():
    L = _C.lib()
    assert L.yanerf_id_flag(None) == 1 and b"null" in L.yanerf_last_error()
    p, q = ctypes.c_void_p(16), ctypes.c_void_p(32)
    for a in ((None, p), (p, None), (p, p)):
        assert L.yanerf_flag_take(*a, None) == 1 and b"pointers" in L.yanerf_last_error()


def test_binding_of_another_torch_is_refused(monkeypatch, tmp_path):
    """The binding uses torch's C++ ABI: one built against another version does not run, whatever its sources were."""
    assert _C.torch_ops().torch_version() == torch.__version__
    monkeypatch.setattr(_C, "_torch_ops", None)
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "1.0.0")
        with pytest.raises(_C.HipError, match="built against torch"):
            _C.torch_ops()
    with monkeypatch.context() as m:
        other = tmp_path / "_codes_torch.so"
        other.write_bytes(b"not a library of this torch")
        m.setattr(_C, "TORCH_LIB_PATH", other)
        with pytest.raises(_C.HipError, match="does not load"):
            _C.torch_ops()
    assert _C.torch_ops().torch_version() == torch.__version__


def test_the_library_builds_without_torch():
    """make's default is the C ABI's library: no step of it runs Python, g++ or names torch; `all` builds the binding too."""
    csrc = _C.PKG / "csrc"
    plan = lambda *goal: subprocess.run(["make", "-n", "-B", "-C", str(csrc), "PYTHON=false", *goal], check=True,
                                        capture_output=True, text=True).stdout
    assert "libyanerf_hip.so" in plan() and "torch" not in plan() and "g++" not in plan()
    assert "libyanerf_hip.so" in plan("all") and "_codes_torch.so" in plan("all")


@pytest.mark.parametrize("scale,p", [(3.5e38, 0.0), (-1e39, 0.0), (1e300, 0.0), (3e38, 0.5), (1e308, 0.99), (1e-38, 0.0),
                                     (-1e-45, 0.0), (1e-320, 0.5)])
def test_factors_outside_fp32_are_refused(scale, p):
    """A factor that fp32 holds as infinity makes a row of zeros NaN, one below its normal numbers loses its digits."""
    L, D16, m = _C.lib(), ctypes.c_void_p(16), _C.torch_ops()
    assert L.yanerf_embedding_forward(D16, 0, 4, D16, 8, 3, 5, 4, scale, p, 1, 2, None, None, D16, 0, None, None) == 1
    assert b"factor" in L.yanerf_last_error()
    assert L.yanerf_embedding_backward(D16, 0, D16, 8, 3, 5, 4, -1, scale, p, 1, 2, None, D16, 0, D16, None) == 1
    assert b"factor" in L.yanerf_last_error()
    with pytest.raises(ValueError, match="factor"):
        m.embedding(torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64), scale, None, p, 0, 0, None, -1, 0)


def test_rng_used_is_not_rng_base():
    """One workgroup would write the offset while the others still read the base."""
    L, D16, b, u = _C.lib(), ctypes.c_void_p(16), ctypes.c_void_p(64), ctypes.c_void_p(128)
    assert L.yanerf_dropout(D16, 0, 8, 0.5, 1, 2, b, b, D16, None) == 1 and b"rng_used" in L.yanerf_last_error()
    assert L.yanerf_embedding_forward(D16, 0, 4, D16, 8, 3, 5, 4, 1.0, 0.5, 1, 2, b, b, D16, 0, None, None) == 1
    assert b"rng_used" in L.yanerf_last_error()
    assert L.yanerf_dropout(D16, 0, 0, 0.5, 1, 2, b, u, D16, None) == 0 and L.yanerf_dropout(D16, 0, 0, 0.5, 1, 2, None, None, D16, None) == 0


def test_module_stream_and_seeds(monkeypatch):
    """The default masks' stream as ops.dropout describes it: another seed starts it anew, the same seed goes on, set_state
    starts it anew at the same seed."""
    from yanerf_amd import ops
    monkeypatch.setattr(ops, "_capturing", lambda dev: False)
    before, seed = ops.RNG.get_state(), torch.initial_seed()
    try:
        torch.manual_seed(123)
        ops.RNG.set_state((None, 0))
        assert [ops._mask_rng("dropout", 0.5, None, None, 100, 0) for _ in range(2)] == [(123, 0), (123, 100)]
        torch.manual_seed(123)
        assert ops._mask_rng("dropout", 0.5, None, None, 100, 0) == (123, 200)
        torch.manual_seed(124)
        assert ops._mask_rng("dropout", 0.5, None, None, 100, 0) == (124, 0)
        torch.manual_seed(123)
        assert ops._mask_rng("dropout", 0.5, None, None, 100, 0) == (123, 0)
        ops.RNG.set_state((None, 0))
        assert ops._mask_rng("dropout", 0.5, None, None, 100, 0) == (123, 0)
        assert ops._mask_rng("dropout", 0.5, (-1, 2 ** 64 + 7), None, 100, 0) == (2 ** 64 - 1, 7)
        assert ops.RNG.get_state() == (123, 100)
    finally:
        torch.manual_seed(seed)
        ops.RNG.set_state(before)


def test_identity_mapper_passes_on():
    """Without dropout, and with it in evaluation mode, the mapper is the reference's: what it is given comes back."""
    from yanerf_amd.pipelines.feature_extractors import FEATURE_EXTRACTORS
    codes = torch.ones(2, 4)
    m = FEATURE_EXTRACTORS.build(dict(type="IdentityMapper"))
    out = m(global_codes=codes, other=3)
    assert out["global_codes"] is codes and out["other"] == 3 and m() == {} and not m.state_dict()
    m = FEATURE_EXTRACTORS.build(dict(type="IdentityMapper", dropout=0.5))
    assert m(other=3, global_codes=None) == {"other": 3, "global_codes": None}
    with pytest.raises(RuntimeError, match="HIP kernels"):
        m(global_codes=codes)
    assert m.eval()(global_codes=codes)["global_codes"] is codes
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            FEATURE_EXTRACTORS.build(dict(type="IdentityMapper", dropout=p))


def test_recorders_leave_no_id_flag():
    """A thread's first checked lookup under a recorder is refused before the recorder's tensor becomes the thread's flag."""
    import threading
    from torch._subclasses.fake_tensor import FakeTensorMode
    from yanerf_amd import ops
    seen = []

    def work():
        with FakeTensorMode(allow_non_fake_inputs=True):
            try:
                ops._id_flag(0, own=True)
            except RuntimeError as e:
                seen.append(str(e))
        seen.append(dict(ops._OWN_FLAGS.__dict__))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert "cannot be recorded" in seen[0] and seen[1:] == [{}]
