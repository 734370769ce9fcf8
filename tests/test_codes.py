"""Learned codes on the CPU: refusals of the Python entry points and of the C ABI (nothing launches), CodeTable's
arguments, and the mask's generator against its published test vectors."""
import ctypes

import numpy as np
import pytest
import torch

import codes_reference as R
import yanerf_boot  # noqa: F401
from yanerf_amd import _C, ops
from yanerf_amd.pipelines.feature_extractors import FEATURE_EXTRACTORS


def test_philox_known_answers():
    """The generator's published vectors (Random123 kat_vectors, philox4x32 10 rounds): all-zero input and the
    digits of pi."""
    z = R.philox_words(0, 1, 0, 0)
    assert [f"{int(w):08x}" for w in z] == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]
    pi = R.philox_words((0x85A308D3 << 32) | 0x243F6A88, 1, (0x299F31D0 << 32) | 0xA4093822,
                        (0x03707344 << 32) | 0x13198A2E)
    assert [f"{int(w):08x}" for w in pi] == ["d16cfe09", "94fdcceb", "5001e420", "24126ea1"]


def test_entry_points_refuse_host_tensors():
    with pytest.raises(RuntimeError, match="HIP kernels"):
        ops.dropout(torch.zeros(4), 0.5)
    with pytest.raises(RuntimeError, match="HIP kernels"):
        ops.embedding(torch.zeros(4, 2), torch.zeros(3, dtype=torch.int64))


def test_torch_binding_loads_with_the_sources_build_id():
    m = _C.torch_ops()
    assert m.build_id() == _C.source_id(_C.TORCH_SOURCES)


def test_torch_binding_refusals():
    """The native checks, on host tensors below the Python entry points: nothing launches."""
    m = _C.torch_ops()
    t, i = torch.zeros(6, 4), torch.zeros(3, dtype=torch.int64)
    for args, exc, msg in [((t[0], i), ValueError, "V, D"), ((t.double(), i), TypeError, "Double"),
                           ((t, i.short()), TypeError, "int32 or int64"), ((t[:0], i), IndexError, "empty table")]:
        with pytest.raises(exc, match=msg):
            m.embedding(*args, 1.0, None, 0.0, 0, 0, None, -1, 0)
    for kw, msg in [(dict(pad=6), "padding_idx"), (dict(pad=-7), "padding_idx"), (dict(scale=float("inf")), "scale"),
                    (dict(p=1.5), "probability"), (dict(p=float("nan")), "probability"), (dict(base=t), "rng_base")]:
        a = dict(scale=1.0, pad=None, p=0.0, base=None)
        a.update(kw)
        with pytest.raises(ValueError, match=msg):
            m.embedding(t, i, a["scale"], a["pad"], a["p"], 0, 0, a["base"], -1, 0)
    with pytest.raises(TypeError):
        m.dropout(i, 0.5, 0, 0, None)
    with pytest.raises(ValueError, match="probability"):
        m.dropout(t, -0.5, 0, 0, None)
    with pytest.raises(ValueError, match="rng_base"):
        m.dropout(t, 0.5, 0, 0, torch.zeros(1, dtype=torch.int64))


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    m = _C.torch_ops()
    with fwd.dual_level():
        t = fwd.make_dual(torch.zeros(6, 4), torch.ones(6, 4))
        with pytest.raises(RuntimeError, match="forward-mode"):
            m.embedding(t, torch.zeros(3, dtype=torch.int64), 1.0, None, 0.0, 0, 0, None, -1, 0)
        with pytest.raises(RuntimeError, match="forward-mode"):
            m.dropout(t, 0.5, 0, 0, None)


D16 = ctypes.c_void_p(16)


def err():
    return _C.lib().yanerf_last_error().decode()


def test_dropout_c_refusals():
    L = _C.lib()
    for args, msg in [((D16, 3, 8, 0.5), "type"), ((D16, 0, -1, 0.5), "range"), ((D16, 0, (1 << 36) + 1, 0.5), "range"),
                      ((D16, 0, 8, -0.1), "probability"), ((D16, 0, 8, 1.5), "probability"),
                      ((D16, 0, 8, float("nan")), "probability"), ((None, 0, 8, 0.5), "null")]:
        assert L.yanerf_dropout(*args, 1, 2, None, None, D16, None) == 1
        assert msg in err(), args
    assert L.yanerf_dropout(D16, 0, 8, 0.5, 1, 2, None, None, None, None) == 1 and "null" in err()
    assert L.yanerf_dropout(None, 0, 0, 0.5, 1, 2, None, None, None, None) == 0  # nothing to do


def fwd(**kw):
    a = dict(table=D16, tt=0, stride=4, ids=D16, ib=8, N=3, V=5, D=4, scale=1.0, p=0.0, out=D16, ot=0)
    a.update(kw)
    return _C.lib().yanerf_embedding_forward(a["table"], a["tt"], a["stride"], a["ids"], a["ib"], a["N"], a["V"], a["D"],
                                             a["scale"], a["p"], 1, 2, None, None, a["out"], a["ot"], None, None)


def bwd(**kw):
    a = dict(g=D16, gt=0, ids=D16, ib=8, N=3, V=5, D=4, pad=-1, scale=1.0, p=0.0, grad=D16, tt=0, ws=D16)
    a.update(kw)
    return _C.lib().yanerf_embedding_backward(a["g"], a["gt"], a["ids"], a["ib"], a["N"], a["V"], a["D"], a["pad"],
                                              a["scale"], a["p"], 1, 2, None, a["grad"], a["tt"], a["ws"], None)


@pytest.mark.parametrize("call", [fwd, bwd])
@pytest.mark.parametrize("kw,msg", [
    (dict(tt=7), "type"), (dict(ib=2), "ids of 2"), (dict(N=-1), "negative"), (dict(V=-1), "negative"),
    (dict(D=-1), "negative"), (dict(N=1 << 31), "2^31"), (dict(V=1 << 31), "2^31"), (dict(N=1 << 30, D=1 << 9), "2^36"), (dict(D=(1 << 24) + 1), "2^24"),
    (dict(V=1 << 30, D=1 << 9), "2^36"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(p=1.01), "probability"), (dict(p=float("nan")), "probability"), (dict(ids=None), "null")])
def test_embedding_c_refusals(call, kw, msg):
    assert call(**kw) == 1
    assert msg in err(), (kw, err())


def test_embedding_c_refusals_of_one_direction():
    for kw, msg in [(dict(table=None), "null"), (dict(out=None), "null"), (dict(V=0), "empty table"),
                    (dict(ot=-1), "type"), (dict(stride=-4), "stride")]:
        assert fwd(**kw) == 1 and msg in err(), kw
    for kw, msg in [(dict(g=None), "null"), (dict(grad=None), "null"), (dict(ws=None, N=5000), "null"), (dict(gt=9), "type"),
                    (dict(ws=ctypes.c_void_p(24)), "16 bytes"),
                    (dict(pad=5), "padding_idx"), (dict(pad=-2), "padding_idx")]:
        assert bwd(**kw) == 1 and msg in err(), kw
    assert fwd(N=0, table=None, ids=None, out=None) == 0 and fwd(D=0, table=None, ids=None, out=None) == 0
    assert bwd(V=0, grad=None) == 0 and bwd(D=0, grad=None) == 0
    L = _C.lib()
    assert L.yanerf_embedding_bwd_workspace_bytes(-1, 5, 4) == -1
    assert L.yanerf_embedding_bwd_workspace_bytes(1 << 31, 5, 4) == -1
    assert L.yanerf_embedding_bwd_workspace_bytes(0, 5, 4) == 0
    assert L.yanerf_embedding_bwd_workspace_bytes(1000, 5, 4) == 0  # one launch, nothing kept between
    assert L.yanerf_embedding_bwd_workspace_bytes(5000, 5, 4) > 0


def test_workspace_query_over_the_range():
    """Every allowed size has a plan, from one id, row and column to the largest, and the workspace stays within what the
    pairs (16 bytes an id), a few copies of g's rows in fp32 and the smaller tables need."""
    L = _C.lib()
    for n in (1, 2, 4096, 4097, 16384, 16385, 131072, 10 ** 6, 2 ** 31 - 1):
        for v in (1, 2, 17, 100, 128, 129, 1023, 1024, 50000, 10 ** 6, 2 ** 31 - 1):
            for d in (1, 2, 3, 7, 8, 9, 48, 65, 1000, 1024, 1001, 2 ** 24 - 1, 2 ** 24):
                if n * d > 2 ** 36 or v * d > 2 ** 36:
                    assert L.yanerf_embedding_bwd_workspace_bytes(n, v, d) == -1
                    continue
                b = L.yanerf_embedding_bwd_workspace_bytes(n, v, d)
                assert (0 if n <= 4096 else 1) <= b <= 64 * n + 16 * n * d + 2 ** 16 * d + 2 ** 26, (n, v, d, b)


def test_code_table_arguments():
    build = lambda **kw: FEATURE_EXTRACTORS.build(dict(type="CodeTable", **kw))
    m = build(num_codes=5, latent_dim=2, padding_idx=-1)
    assert m.table.shape == (5, 2) and not m.table[-1].any() and m.table[:4].abs().sum() > 0
    for kw, exc in [(dict(num_codes=0, latent_dim=2), ValueError), (dict(num_codes=2, latent_dim=0), ValueError),
                    (dict(num_codes=2, latent_dim=2, dropout=1.5), ValueError),
                    (dict(num_codes=2, latent_dim=2, padding_idx=2), ValueError)]:
        with pytest.raises(exc):
            build(**kw)
    with pytest.raises(KeyError):
        m(other=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(IndexError):
        m(image_ids=torch.tensor([5]))
    with pytest.raises(IndexError):
        m(image_ids=torch.tensor([-1]))
    with pytest.raises(TypeError):
        m(image_ids=torch.tensor([1.0]))
    with pytest.raises(ValueError):
        m(image_ids=torch.tensor([[1]]))


def test_fused_trainer_refuses_codes():
    """The fused trainer runs no feature extractor: a conditional config is refused and not trained without its codes."""
    from yanerf_amd.train import NeRFTrainer
    from yanerf_amd.utils.config import Config
    cfg = Config.fromfile(str(yanerf_boot.PKG_DIR / "configs/nerf/lego.yml")).pipeline
    cfg.model.latent_dim = 4
    cfg.feature_extractor = [dict(type="CodeTable", num_codes=100, latent_dim=4)]
    with pytest.raises(NotImplementedError, match="latent_dim"):
        NeRFTrainer(cfg, device="cpu")


def test_reference_mask_rate():
    """The keep rate of the definition's mask: 2^16 draws at p = 0.3, five standard deviations."""
    k = R.keep_mask(1 << 16, 0.3, 7, 9)
    assert abs(k.mean() - 0.7) < 5 * np.sqrt(0.21 / k.size)
