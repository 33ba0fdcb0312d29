"""The 8-bit product and the orthogonalised update without a GPU: what the entry points refuse on the host
before any launch, and what the Python layer refuses before it calls them."""
import ctypes
import math

import pytest
import torch

from yolo_amd import Int8Linear, Muon, YOLOv1Head, _lib, linear_i8, muon_step, orthogonalize, quantize_rows

FAKE = 0x1000  # never dereferenced: every call below fails its host-side checks first
BIG = 1 << 40


def _linear(**kw):
    a = dict(x=FAKE, xd=_lib.YH_F32, ldx=64, sx=None, w=FAKE, ldw=64, sw=FAKE, bias=None, y=FAKE, yd=_lib.YH_F32, ldy=800,
             M=600, N=800, K=64, ws=FAKE, nbytes=BIG)
    a.update(kw)
    return _lib.load().yh_linear_i8(a["x"], a["xd"], a["ldx"], a["sx"], a["w"], a["ldw"], a["sw"], a["bias"], a["y"], a["yd"],
                                    a["ldy"], a["M"], a["N"], a["K"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("kw,rc", [
    (dict(K=0), _lib.YH_ERR_SHAPE),
    (dict(K=131072, ldx=131072, ldw=131072), _lib.YH_ERR_SHAPE),
    (dict(M=-1), _lib.YH_ERR_SHAPE),
    (dict(M=1 << 22), _lib.YH_ERR_SHAPE),
    (dict(ldx=63), _lib.YH_ERR_SHAPE),
    (dict(ldw=48), _lib.YH_ERR_SHAPE),
    (dict(ldy=799), _lib.YH_ERR_SHAPE),
    (dict(xd=4), _lib.YH_ERR_ARG),
    (dict(yd=_lib.YH_I8), _lib.YH_ERR_ARG),
    (dict(sx=FAKE), _lib.YH_ERR_ARG),                    # scales for an x that is not int8
    (dict(xd=_lib.YH_I8), _lib.YH_ERR_ARG),              # int8 without them
    (dict(x=0), _lib.YH_ERR_NULL),
    (dict(w=0), _lib.YH_ERR_NULL),
    (dict(sw=0), _lib.YH_ERR_NULL),
    (dict(y=0), _lib.YH_ERR_NULL),
    (dict(ws=0), _lib.YH_ERR_WORKSPACE),
    (dict(nbytes=8), _lib.YH_ERR_WORKSPACE),
    (dict(w=FAKE + 8), _lib.YH_ERR_ALIGN),
    (dict(ldw=72), _lib.YH_ERR_ALIGN),
    (dict(ws=FAKE + 16), _lib.YH_ERR_ALIGN),
    (dict(bias=FAKE + 2), _lib.YH_ERR_ALIGN),
    (dict(M=0, x=0, y=0), 0),
    (dict(N=0, w=0, y=0), 0),
])
def test_linear_i8_argument_errors(kw, rc):
    assert _linear(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(K=0), _lib.YH_ERR_SHAPE), (dict(ldx=99), _lib.YH_ERR_SHAPE), (dict(ldq=99), _lib.YH_ERR_SHAPE),
    (dict(xd=_lib.YH_I8), _lib.YH_ERR_ARG), (dict(x=0), _lib.YH_ERR_NULL), (dict(scale=0), _lib.YH_ERR_NULL),
    (dict(ldq=120), _lib.YH_ERR_ALIGN), (dict(q=FAKE + 4), _lib.YH_ERR_ALIGN), (dict(rows=0, x=0), 0),
])
def test_quantize_rows_argument_errors(kw, rc):
    a = dict(x=FAKE, xd=_lib.YH_BF16, ldx=100, q=FAKE, ldq=112, scale=FAKE, rows=3, K=100)
    a.update(kw)
    assert _lib.load().yh_quantize_rows(a["x"], a["xd"], a["ldx"], a["q"], a["ldq"], a["scale"], a["rows"], a["K"], None) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(rows=0), _lib.YH_ERR_SHAPE), (dict(rows=32769, cols=32769, ldg=32769, ldo=32769), _lib.YH_ERR_SHAPE),
    (dict(cols=(1 << 24) + 1, ldg=1 << 25, ldo=1 << 25), _lib.YH_ERR_SHAPE), (dict(count=65536), _lib.YH_ERR_SHAPE),
    (dict(ldg=15), _lib.YH_ERR_SHAPE), (dict(ldo=15), _lib.YH_ERR_SHAPE), (dict(count=2, os=127), _lib.YH_ERR_SHAPE),
    (dict(gd=_lib.YH_I8), _lib.YH_ERR_ARG), (dict(od=7), _lib.YH_ERR_ARG), (dict(steps=0), _lib.YH_ERR_ARG),
    (dict(steps=65), _lib.YH_ERR_ARG), (dict(eps=-1.0), _lib.YH_ERR_ARG), (dict(eps=math.nan), _lib.YH_ERR_ARG),
    (dict(a=math.inf), _lib.YH_ERR_ARG), (dict(g=0), _lib.YH_ERR_NULL), (dict(out=0), _lib.YH_ERR_NULL),
    (dict(ws=0), _lib.YH_ERR_WORKSPACE), (dict(nbytes=64), _lib.YH_ERR_WORKSPACE), (dict(g=FAKE + 2), _lib.YH_ERR_ALIGN),
    (dict(ws=FAKE + 64), _lib.YH_ERR_ALIGN), (dict(count=0, g=0), 0),
])
def test_orthogonalize_argument_errors(kw, rc):
    a = dict(g=FAKE, gd=_lib.YH_F32, gs=128, ldg=16, out=FAKE, od=_lib.YH_BF16, os=128, ldo=16, count=1, rows=8, cols=16,
             a=3.0, eps=1e-7, steps=5, ws=FAKE, nbytes=BIG)
    a.update(kw)
    assert _lib.load().yh_orthogonalize(a["g"], a["gd"], a["gs"], a["ldg"], a["out"], a["od"], a["os"], a["ldo"], a["count"],
                                        a["rows"], a["cols"], a["a"], -4.0, 2.0, a["steps"], a["eps"], a["ws"], a["nbytes"],
                                        None) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(count=33), _lib.YH_ERR_SHAPE), (dict(count=-1), _lib.YH_ERR_SHAPE), (dict(rows=0), _lib.YH_ERR_SHAPE),
    (dict(pd=_lib.YH_I8), _lib.YH_ERR_ARG), (dict(lr=math.nan), _lib.YH_ERR_ARG), (dict(scale=math.inf), _lib.YH_ERR_ARG),
    (dict(steps=0), _lib.YH_ERR_ARG), (dict(params=None), _lib.YH_ERR_NULL), (dict(first=0), _lib.YH_ERR_NULL),
    (dict(first=FAKE + 2), _lib.YH_ERR_ALIGN), (dict(nbytes=64), _lib.YH_ERR_WORKSPACE), (dict(ws=FAKE + 64), _lib.YH_ERR_ALIGN),
    (dict(count=0), 0),
])
def test_muon_step_argument_errors(kw, rc):
    a = dict(count=1, rows=8, cols=16, pd=_lib.YH_F32, lr=0.1, scale=1.0, steps=5, first=FAKE, params=1, ws=FAKE, nbytes=BIG)
    a.update(kw)
    lists = (ctypes.c_void_p * 33)(*([a["first"]] + [FAKE] * 32))
    assert _lib.load().yh_muon_step(lists if a["params"] else None, a["pd"], lists, _lib.YH_F32, lists, a["count"], a["rows"],
                                    a["cols"], a["lr"], 0.9, 1, 0.0, a["scale"], 3.0, -4.0, 2.0, a["steps"], 1e-7, a["ws"],
                                    a["nbytes"], None) == rc


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.yh_linear_i8_workspace_bytes(_lib.YH_F32, 0, 8, 64) == 0 and lib.yh_linear_i8_workspace_bytes(_lib.YH_F32, 4, 8, 0) == 0
    assert lib.yh_linear_i8_workspace_bytes(_lib.YH_I8, 600, 800, 200) >= 600 * 256
    assert lib.yh_linear_i8_workspace_bytes(_lib.YH_F32, 3, 8, 200) == 0          # quantised on the way
    assert lib.yh_linear_i8_workspace_bytes(_lib.YH_F32, 30, 8, 4096) >= 30 * 4096 + 30 * 4
    assert lib.yh_orthogonalize_workspace_bytes(0, 8, 8) == 0 and lib.yh_orthogonalize_workspace_bytes(1, 0, 8) == 0
    assert lib.yh_orthogonalize_workspace_bytes(1, 64, 147) == lib.yh_orthogonalize_workspace_bytes(1, 147, 64) > 0


def test_python_layer_refuses():
    x, w, s = torch.zeros(2, 64), torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3)
    with pytest.raises(ValueError, match="GPU"):
        linear_i8(x, w, s)
    with pytest.raises(ValueError, match="GPU"):
        quantize_rows(x)
    with pytest.raises(ValueError, match="gradient"):
        linear_i8(x.clone().requires_grad_(True), w, s)
    with pytest.raises(ValueError, match="GPU"):
        orthogonalize(x)
    with pytest.raises(ValueError, match="GPU"):
        muon_step([x], [x.clone()], [x.clone()], lr=0.1)
    with pytest.raises(ValueError, match="two axes"):
        muon_step([x[0]], [x[0]], [x[0]], lr=0.1)
    with pytest.raises(ValueError, match="1 params, 0 grads"):
        muon_step([x], [], [x], lr=0.1)
    muon_step([], [], [], lr=0.1)
    with pytest.raises(ValueError, match="two or more axes"):
        Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="steps"):
        Muon([torch.nn.Parameter(x)], steps=0)
    layer = Int8Linear(w, s)
    assert layer.weight.shape == (3, 64) and layer.weight.stride(0) == 128
    with pytest.raises(ValueError, match="output channels"):
        YOLOv1Head().postprocess_linear(x, layer)


@pytest.mark.parametrize("coeffs,steps", [((3.0, -4.0, 2.0), 5), ((2.0, 2.0, 1.0), 2), ((121.0, 0.0, 0.0), 1), ((1e30, 0.0, 0.0), 1),
                                          ((0.0, 500.0, -500.0), 1), ((1.0, 121.0, 0.0), 1), ((100.0, -99.0, 0.0), 2),
                                          ((3e38, 3e38, 3e38), 64)])
def test_coefficients_that_leave_the_range_are_refused(coeffs, steps):
    """In [0, 1] the singular values of these reach s^2, |b s^2 + c s^4| or s^2 |a + b s^2 + c s^4| past 120 before a step;
    shown here on a grid."""
    s, worst = torch.linspace(0, 1, 20001, dtype=torch.float64), 0.0
    a, b, c = coeffs
    for _ in range(steps):
        z = s * s
        r = b * z + c * z * z
        worst = max(worst, z.max().item(), r.abs().max().item(), (z * (a + r)).abs().max().item())
        s = (s * (a + r)).clamp(-1e9, 1e9)
    lib, lists = _lib.load(), (ctypes.c_void_p * 1)(FAKE)
    assert worst > 120
    assert lib.yh_orthogonalize(FAKE, _lib.YH_F32, 128, 16, FAKE, _lib.YH_F32, 128, 16, 1, 8, 16, *coeffs, steps, 1e-7, FAKE, BIG,
                                None) == _lib.YH_ERR_ARG
    assert lib.yh_muon_step(lists, _lib.YH_F32, lists, _lib.YH_F32, lists, 1, 8, 16, 0.1, 0.9, 1, 0.0, 1.0, *coeffs, steps, 1e-7,
                            FAKE, BIG, None) == _lib.YH_ERR_ARG


def test_momenta_stay_fp32_through_a_state_dict():
    """torch casts the state of a 16-bit weight to 16 bits when it is loaded; momenta are not."""
    weights = [torch.nn.Parameter(torch.zeros(3, 5, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(4, 2))]
    first, second = Muon(weights), Muon(weights, lr=1.0)
    for p in weights:
        first.state[p]["momentum_buffer"] = torch.randn(p.shape)
    second.load_state_dict(first.state_dict())
    for p in weights:
        got, saved = (o.state[p]["momentum_buffer"] for o in (second, first))
        assert got.dtype == torch.float32 and torch.equal(got, saved) and got.data_ptr() != saved.data_ptr()
    assert second.param_groups[0]["lr"] == 0.02


def test_the_first_step_of_a_weight_is_not_captured(monkeypatch):
    """A replay would set the momentum back to zero each time."""
    w = torch.nn.Parameter(torch.zeros(3, 5))
    w.grad = torch.ones(3, 5)
    optim = Muon([w])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        optim.step()
    assert not optim.state[w]
