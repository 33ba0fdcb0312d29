"""A gradient that is asked for is refused by the operators without one, never dropped.  No GPU: what is asked for is
looked at before where the tensors live."""
import pytest
import torch
from torch.autograd import forward_ad

from yolo_amd import Int8Linear, linear_i8, muon_step, orthogonalize, quantize_rows

W, S = torch.zeros(3, 64, dtype=torch.int8), torch.ones(3)


@pytest.mark.parametrize("name", ["weight_scale", "bias", "x_scale"])
def test_a_gradient_of_any_argument_is_refused(name):
    x = torch.zeros(2, 64, dtype=torch.int8) if name == "x_scale" else torch.zeros(2, 64)
    kw = dict(weight_scale=S, bias=torch.zeros(3), x_scale=torch.ones(2) if name == "x_scale" else None)
    kw[name] = kw[name].clone().requires_grad_(True)
    with pytest.raises(ValueError, match=f"{name}: requires a gradient"):
        linear_i8(x, W, **kw)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):       # not asked for
        linear_i8(x, W, **kw)


def test_a_bias_that_is_a_parameter_is_copied_by_the_layer():
    layer = Int8Linear(W, S.clone().requires_grad_(True), torch.nn.Parameter(torch.zeros(3)))
    assert not layer.bias.requires_grad and not layer.weight_scale.requires_grad


@pytest.mark.parametrize("grad_mode", [True, False])
def test_a_tangent_is_refused(grad_mode):
    x, scale = torch.randn(4, 64), torch.ones(4)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t))  # noqa: E731
        for call in (lambda: quantize_rows(dual(x)), lambda: linear_i8(dual(x), W, S), lambda: linear_i8(x, W, dual(S)),
                     lambda: linear_i8(x, W, S, bias=dual(torch.zeros(3))), lambda: orthogonalize(dual(x)),
                     lambda: linear_i8(x.to(torch.int8), W, S, x_scale=dual(scale)),
                     lambda: muon_step([x], [dual(x)], [x.clone()], lr=0.1), lambda: muon_step([dual(x)], [x], [x.clone()], lr=0.1),
                     lambda: muon_step([x], [x.clone()], [dual(x)], lr=0.1)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        with pytest.raises(ValueError, match="GPU"):
            linear_i8(x, W, S)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda v: orthogonalize(v), (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("what", [None, 3.0, [[1.0, 2.0]], "x"])
def test_what_is_no_tensor_is_named(what):
    for call in (lambda: linear_i8(what, W, S), lambda: quantize_rows(what), lambda: orthogonalize(what)):
        with pytest.raises(TypeError, match="expected a torch.Tensor"):
            call()
    for bad in (lambda: muon_step([what], [S], [S], lr=0.1), lambda: muon_step([W.float()], [what], [S], lr=0.1)):
        with pytest.raises(TypeError, match="expected a torch.Tensor"):
            bad()
