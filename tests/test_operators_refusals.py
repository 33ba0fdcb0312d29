"""Refusals name what is refused, and the limits that are stated are those that hold.  Without a GPU but for the last."""
import math

import pytest
import torch

from yolo_amd import _lib, linear_i8, muon_step, orthogonalize, quantize_rows

X = torch.zeros(4, 6)


@pytest.mark.parametrize("name", ["lr", "momentum", "weight_decay", "scale"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 1e39])
def test_numbers_that_fp32_does_not_hold_are_named(name, value):
    with pytest.raises(_lib.YoloHeadError, match=f"^{name}: .*finite") as caught:
        muon_step([X], [X.clone()], [X.clone()], **{"lr": 0.1, name: value})
    assert caught.value.rc == _lib.YH_ERR_ARG


@pytest.mark.parametrize("call", [lambda **kw: orthogonalize(X, **kw), lambda **kw: muon_step([X], [X.clone()], [X.clone()], lr=0.1, **kw)])
def test_coefficients_and_eps_are_named(call):
    for at in range(3):
        coeffs = [3.4445, -4.7750, 2.0315]
        coeffs[at] = math.nan if at else 1e39
        with pytest.raises(_lib.YoloHeadError, match=rf"^coeffs\[{at}\]: .*finite"):
            call(coeffs=coeffs)
    for coeffs in ((1.0, 2.0), (1.0, 2.0, 3.0, 4.0)):
        with pytest.raises(ValueError, match="coeffs: expected three"):
            call(coeffs=coeffs)
    for eps in (1e39, math.nan, -1.0):
        with pytest.raises(ValueError, match="^eps: "):
            call(eps=eps)


def test_the_stated_limits_are_those_of_the_library():
    """The header: at most 65,535 matrices, shorter side <= 32,768, longer <= 2^24, and in all fewer than 2^24 tiles of 32 x 32."""
    size = _lib.load().yh_orthogonalize_workspace_bytes
    for count, rows, cols, fine in [(65535, 8, 8, True), (65536, 8, 8, False), (100000, 8, 8, False), (1, 32768, 32768, True),
                                    (1, 32769, 32769, False), (1, 1024, 1 << 24, False), (1, 2048, 1 << 23, False),
                                    (1, 992, 1 << 24, True), (1, 31 * 32 + 1, 1 << 24, False), (33, 992, 1 << 19, True),
                                    (34, 992, 1 << 19, False), (1, 32, (1 << 24) + 1, False), (1, 1 << 24, 32, True)]:
        tiles = count * -(-rows // 32) * -(-cols // 32)
        stated = count <= 65535 and min(rows, cols) <= 32768 and max(rows, cols) <= 1 << 24 and tiles < 1 << 24
        assert (size(count, rows, cols) > 0) == fine == stated, (count, rows, cols)
    size = _lib.load().yh_linear_i8_workspace_bytes
    for m, n, fine in [(_lib.YH_MAX_I8_ROWS, 17, True), (_lib.YH_MAX_I8_ROWS + 1, 17, False), (17, _lib.YH_MAX_I8_ROWS, True),
                       (17, _lib.YH_MAX_I8_ROWS + 1, False), (1 << 17, (1 << 17) - 32, True), (1 << 17, 1 << 17, False)]:
        stated = max(m, n) <= _lib.YH_MAX_I8_ROWS and -(-m // 32) * -(-n // 32) < 1 << 24
        assert (size(_lib.YH_F32, m, n, 4096) > 0) == fine == stated, (m, n)


@pytest.mark.gpu
def test_refused_sizes_and_coefficients_state_their_limits(dev):
    x = torch.zeros(4, 6, device=dev)
    with pytest.raises(ValueError, match="65,535"):
        orthogonalize(torch.zeros(65536, 2, 2, device=dev))
    assert not orthogonalize(torch.zeros(65535, 2, 2, device=dev)).any()
    for call in (lambda: orthogonalize(x, coeffs=(3.0, -4.0, 2.0)),
                 lambda: muon_step([x], [x.clone()], [x.clone()], lr=0.1, coeffs=(3.0, -4.0, 2.0))):
        with pytest.raises(_lib.YoloHeadError, match="coefficients.*120"):
            call()
    many = torch.zeros(1, 8, device=dev).expand(_lib.YH_MAX_I8_ROWS + 1, 8)
    with pytest.raises(ValueError, match="4,194,303"):
        quantize_rows(many)
    w, t = quantize_rows(torch.ones(3, 8, device=dev))
    with pytest.raises(ValueError, match="4,194,303"):
        linear_i8(many, w, t)
    wide = torch.zeros(1, 16, dtype=torch.int8, device=dev).expand(_lib.YH_MAX_I8_ROWS + 1, 16)
    with pytest.raises(ValueError, match="weight"):
        linear_i8(x[:, :1].expand(4, 16).contiguous(), wide, torch.zeros(1, device=dev).expand(_lib.YH_MAX_I8_ROWS + 1))
    a, b = torch.zeros(1 << 17, 16, dtype=torch.int8, device=dev), torch.zeros(1 << 17, device=dev)
    with pytest.raises(ValueError, match="tiles"):
        linear_i8(a, a, b, x_scale=b, out_dtype=torch.float16)


@pytest.mark.gpu
def test_a_weight_elsewhere_is_named(dev):
    x = torch.ones(4, 16, device=dev)
    w, t = quantize_rows(torch.ones(3, 16, device=dev))
    with pytest.raises(ValueError, match=r"weight: on cpu, x is on cuda:0"):
        linear_i8(x, torch.zeros(3, 16, dtype=torch.int8), t)
