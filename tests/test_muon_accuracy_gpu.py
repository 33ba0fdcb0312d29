"""How far results of the orthogonalised update are from its formula in 64 bits before they are rounded to their type.

Bounds.  The documented contract: 1e-4 of the whole matrix (Frobenius norms) for fp32 and fp16 results, 1e-3 for bf16 ones.  It
was set from 29 shapes (16 x 16 to 4096 x 9216) and 18 spectra (noise; 1 to 64 strong directions over 0.1 to 10 % of noise;
one to four decades), where three steps and two end at most 5.5e-5 off and five steps on one X X' 8.2e-4.  The rounding to the
result's type is measured, not bounded: it is that of the exact result, and adds to the error in squares, since the two are
independent (their product, added over rows x cols numbers, is of the order of rounding * error / sqrt(rows * cols):
2 / sqrt(rows * cols) of the larger square, 4 deviations of it below)."""
import math

import pytest
import torch

from yolo_amd import muon_step, orthogonalize

pytestmark = pytest.mark.gpu
COEFFS = (3.4445, -4.7750, 2.0315)
CONTRACT = {torch.float32: 1e-4, torch.float16: 1e-4, torch.bfloat16: 1e-3}


def polar(g, steps=5):
    a, b, c = COEFFS
    x = g.double() / (g.double().norm() + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for _ in range(steps):
        w = x @ x.t()
        x = a * x + (b * w + c * (w @ w)) @ x
    return x.t() if tall else x


def gradient(rows, cols, kind, gen):
    if kind == "noise":
        return torch.randn(rows, cols, generator=gen)
    if kind == "few strong":
        rank, strength, floor = 8, torch.ones(min(8, rows, cols)), 0.01
    elif kind == "one strong":
        rank, strength, floor = 1, torch.ones(1), 0.01
    else:                                                 # "graded"
        rank, strength, floor = 16, torch.logspace(0, -1.5, min(16, rows, cols)), 0.1
    rank = min(rank, rows, cols)
    strong = (torch.randn(rows, rank, generator=gen) * strength) @ torch.randn(rank, cols, generator=gen)
    return 1e-3 * (strong + floor * torch.randn(rows, cols, generator=gen))


def check(got, want, contract):
    """got, of its type, is want + an error of at most contract, rounded."""
    size = want.norm().item()
    err = (got.double().to(want.device) - want).norm().item() / size
    rounding = (want.to(got.dtype).double() - want).norm().item() / size
    bound = rounding ** 2 + contract ** 2 + 4 * 2 / math.sqrt(want.numel()) * rounding * max(rounding, contract)
    assert err ** 2 <= bound, (err, rounding, math.sqrt(max(err ** 2 - rounding ** 2, 0.0)))


@pytest.mark.parametrize("kind", ["noise", "few strong", "one strong", "graded"])
@pytest.mark.parametrize("rows,cols", [(64, 147), (90, 300), (128, 1152), (1000, 130), (192, 576), (300, 1000), (512, 2304)])
def test_results_before_their_rounding(dev, rows, cols, kind):
    g = gradient(rows, cols, kind, torch.Generator().manual_seed(rows + 2 * cols))
    for g_dtype in (torch.float32, torch.float16, torch.bfloat16):
        typed = g.to(g_dtype)
        want = polar(typed.to(dev))
        for out, contract in CONTRACT.items():
            check(orthogonalize(typed.to(dev), out_dtype=out), want, contract)


@pytest.mark.parametrize("p_dtype", list(CONTRACT))
def test_steps_of_zero_weights(dev, p_dtype):
    """A weight of zeros becomes the update itself, rounded to the weight's type."""
    g = gradient(128, 1152, "graded", torch.Generator().manual_seed(3))
    p, m = torch.zeros(128, 1152, dtype=p_dtype, device=dev), torch.zeros(128, 1152, device=dev)
    muon_step([p], [g.to(dev)], [m], lr=1.0, momentum=0.0, scale=1.0)
    check(-p, polar(g.to(dev)), CONTRACT[p_dtype])


@pytest.mark.parametrize("kind", ["noise", "few strong", "one strong", "graded"])
@pytest.mark.parametrize("rows,cols,count", [(513, 4097, 1), (4097, 513, 1), (200, 1100, 9), (1470, 1470, 1)])
def test_three_steps_of_16_bit_gradients(dev, rows, cols, count, kind):
    """X held in fp16 alone (16-bit gradient and result, one X X'), with results whose rounding is small enough to see
    both planes of S: fp16 alone would end 1e-3 off and more."""
    gen = torch.Generator().manual_seed(rows + 3 * cols)
    g = torch.stack([gradient(rows, cols, kind, gen) for _ in range(count)])
    for g_dtype in (torch.float16, torch.bfloat16):
        typed = g.to(g_dtype).to(dev)
        got = orthogonalize(typed, steps=3, out_dtype=torch.float16)
        for i in range(0, count, 4):
            check(got[i], polar(typed[i], 3), CONTRACT[torch.float16])
