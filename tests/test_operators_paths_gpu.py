"""The 8-bit product and the orthogonalised update at sizes that take their large tiles and cut the contraction in slices, every
number of the result against 64 bits (on the GPU: sums of whole numbers below 2^53 are exact there).

Bounds.  8-bit product: the conversion to fp32, the two scales and the bias round once each, 3 * 2^-24 of |acc s t| (one more
for their products) and 2 * 2^-24 of the sum, then half a step of the result's type.  Update: 1e-4 of the whole matrix for fp32
results is the contract; a weight of fp32 adds the rounding of decay, step, their products and the difference, 2^-22 of it and of
the update; a momentum rounds three times."""
import math

import pytest
import torch

from yolo_amd import _lib, linear_i8, muon_step, orthogonalize, quantize_rows

pytestmark = pytest.mark.gpu


def partial_bytes(dtype, m, n, k):
    """What the workspace holds beyond the quantised rows, their scales and the parts' largest numbers: the slices' sums."""
    up = lambda b: (b + 255) // 256 * 256  # noqa: E731
    total = _lib.load().yh_linear_i8_workspace_bytes(_lib.DTYPE_CODES[dtype], m, n, k)
    return total - up(m * ((k + 127) // 128 * 128)) - up(4 * m) - (up(64 * m) if m < 256 else 0)


# (m, k, n), slices of the contraction: whole ones, a shorter last one, channels that no vector divides, every tile
SLICED = [((64, 50176, 4096), 4), ((50, 50176, 1470), 8), ((17, 9000, 333), 15), ((33, 20000, 1470), 8), ((100, 65537, 130), 16),
          ((300, 50000, 514), 16), ((500, 50001, 4095), 4), ((40, 131071, 64), 16)]
WHOLE = [((1024, 4096, 4096), 1), ((1000, 4100, 4095), 1), ((700, 3000, 4001), 1), ((1100, 2000, 4001), 1), ((2047, 4001, 4095), 1),
         ((4001, 513, 3001), 1)]


@pytest.mark.parametrize("size,slices", SLICED + WHOLE)
@pytest.mark.parametrize("dtype,out,bias", [(torch.bfloat16, torch.bfloat16, True), (torch.float32, torch.float32, True),
                                            (torch.int8, torch.float16, False)])
def test_linear_i8_in_slices_and_large_tiles(dev, size, slices, dtype, out, bias):
    m, k, n = size
    gen = torch.Generator(device=dev).manual_seed(m + k + n)
    extra = partial_bytes(dtype, m, n, k)
    assert (extra > 0) == (slices > 1) and extra >= (slices > 1) * 4 * slices * m * n
    w, t = quantize_rows(torch.randn(n, k, generator=gen, device=dev) / k ** 0.5)
    b = torch.randn(n, generator=gen, device=dev) if bias else None
    if dtype == torch.int8:
        x = torch.randint(-128, 128, (m, k), generator=gen, dtype=torch.int8, device=dev)
        s = torch.rand(m, generator=gen, device=dev) / k ** 0.5
        y = linear_i8(x, w, t, x_scale=s, out_dtype=out)
        q = x.double()
    else:
        x = torch.nn.functional.leaky_relu(torch.randn(m, k, generator=gen, device=dev), 0.1).to(dtype)
        y = linear_i8(x, w, t, bias=b, out_dtype=out)
        top = x.double().abs().amax(1, keepdim=True)
        q, s = torch.round(127 * x.double() / top), top[:, 0].float() / 127
    scaled = (q @ w.double().t()) * s.double()[:, None] * t.double()
    want = scaled if b is None else scaled + b.double()
    half = torch.finfo(out).eps / 2 if out != torch.float32 else 0.0
    bound = 4 * 2.0 ** -24 * scaled.abs() + 2 * 2.0 ** -24 * want.abs()
    bound = bound + half * (want.abs() + bound) + (2.0 ** -25 if out == torch.float16 else 0.0) + 1e-37
    err = (y.double() - want).abs()
    assert bool((err <= bound).all()), (err / bound).max()
    if bias is False:
        assert torch.equal(y, linear_i8(x, w, t, x_scale=s, out_dtype=out))


def polar(x):
    a, b, c = 3.4445, -4.7750, 2.0315
    x = x / (x.norm() + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for _ in range(5):
        w = x @ x.t()
        x = a * x + (b * w + c * (w @ w)) @ x
    return x.t() if tall else x


def gradient(count, rows, cols, gen, dev):
    strong = torch.randn(count, rows, 16, generator=gen, device=dev) * torch.logspace(0, -1.5, 16, device=dev)
    return 1e-3 * (strong @ torch.randn(count, 16, cols, generator=gen, device=dev)
                   + 0.1 * torch.randn(count, rows, cols, generator=gen, device=dev))


@pytest.mark.parametrize("rows,cols,count", [(4096, 1470, 1), (1024, 9216, 1), (1000, 9001, 4), (600, 50001, 1), (20001, 1100, 2),
                                             (2048, 4097, 2)])
def test_orthogonalize_in_slices_and_large_tiles(dev, rows, cols, count):
    g = gradient(count, rows, cols, torch.Generator(device=dev).manual_seed(rows + cols), dev)
    got = orthogonalize(g, out_dtype=torch.float32)
    for i in range(count):
        want = polar(g[i].double())
        assert (got[i].double() - want).norm() <= 1e-4 * want.norm(), i
    typed = g.to(torch.float16)                           # X in fp16 alone: one X X' for three steps
    got = orthogonalize(typed, steps=3, out_dtype=torch.float16)
    again = orthogonalize(typed, steps=3, out_dtype=torch.float32)
    # each within 1e-4 of the exact result, and the rounding to fp16 (2^-11 of every number at most)
    for i in range(count):
        assert (got[i].double() - again[i].double()).norm() <= (2e-4 + 2.0 ** -11) * again[i].double().norm(), i


@pytest.mark.parametrize("rows,cols,count,g_dtype", [(1024, 9216, 4, torch.bfloat16), (4096, 1470, 1, torch.float32)])
def test_muon_step_in_slices_and_large_tiles(dev, rows, cols, count, g_dtype):
    gen = torch.Generator(device=dev).manual_seed(rows)
    g = gradient(count, rows, cols, gen, dev).to(g_dtype)
    m = 5 * gradient(count, rows, cols, gen, dev)
    p = (2 * torch.rand(count, rows, cols, generator=gen, device=dev) - 1) / math.sqrt(cols)
    ps, ms = [t.clone() for t in p], [t.clone() for t in m]
    muon_step(ps, list(g), ms, lr=0.02, weight_decay=0.01)
    for i in range(count):
        wm = 0.95 * m[i].double() + g[i].double()
        bound = 2.0 ** -24 * (3 * 0.95 * m[i].double().abs() + g[i].double().abs()) * 1.0001
        assert bool(((ms[i].double() - wm).abs() <= bound).all()), i
        step = 0.02 * math.sqrt(max(1.0, rows / cols))
        o = polar(g[i].double() + 0.95 * wm)
        want = (1 - 0.02 * 0.01) * p[i].double() - step * o
        size = step * o.norm()
        assert (ps[i].double() - want).norm() <= 2.0 ** -22 * (want.norm() + size) + 1e-4 * size, i
