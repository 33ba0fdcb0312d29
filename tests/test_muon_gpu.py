"""The orthogonalised update against its formula in 64 bits.

Bounds.  The matrices are held in two fp16 numbers (22 bits), products are summed in fp32.  An error of X X' grows by
a^2 = 11.9 from step to step, so a bound of the worst case says little; emulated on the CPU with the same roundings
(64 x 147 to 1024 x 1024; noise, singular values over four decades, eight strong directions over 1 % of noise) the
result ends at most 3.1e-5 off (relative, whole matrix) with one X X' for three steps and 1.9e-4 with one for five.
The bounds below are three times that: 1e-4 for fp32 results, 6e-4 for 16-bit ones plus their rounding
(torch.finfo(t).eps / 2)."""
import math

import pytest
import torch

from yolo_amd import Muon, YOLOv1Head, _lib, muon_step, orthogonalize, synth

pytestmark = pytest.mark.gpu
COEFFS = (3.4445, -4.7750, 2.0315)
FAR = {torch.float32: 1e-4, torch.bfloat16: 6e-4 + 2.0 ** -8, torch.float16: 6e-4 + 2.0 ** -11}


def polar(g, steps=5, coeffs=COEFFS, eps=1e-7):
    a, b, c = coeffs
    x = g.double()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(steps):
        w = x @ x.t()
        x = a * x + (b * w + c * w @ w) @ x
    return x.t() if tall else x


def gradient(rows, cols, kind, gen):
    if kind == "noise":
        return torch.randn(rows, cols, generator=gen)
    rank = min(8, rows, cols)
    strong = torch.randn(rows, rank, generator=gen) @ torch.randn(rank, cols, generator=gen)
    return 1e-3 * (strong + 0.05 * torch.randn(rows, cols, generator=gen))


def off(got, want):
    return ((got.cpu().double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 50), (50, 1), (2, 3), (31, 33), (64, 147), (147, 64), (65, 128), (128, 129),
                                       (192, 576), (257, 255), (300, 1000), (1000, 130), (512, 2304), (700, 700)])
def test_orthogonalize(dev, rows, cols, out):
    gen = torch.Generator().manual_seed(rows * 7 + cols)
    for kind, dtype in (("noise", torch.float32), ("strong", torch.bfloat16), ("strong", torch.float16)):
        g = gradient(rows, cols, kind, gen).to(dtype)
        got = orthogonalize(g.to(dev), out_dtype=out)
        assert got.shape == g.shape and got.dtype == out
        assert off(got, polar(g)) <= FAR[out], kind
        assert torch.equal(got, orthogonalize(g.to(dev), out_dtype=out))


@pytest.mark.parametrize("g_dtype,out", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("rows,cols,count", [(129, 15601, 1), (513, 4097, 1), (4097, 513, 1), (1000, 1003, 2), (1470, 1470, 1),
                                             (200, 1100, 9)])
def test_16_bit_gradients(dev, rows, cols, count, g_dtype, out):
    """Large enough that X is held in fp16 alone: what 16-bit numbers hold, fp16 holds times a power of two, but for
    numbers below 2^-14 of the scaled matrix (mean square about 1), which are off by 2^-25 at most: less than 22 bits."""
    gen = torch.Generator().manual_seed(rows + cols)
    for kind, power in (("noise", 0), ("strong", 0), ("noise", -20), ("spikes", 10 if g_dtype == torch.bfloat16 else 0)):
        g = torch.stack([gradient(rows, cols, "strong" if kind == "strong" else "noise", gen) for _ in range(count)])
        if kind == "spikes":
            g *= 1e-3
            g[:, 3, 5] = 300.0
            g[:, rows - 1, cols - 1] = -40.0
        if power:
            g = g * 2.0 ** power
        g = g.to(g_dtype)
        got = orthogonalize(g.to(dev), out_dtype=out)
        for i in range(0, count, 8):
            assert off(got[i], polar(g[i])) <= FAR[out], (kind, i)
        wide = torch.full((count, rows + 2, cols + 3), 7.0, dtype=g_dtype, device=dev)
        wide[:, 1:-1, 1:-2] = g.to(dev)
        assert torch.equal(orthogonalize(wide[:, 1:-1, 1:-2], out_dtype=out), got)
    bad = torch.stack([g[0], torch.zeros_like(g[0]), g[0], g[0], g[0]]).to(dev)
    bad[2, rows - 1, 3] = float("nan")
    bad[3, 0, cols - 1] = float("-inf")
    got = orthogonalize(bad, out_dtype=out)
    assert torch.equal(got[4], got[0]) and not got[1].any() and torch.isnan(got[2:4]).all()


@pytest.mark.parametrize("rows,cols,count", [(130, 150, 48), (263, 263, 48), (330, 326, 32), (326, 330, 64), (1150, 2500, 2)])
def test_every_tile_of_the_products(dev, rows, cols, count):
    """Batches that fill the card with each of the tiles the products are cut into."""
    gen = torch.Generator().manual_seed(count)
    g = torch.randn(count, rows, cols, generator=gen)
    for dtype, out in ((torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.float16)):
        typed = g.to(dtype)
        got = orthogonalize(typed.to(dev), out_dtype=out)
        for i in (0, count // 2, count - 1):
            assert off(got[i], polar(typed[i])) <= FAR[out], (dtype, out, i)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 9])
@pytest.mark.parametrize("rows,cols", [(40, 100), (100, 40), (130, 260)])
def test_any_number_of_steps(dev, rows, cols, steps):
    gen = torch.Generator().manual_seed(steps)
    g = gradient(rows, cols, "noise", gen)
    assert off(orthogonalize(g.to(dev), steps=steps, out_dtype=torch.float32), polar(g, steps)) <= 1e-4
    assert off(orthogonalize(g.to(dev), steps=steps), polar(g, steps)) <= FAR[torch.bfloat16]


@pytest.mark.parametrize("coeffs,steps", [((1.5, -0.5, 0.0), 10), ((2.0, -1.5, 0.5), 8), ((15 / 8, -10 / 8, 3 / 8), 8)])
def test_other_coefficients(dev, coeffs, steps):
    gen = torch.Generator().manual_seed(3)
    g = gradient(48, 200, "noise", gen)
    got = orthogonalize(g.to(dev), steps=steps, coeffs=coeffs, out_dtype=torch.float32)
    assert off(got, polar(g, steps, coeffs)) <= 1e-4


def test_batches_and_strides(dev):
    gen = torch.Generator().manual_seed(4)
    g = torch.randn(2, 3, 33, 70, generator=gen).to(dev)
    want = torch.stack([orthogonalize(m) for m in g.view(6, 33, 70)]).view(2, 3, 33, 70)
    assert torch.equal(orthogonalize(g), want)
    store = torch.full((6, 40, 81), 9.0, device=dev)
    store[:, 3:36, 5:75] = g.view(6, 33, 70)
    assert torch.equal(orthogonalize(store[:, 3:36, 5:75]), want.view(6, 33, 70))
    assert torch.equal(orthogonalize(store[::2, 3:36, 5:75]), want.view(6, 33, 70)[::2])
    assert torch.equal(orthogonalize(store[1, 3:36, 5:75]), want.view(6, 33, 70)[1])
    assert torch.equal(orthogonalize(g[0, 0].expand(3, 33, 70)), want[0, 0].expand(3, 33, 70))
    tall = orthogonalize(g[0, 0].t().contiguous(), out_dtype=torch.float32)
    assert (tall.t() - orthogonalize(g[0, 0], out_dtype=torch.float32)).abs().max() < 1e-4
    assert orthogonalize(g[:0]).shape == (0, 3, 33, 70) and orthogonalize(g[..., :0]).shape == (2, 3, 33, 0)
    with pytest.raises(ValueError, match="next to each other"):
        orthogonalize(g[0, 0].t())
    with pytest.raises(ValueError, match="gradient"):
        orthogonalize(g.requires_grad_(True))


def test_scale_zeros_and_what_is_not_a_number(dev):
    gen = torch.Generator().manual_seed(5)
    g = torch.randn(40, 90, generator=gen).to(dev)
    want = orthogonalize(g, eps=0.0, out_dtype=torch.float32)
    for power in (-100, -60, 60, 100):      # squares below and above the range of fp32 (entries stay inside it)
        # the norm, added in 64 bits, is the same number but for its power of two
        assert torch.equal(orthogonalize(g * 2.0 ** power, eps=0.0, out_dtype=torch.float32), want), power
    # norms around and far below eps: X is small and stays so, to its last bits
    for power, steps in ((-20, 5), (-30, 5), (-40, 5), (-60, 5), (-100, 5), (-30, 8), (-45, 8)):
        small = g * 2.0 ** power
        got = orthogonalize(small, steps=steps, out_dtype=torch.float32)
        assert off(got, polar(small.cpu(), steps)) <= 1e-4, (power, steps)
        assert off(orthogonalize(small, steps=steps), polar(small.cpu(), steps)) <= FAR[torch.bfloat16], (power, steps)
    batch = torch.stack([g, torch.zeros_like(g), g, g, g])
    batch[2, 17, 3] = float("nan")
    batch[3, 0, 0] = float("inf")
    got = orthogonalize(batch)
    assert torch.equal(got[0], orthogonalize(g)) and torch.equal(got[4], got[0])
    assert not got[1].any() and torch.isnan(got[2:4]).all()
    spike = torch.zeros(64, 500, device=dev)
    spike[3, 400] = 5.0
    assert off(orthogonalize(spike, out_dtype=torch.float32), polar(spike.cpu())) <= 1e-4


def test_many_steps_of_tiny_gradients(dev):
    """|X_0| far below 1 and enough steps for it to grow back: what is held of X grows by 3.4445 a step until the singular
    values have reached their range, and stays inside fp16's."""
    gen = torch.Generator().manual_seed(6)
    line = torch.zeros(40, 90)
    line[7, 30] = 1.0                                     # all of the norm in one number
    noise = torch.randn(40, 90, generator=gen)
    noise /= noise.norm()
    wide = torch.randn(200, 260, generator=gen)
    for name, g in (("line", line), ("noise", noise), ("wide", wide / wide.norm()), ("tall", (wide / wide.norm()).t().contiguous())):
        for norm, steps in ((1e-11, 9), (1e-12, 12), (1e-13, 16), (1e-15, 20), (1e-25, 40), (1.0, 30)):
            small = g * norm
            for out in (torch.float32, torch.float16):
                got, want = orthogonalize(small.to(dev), steps=steps, out_dtype=out), polar(small, steps)
                assert torch.isfinite(got).all() and got.any(), (name, norm, steps)
                if want.norm() > 1e-3 and name == "line":
                    assert off(got, want) <= FAR[out], (name, norm, steps)


@pytest.mark.parametrize("coeffs,steps", [((2.0, 2.0, 1.0), 1), ((100.0, -99.0, 0.0), 1), ((1.0, 60.0, -59.0), 1), ((0.5, 0.0, 0.0), 40),
                                          ((0.0, 1.0, 0.0), 1), ((-1.5, 0.5, 0.0), 7), ((1.5, -0.5, 0.0), 64)])
def test_coefficients_within_range(dev, coeffs, steps):
    gen = torch.Generator().manual_seed(8)
    for rows, cols in ((30, 70), (150, 140)):
        g = gradient(rows, cols, "noise", gen)
        got = orthogonalize(g.to(dev), steps=steps, coeffs=coeffs, out_dtype=torch.float32)
        assert off(got, polar(g, steps, coeffs)) <= 1e-4


def test_coefficients_out_of_range_name_themselves(dev):
    x = torch.randn(8, 16, device=dev)
    before = x.clone()
    with pytest.raises(_lib.YoloHeadError, match="coefficients"):
        orthogonalize(x, coeffs=(3.0, -4.0, 2.0))
    with pytest.raises(_lib.YoloHeadError, match="coefficients"):
        muon_step([x], [x.clone()], [x.clone()], lr=0.1, coeffs=(30.0, 0.0, 0.0))
    with pytest.raises(_lib.YoloHeadError, match="finite"):
        muon_step([x], [x.clone()], [x.clone()], lr=math.nan)
    assert torch.equal(x, before)


def test_state_dict_of_16_bit_weights(dev):
    torch.manual_seed(1)
    w = torch.nn.Parameter(torch.randn(24, 40, device=dev, dtype=torch.bfloat16))
    optim = Muon([w], lr=0.1)
    grads = [torch.randn_like(w) for _ in range(3)]
    for g in grads[:2]:
        w.grad = g
        optim.step()
    other = torch.nn.Parameter(w.detach().clone())
    loaded = Muon([other])
    loaded.load_state_dict(optim.state_dict())
    w.grad, other.grad = grads[2], grads[2].clone()
    optim.step()
    loaded.step()
    assert torch.equal(w.detach(), other.detach())


def test_large_matrix(dev):
    """Offsets past 2^32 bytes in the split copies (70 x 2^24 numbers of 4 bytes)."""
    rows, cols = 70, 1 << 24
    g = torch.zeros(rows, cols, dtype=torch.bfloat16, device=dev)
    at = torch.arange(rows, device=dev)
    g[at, cols - 1 - 31 * at] = 3.0                     # orthogonal rows, at the far end: all singular values are equal
    got = orthogonalize(g)
    want = polar(torch.eye(rows) * 3.0)[0, 0].item()
    hit = got[at, cols - 1 - 31 * at].float()
    assert ((hit - want).abs() <= want * FAR[torch.bfloat16]).all()
    got[at, cols - 1 - 31 * at] = 0
    assert not got.any()


def test_large_16_bit_matrix(dev):
    """The same where X is held in fp16 alone (offsets past 2^32 bytes)."""
    rows, cols = 130, 1 << 24
    g = torch.zeros(rows, cols, dtype=torch.float16, device=dev)
    at = torch.arange(rows, device=dev)
    g[at, cols - 1 - 31 * at] = 3.0
    got = orthogonalize(g)
    want = polar(torch.eye(rows) * 3.0)[0, 0].item()
    hit = got[at, cols - 1 - 31 * at].float()
    assert ((hit - want).abs() <= want * FAR[got.dtype]).all()
    got[at, cols - 1 - 31 * at] = 0
    assert not got.any()


def _want(p, g, m, lr, momentum, wd, nesterov, scale=None):
    m = momentum * m.double() + g.double()
    o = polar((g.double() + momentum * m if nesterov else m).view(g.shape[0], -1)).view(g.shape)
    rows, cols = g.shape[0], g.numel() // g.shape[0]
    step = lr * (math.sqrt(max(1.0, rows / cols)) if scale is None else scale)
    return (1 - lr * wd) * p.double() - step * o, m, step * o.norm().item()


@pytest.mark.parametrize("p_dtype,g_dtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                             (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("shape,count", [((64, 3, 7, 7), 1), ((192, 64, 3, 3), 3), ((300, 130), 2), ((8, 8), 35), ((1, 9), 2), ((33, 1), 1)])
def test_muon_step(dev, shape, count, p_dtype, g_dtype):
    gen = torch.Generator().manual_seed(count + shape[0])
    p = [(0.1 * torch.randn(shape, generator=gen)).to(p_dtype) for _ in range(count)]
    g = [(1e-2 * torch.randn(shape, generator=gen)).to(g_dtype) for _ in range(count)]
    m = [5e-2 * torch.randn(shape, generator=gen) for _ in range(count)]
    for nesterov, scale in ((True, None), (False, 0.3)):
        dp, dg, dm = ([t.to(dev) for t in some] for some in (p, g, m))
        versions = [t._version for t in dp + dm]
        muon_step(dp, dg, dm, lr=0.05, momentum=0.9, weight_decay=0.1, nesterov=nesterov, scale=scale)
        assert all(t._version > v for t, v in zip(dp + dm, versions))
        for i in range(count):
            wp, wm, size = _want(p[i], g[i], m[i], 0.05, 0.9, 0.1, nesterov, scale)
            # 0.9 as an fp32 number, its product with m and the sum round once each: 2^-24 (0.9 |m| + 0.9 |m| + 0.9 |m| + |g|)
            bound = 2.0 ** -24 * (2.7 * m[i].double().abs() + g[i].double().abs()) * 1.0001
            assert bool(((dm[i].cpu().double() - wm).abs() <= bound).all())
            # decay and step as fp32 numbers, their products and the difference: 2^-22 of p; the update; the type's rounding
            half = 0.0 if p_dtype == torch.float32 else torch.finfo(p_dtype).eps / 2
            far = (1e-4 if p_dtype == torch.float32 else 6e-4) * size
            err = (dp[i].cpu().double() - wp).norm().item()
            assert err <= (2.0 ** -22 + half) * (wp.norm().item() + size) + far
            assert torch.equal(dg[i].cpu(), g[i])


def test_muon_step_refusals(dev):
    p = [torch.zeros(4, 6, device=dev) for _ in range(3)]
    with pytest.raises(ValueError, match="twice"):
        muon_step([p[0], p[0]], [p[1], p[1]], [p[2], torch.zeros_like(p[2])], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        muon_step([p[0]], [p[0]], [p[2]], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        muon_step([p[0]], [p[1]], [p[0]], lr=0.1)
    whole = torch.zeros(10, 6, device=dev)
    with pytest.raises(ValueError, match="twice"):
        muon_step([whole[:4], whole[3:7]], [p[0], p[1]], [p[2], torch.zeros_like(p[2])], lr=0.1)
    with pytest.raises(ValueError, match="shape"):
        muon_step([p[0]], [p[1][:3]], [p[2]], lr=0.1)
    with pytest.raises(ValueError, match="dtype"):
        muon_step([p[0]], [p[1]], [p[2].half()], lr=0.1)
    with pytest.raises(ValueError, match="contiguous"):
        muon_step([torch.zeros(6, 4, device=dev).t()], [p[1]], [p[2]], lr=0.1)
    with pytest.raises(ValueError, match="steps"):
        muon_step([p[0]], [p[1]], [p[2]], lr=0.1, steps=0)
    with pytest.raises(_lib.YoloHeadError):
        muon_step([p[0]], [p[1]], [p[2]], lr=float("nan"))


@pytest.mark.parametrize("rows,cols,count", [(40, 90, 2), (90, 40, 2), (129, 8000, 1), (8000, 129, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_lies_between_the_rows_of_the_result_stays(dev, rows, cols, count, dtype):
    """Results at strides of their own, stored 16 bytes, a pair or one number at a time."""
    gen = torch.Generator().manual_seed(12)
    lib, code = _lib.load(), _lib.DTYPE_CODES[dtype]
    g = torch.randn(count, rows, cols, generator=gen).to(dtype).to(dev)
    want = orthogonalize(g, out_dtype=dtype)
    nbytes = lib.yh_orthogonalize_workspace_bytes(count, rows, cols)
    ws = torch.empty(nbytes + 256, dtype=torch.uint8, device=dev)
    ws[nbytes:] = 77
    for ldo, at in ((cols + 8, 0), (cols + 6, 2), (cols + 5, 1)):
        stride = rows * ldo + 8
        out = torch.full((count * stride + 64,), 7.0, dtype=dtype, device=dev)
        _lib.check(lib.yh_orthogonalize(g.data_ptr(), code, rows * cols, cols, out[at:].data_ptr(), code, stride, ldo, count, rows, cols,
                                        *COEFFS, 5, 1e-7, ws.data_ptr(), nbytes, torch.cuda.current_stream(dev).cuda_stream))
        inside = torch.zeros_like(out, dtype=torch.bool)
        for i in range(count):
            where = ((rows, cols), (ldo, 1), at + i * stride)
            assert torch.equal(out.as_strided(*where), want[i]), (ldo, i)
            inside.as_strided(*where).fill_(True)
        assert (out[~inside] == 7).all(), ldo
        assert (ws[nbytes:] == 77).all()


def test_captured_with_16_bit_gradients(dev):
    """The form that holds X in fp16 alone, captured and replayed between eager calls."""
    gen = torch.Generator().manual_seed(13)
    g = torch.randn(2, 513, 1200, generator=gen).to(torch.bfloat16).to(dev)
    orthogonalize(g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = orthogonalize(g)
    for turn in range(4):
        g.copy_(torch.randn(g.shape, generator=gen))
        want = orthogonalize(g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), turn


def test_under_inference_mode(dev):
    with torch.inference_mode():
        p, g, m = (torch.ones(20, 30, device=dev) for _ in range(3))
        muon_step([p], [g], [m], lr=0.1)
        assert (p < 1).all() and torch.allclose(m, torch.full_like(m, 1.95))


def test_streams_and_captured_graphs(dev):
    gen = torch.Generator().manual_seed(11)
    shapes = [(64, 147), (130, 300), (300, 130)]
    gs = [torch.randn(s, generator=gen).to(dev) for s in shapes]
    want = [orthogonalize(g, steps=7) for g in gs]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = [orthogonalize(g, steps=7) for g in gs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # eager and captured steps of the same state, in turn
    new = lambda: ([torch.randn(s, generator=torch.Generator().manual_seed(1)).to(dev) for s in shapes],  # noqa: E731
                   [torch.zeros(s, device=dev) for s in shapes])
    (pe, me), (pc, mc) = new(), new()
    step = lambda ps, ms: [muon_step([p], [g], [m], lr=0.02, weight_decay=0.01) for p, g, m in zip(ps, gs, ms)]  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pc, mc)
    for turn in range(4):
        for g in gs:
            g.copy_(torch.randn(g.shape, generator=gen))
        step(pe, me)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(pe + me, pc + mc)), turn


def test_optimizer(dev):
    """Muon over a network's weights is muon_step shape by shape; its state survives a round trip."""
    from copy import deepcopy

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 16, 3), torch.nn.Conv2d(16, 16, 3), torch.nn.Conv2d(16, 16, 3), torch.nn.Flatten(),
                              torch.nn.Linear(16 * 16, 40)).to(dev)
    weights = [p for p in net.parameters() if p.dim() >= 2]
    twin = deepcopy(weights)
    optim = Muon(weights, lr=0.03, weight_decay=0.02)
    momenta = [torch.zeros_like(p) for p in twin]
    x = torch.randn(4, 3, 10, 10, device=dev)
    for turn in range(3):
        optim.zero_grad()
        net(x).square().sum().backward()
        with torch.no_grad():
            for p, w, m in zip(twin, weights, momenta):
                muon_step([p], [w.grad], [m], lr=0.03, weight_decay=0.02)
        optim.step()
        assert all(torch.equal(p.detach(), w.detach()) for p, w in zip(twin, weights)), turn
        if turn == 1:
            state = deepcopy(optim.state_dict())
            optim = Muon(weights, lr=1.0)
            optim.load_state_dict(state)
    frozen = weights[0].detach().clone()
    optim.zero_grad()
    optim.step()                                          # no gradients: nothing moves
    assert torch.equal(frozen, weights[0].detach())


def test_training_example(dev, capsys, monkeypatch):
    """examples/train_step.py with orthogonalised updates and the last layer in 8 bits runs; its gradients are finite and
    reach every weight."""
    import os
    import sys

    monkeypatch.syspath_prepend(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    train_step = __import__("train_step")
    made = []
    make = train_step.make_backbone
    monkeypatch.setattr(train_step, "make_backbone", lambda *a, **k: made.append(make(*a, **k)) or made[-1])
    train_step.main(["--batch", "2", "--steps", "2", "--width", "0.125", "--optim", "muon", "--int8"])
    assert "detections kept per image" in capsys.readouterr().out
    for name, p in made[0].named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and torch.isfinite(p).all(), name
        assert p.grad.any(), name
    sys.modules.pop("train_step", None)


def test_training_step_of_the_head(dev):
    """Loss and gradient of the head, a Muon step of the layers in front of it, the last layer served in 8 bits."""
    from yolo_amd import Int8Linear

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(256, 300), torch.nn.LeakyReLU(0.1), torch.nn.Linear(300, 1470)).to(dev)
    head = YOLOv1Head(backbone=net)
    x = torch.randn(24, 256, device=dev)
    _, gx, gc, om = (t.to(dev) for t in synth.make_inputs(24, seed=2))
    optim = Muon([net[0].weight, net[2].weight], lr=0.02)
    rest = torch.optim.SGD([net[0].bias, net[2].bias], lr=1e-3)
    for _ in range(2):
        loss = head.get_loss(x, gx, gc, om)
        optim.zero_grad()
        rest.zero_grad()
        loss.backward()
        before = [net[i].weight.detach().clone() for i in (0, 2)]
        grads = [net[i].weight.grad.clone() for i in (0, 2)]
        held = [optim.state[net[i].weight].get("momentum_buffer", torch.zeros_like(before[0])) for i in (0, 2)]
        held = [h.clone() if h.shape == b.shape else torch.zeros_like(b) for h, b in zip(held, before)]
        optim.step()
        rest.step()
        for i, b, g, m in zip((0, 2), before, grads, held):
            wp, _, size = _want(b.cpu(), g.cpu(), m.cpu(), 0.02, 0.95, 0.0, True)
            err = (net[i].weight.detach().cpu().double() - wp).norm().item()
            assert err <= 2.0 ** -22 * (wp.norm().item() + size) + 1e-4 * size
    net.eval()
    with torch.no_grad():
        hidden = net[1](net[0](x))
        layer = Int8Linear.from_linear(net[2])
        dets, count = head.postprocess_linear(hidden, layer, 0.0, 0.5)
        want = head.postprocess(layer(hidden).view(-1, 30, 7, 7), 0.0, 0.5)
    assert torch.equal(dets, want[0]) and torch.equal(count, want[1]) and int(count.sum()) > 0
