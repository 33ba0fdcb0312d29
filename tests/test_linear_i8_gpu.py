"""The linear layer's product in 8-bit integers against its definition in 64 bits.

Bounds.  The integer sum is exact.  Its conversion to fp32, the two scales and the bias round once each: 3 * 2^-24 of
|acc s t| (two factors of (1 + 2^-24) on top are below one more 2^-24) and 2^-24 of the sum with the bias; the result is
then off by at most half a step of its type.  The quantised values and their scales have one right answer."""
import pytest
import torch

from yolo_amd import Int8Linear, YOLOv1Head, _lib, linear_i8, quantize_rows, synth

pytestmark = pytest.mark.gpu
FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def quantized(x):
    """The definition, in 64 bits: (whole numbers, fp32 scale)."""
    x = x.double().cpu()
    top = x.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(127 * x / top.clamp_min(1e-300)), 0.0)
    return q, top[:, 0].float() / 127


def weights(n, k, gen, dev):
    return quantize_rows((torch.randn(n, k, generator=gen) / k ** 0.5).to(dev))


def check(y, q, s, w, t, bias):
    acc = q.double() @ w.cpu().double().t()
    scaled = acc * s.double().cpu()[:, None] * t.cpu().double()
    want = scaled if bias is None else scaled + bias.cpu().double()
    half = torch.finfo(y.dtype).eps / 2 if y.dtype != torch.float32 else 0.0
    bound = 4 * 2.0 ** -24 * scaled.abs() + 2 * 2.0 ** -24 * want.abs()
    bound = bound + half * (want.abs() + bound) + (2.0 ** -25 if y.dtype == torch.float16 else 0.0) + 1e-37
    err = (y.cpu().double() - want).abs()
    assert bool((err <= bound).all()), (err / bound).max()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 4096), (3, 147), (5, 128), (2, 129), (300, 1000), (2, 9000), (1, 50176), (2, 131071)])
def test_quantize_rows_is_the_definition(dev, dtype, m, k):
    gen = torch.Generator().manual_seed(m * k)
    x = torch.nn.functional.leaky_relu(torch.randn(m, k, generator=gen), 0.1).to(dtype)
    x[:, k // 2] = x[:, 0] / 2                      # a value at a border between two whole numbers when x[:, 0] is the largest
    x[0, 0] = x[0].abs().max()
    q, s = quantize_rows(x.to(dev))
    wq, ws = quantized(x)
    assert q.shape == (m, k) and q.stride(0) % 128 == 0
    assert torch.equal(q.cpu().double(), wq) and torch.equal(s.cpu(), ws)
    rows = torch.as_strided(q, (m, q.stride(0)), (q.stride(0), 1))
    assert not rows[:, k:].any()


def test_quantize_rows_ties_zeros_and_what_is_not_a_number(dev):
    # 127 x / 254 = x / 2: every odd whole number is a tie, to even
    x = torch.arange(-254, 255, dtype=torch.float32).repeat(5, 1)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 7] = float("-inf")
    x[4] *= 2.0 ** -140                             # subnormal numbers keep their quotients
    q, s = quantize_rows(x.to(dev))
    want = torch.round(torch.arange(-254, 255, dtype=torch.float64) / 2)
    for row in (0, 4):
        assert torch.equal(q[row].cpu().double(), want)
    assert s[0].item() == 2.0 and not q[1:4].any() and s[1].item() == 0.0
    assert torch.isnan(s[2:4]).all()


SHAPES = [(1, 1, 1), (1, 4096, 1470), (1, 64, 17), (2, 129, 5), (7, 50176, 33), (16, 1000, 64), (17, 640, 100),
          (33, 147, 129), (64, 4096, 257), (65, 300, 1470), (128, 128, 128), (129, 2048, 130), (300, 4096, 1470), (1000, 513, 777)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype,out,bias", [(torch.bfloat16, torch.bfloat16, True), (torch.float32, torch.float32, True),
                                            (torch.float16, torch.float32, False), (torch.float32, torch.float16, False)])
def test_linear_i8(dev, m, k, n, dtype, out, bias):
    gen = torch.Generator().manual_seed(m + k + n)
    x = torch.nn.functional.leaky_relu(torch.randn(m, k, generator=gen), 0.1).to(dtype)
    w, t = weights(n, k, gen, dev)
    b = torch.randn(n, generator=gen) if bias else None
    y = linear_i8(x.to(dev), w, t, bias=None if b is None else b.to(dev), out_dtype=out)
    assert y.shape == (m, n) and y.dtype == out
    q, s = quantized(x)
    check(y, q, s, w, t, b)
    again = linear_i8(x.to(dev), w, t, bias=None if b is None else b.to(dev), out_dtype=out)
    assert torch.equal(y, again)


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_i8_of_quantized_features(dev, m, k, n):
    """int8 in, and whatever lies behind a row of x or of the weight does not matter."""
    gen = torch.Generator().manual_seed(m * 3 + k + n)
    kp = (k + 15) // 16 * 16
    xs = torch.randint(-128, 128, (m, kp), generator=gen, dtype=torch.int8).to(dev)
    w_ = torch.randint(-128, 128, (n, kp), generator=gen, dtype=torch.int8).to(dev)
    s, t = torch.rand(m, generator=gen).to(dev), torch.rand(n, generator=gen).to(dev)
    y = linear_i8(xs[:, :k], w_[:, :k], t, x_scale=s)
    assert y.dtype == torch.float32
    check(y, xs[:, :k].cpu(), s, w_[:, :k], t, None)


@pytest.mark.parametrize("m,k,n,dtype", [(1, 65536, 40, torch.bfloat16), (1, 65537, 40, torch.float32), (1, 131071, 20, torch.float16),
                                         (3, 4096, 40, torch.float32), (4, 4096, 40, torch.float16), (64, 700, 40, torch.bfloat16),
                                         (16, 4096, 40, torch.int8), (16, 4097, 40, torch.int8), (1, 65536, 40, torch.int8)])
def test_on_both_sides_of_what_is_brought_in_on_the_way(dev, m, k, n, dtype):
    """The largest rows that the product's workgroups bring into LDS themselves, and the first that they do not."""
    gen = torch.Generator().manual_seed(m + k)
    w, t = weights(n, k, gen, dev)
    if dtype == torch.int8:
        q, s = torch.randint(-128, 128, (m, k), generator=gen, dtype=torch.int8), torch.rand(m, generator=gen)
        y = linear_i8(q.to(dev), w, t, x_scale=s.to(dev))
        check(y, q, s.to(dev), w, t, None)
    else:
        x = torch.randn(m, k, generator=gen).to(dtype)
        q, s = quantized(x)
        check(linear_i8(x.to(dev), w, t, out_dtype=torch.float32), q, s, w, t, None)


def test_the_largest_sum_there_is(dev):
    k = 131071
    x = torch.full((2, k + 1), -128, dtype=torch.int8, device=dev)
    one = torch.ones(2, device=dev)
    y = linear_i8(x[:, :k], x[:, :k], one, x_scale=one)
    assert torch.equal(y, torch.full((2, 2), float(128 * 128 * k), device=dev))
    x[1] = 127
    y = linear_i8(x[:, :k], x[:, :k], one, x_scale=one)
    want = torch.tensor([[128 * 128 * k, -128 * 127 * k], [-128 * 127 * k, 127 * 127 * k]], dtype=torch.float64)
    assert torch.equal(y.cpu(), want.float())


def test_rows_that_are_not_numbers_and_rows_of_zeros(dev):
    gen = torch.Generator().manual_seed(5)
    w, t = weights(70, 300, gen, dev)
    x = torch.randn(6, 300, generator=gen)
    x[1] = 0
    x[2, 299] = float("inf")
    x[4, 0] = float("nan")
    b = torch.randn(70, generator=gen).to(dev)
    y = linear_i8(x.to(dev), w, t, bias=b)
    assert torch.isnan(y[[2, 4]]).all() and torch.isfinite(y[[0, 1, 3, 5]]).all()
    assert torch.equal(y[1], b)
    clean = linear_i8(x[[0, 3]].to(dev), w, t, bias=b)
    assert torch.equal(y[[0, 3]], clean)


def test_shapes_and_strides(dev):
    gen = torch.Generator().manual_seed(6)
    w, t = weights(40, 96, gen, dev)
    x = torch.randn(3, 5, 96, generator=gen).to(dev)
    want = linear_i8(x.view(15, 96), w, t)
    assert torch.equal(linear_i8(x, w, t), want.view(3, 5, 40))
    assert torch.equal(linear_i8(x[1, 2], w, t), want[7])
    odd = torch.empty(15 * 96 + 1, device=dev)[1:].view(15, 96)       # not on 16 bytes
    odd.copy_(x.view(15, 96))
    assert torch.equal(linear_i8(odd, w, t), want)
    wide = torch.randn(15, 203, generator=gen).to(dev)
    wide[:, 3:99] = x.view(15, 96)                                    # rows at an odd distance, not on 16 bytes
    assert torch.equal(linear_i8(wide[:, 3:99], w, t), want)
    assert torch.equal(linear_i8(x[:, 1], w, t), want.view(3, 5, 40)[:, 1])
    assert torch.equal(linear_i8(x[0, :1].expand(4, 96), w, t), want[:1].expand(4, 40))
    assert linear_i8(x[:0], w, t).shape == (0, 5, 40)
    assert linear_i8(x[0], w[:0], t[:0]).shape == (5, 0)
    assert torch.equal(linear_i8(x.view(15, 96), w[7:8], t[7:8])[:, 0], want[:, 7])
    for bad in (w[:, 1:], w.t(), w[:, :95], w.float(), torch.zeros(40, 97, dtype=torch.int8, device=dev)[:, :96]):
        with pytest.raises(ValueError):
            linear_i8(x, bad, t)
    with pytest.raises(ValueError, match="last axis"):
        linear_i8(x.transpose(1, 2).contiguous().transpose(1, 2), w, t)
    with pytest.raises(ValueError, match="gradient"):
        linear_i8(x.requires_grad_(True), w, t)
    # rows of the weight that end with the memory: 16-byte rows of an exact allocation, and one byte too few
    store = torch.zeros(32, dtype=torch.int8, device=dev)
    linear_i8(torch.ones(2, 10, device=dev), store.as_strided((2, 10), (16, 1)), t[:2])
    short = torch.zeros(31, dtype=torch.int8, device=dev)
    with pytest.raises(ValueError, match="room"):
        linear_i8(torch.ones(2, 10, device=dev), short.as_strided((2, 10), (16, 1)), t[:2])


@pytest.mark.parametrize("m", [3, 70, 300])
def test_what_lies_between_the_rows_of_y_stays(dev, m):
    gen = torch.Generator().manual_seed(8)
    lib, k, n, ldy = _lib.load(), 200, 50, 61
    w, t = weights(n, k, gen, dev)
    x = torch.randn(m, k, generator=gen).to(dev)
    y = torch.full((m + 1, ldy), 7.0, device=dev)
    ws = torch.empty(lib.yh_linear_i8_workspace_bytes(_lib.YH_F32, m, n, k), dtype=torch.uint8, device=dev)
    _lib.check(lib.yh_linear_i8(x.data_ptr(), _lib.YH_F32, k, None, w.data_ptr(), w.stride(0), t.data_ptr(), None, y.data_ptr(),
                                _lib.YH_F32, ldy, m, n, k, ws.data_ptr(), ws.numel(), torch.cuda.current_stream(dev).cuda_stream))
    assert torch.equal(y[:m, :n], linear_i8(x, w, t))
    assert (y[:m, n:] == 7).all() and (y[m] == 7).all()


def test_offsets_past_32_bits(dev):
    gen = torch.Generator().manual_seed(9)
    m, k = 45000, 50176
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=dev)          # 4.5 GB
    w, t = weights(16, k, gen, dev)
    rows = [0, 1, 21400, 21401, 42799, 42800, 42801, m - 1]          # 2^31 and 2^32 bytes lie among them
    some = torch.randn(len(rows), k, generator=gen).to(torch.bfloat16)
    x[rows] = some.to(dev)
    y = linear_i8(x, w, t, out_dtype=torch.float32)
    q, s = quantized(some)
    check(y[rows], q, s, w, t, None)
    y[rows] = 0
    assert not y.any()


def test_streams_and_captured_graphs(dev):
    gen = torch.Generator().manual_seed(10)
    w, t = weights(1470, 4096, gen, dev)
    xs = [torch.randn(m, 4096, generator=gen).to(dev) for m in (1, 48, 200)]
    want = [linear_i8(x, w, t) for x in xs]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = [linear_i8(x, w, t) for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for x in xs:                                                      # every graph has a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, linear_i8(x, w, t)))
    for turn in range(3):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=gen))
        want = [linear_i8(x, w, t) for x in xs]
        for g, y in graphs:
            y.fill_(float("nan"))
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, v) for (_, y), v in zip(graphs, want)), turn


@pytest.mark.parametrize("mode", [0, 1])
def test_features_to_detections(dev, mode):
    """The last layer in 8 bits and the decode kernel: the detections are those of postprocess on the same product."""
    torch.manual_seed(0)
    head = YOLOv1Head()
    last = torch.nn.Linear(512, 1470).to(dev)
    layer = Int8Linear.from_linear(last)
    features = torch.nn.functional.leaky_relu(4 * torch.randn(37, 512, device=dev), 0.1)
    got = head.postprocess_linear(features, layer, 0.5, 0.5, mode, return_idx=True)
    y = layer(features)
    want = head.postprocess(y.view(-1, 30, 7, 7), 0.5, 0.5, mode, return_idx=True)
    # the decode adds the bias in fp32 as the product does
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(got[1].sum()) > 0
    # each weight is off by half a step at most and each feature too: the product's error is a sum of 512 such products
    exact = last(features)
    step_w = layer.weight_scale / 2
    step_x = features.abs().amax(1) / 254
    bound = (features.abs().sum(1)[:, None] * step_w + step_x[:, None] * last.weight.abs().sum(1)
             + 512 * step_x[:, None] * step_w) * 1.0001 + 1e-4
    assert ((y - exact).abs() <= bound).all()
    state = {k: v.clone() for k, v in layer.state_dict().items()}
    other = Int8Linear(torch.zeros_like(layer.weight), torch.zeros_like(layer.weight_scale), torch.zeros(1470, device=dev))
    other.load_state_dict(state)
    assert torch.equal(other(features), y)
