"""Cases, plain forms and exact values of the operators around the head's linear layers.

The layers in front of the head (convolutions of cout x cin*k*k weights, the two fully connected
layers 50176 -> 4096 -> 1470 of a 7x7x30 head) are served by a product in 8-bit integers and
trained by an orthogonalised update:

* ``linear``: ``yolo_amd.linear_i8`` -- y = sx * sw * (xq @ wq.T) + bias, where xq holds x in 8-bit
  integers with a scale for each row (an image's features) and wq the weights with a scale for
  each row (an output channel).
* ``orthogonalize``: ``yolo_amd.orthogonalize`` -- five Newton-Schulz steps towards the nearest
  matrix with orthonormal rows.
* ``muon``: ``yolo_amd.muon_step`` -- momentum, orthogonalised update and weight step of a list of
  weight matrices of one shape, in place.

``run`` computes them in elementary torch operations while ``own`` is false and calls the package
while it is true; both take what ``prepare`` makes.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
COEFFS = (3.4445, -4.7750, 2.0315)   # of the quintic X <- (a + b XX' + c (XX')^2) X
STEPS = 5
EPS = 1e-7


def listed():
    return [
        # one image through the last layer of the 7x7x30 head: latency
        dict(name="linear 1x4096 to 1470", op="linear", m=1, k=4096, n=1470, x="bf16", out="fp32", bias=True, quantized=False),
        # one image through the first fully connected layer: the weights' bytes are all there is
        dict(name="linear 1x50176 to 4096", op="linear", m=1, k=50176, n=4096, x="fp16", out="fp16", bias=True, quantized=False),
        # a training-sized batch through it
        dict(name="linear 64x50176 to 4096", op="linear", m=64, k=50176, n=4096, x="bf16", out="bf16", bias=True, quantized=False),
        # sizes that no tile divides, features that arrive in 8 bits
        dict(name="linear 333x1000 to 777", op="linear", m=333, k=1000, n=777, x="int8", out="bf16", bias=False, quantized=True),
        # the headline batch of the head through its last layer, in the head's own type
        dict(name="linear 4096x4096 to 1470", op="linear", m=4096, k=4096, n=1470, x="fp32", out="fp32", bias=True, quantized=False),
        # bulk evaluation: a square layer, a large batch
        dict(name="linear 8192x4096 to 4096", op="linear", m=8192, k=4096, n=4096, x="bf16", out="bf16", bias=False, quantized=False),
        # the first convolution's gradient: the smallest matrix of the network
        dict(name="orthogonalize 64x147", op="orthogonalize", batch=1, rows=64, cols=147, g="fp32"),
        # the four 256 -> 512 convolutions of one stage at once
        dict(name="orthogonalize 4x512x2304", op="orthogonalize", batch=4, rows=512, cols=2304, g="bf16"),
        # the last layer as torch stores it transposed (taller than wide), an odd number of rows
        dict(name="orthogonalize 4096x1470", op="orthogonalize", batch=1, rows=4096, cols=1470, g="fp32"),
        # the first fully connected layer: the largest matrix of the network
        dict(name="orthogonalize 4096x50176", op="orthogonalize", batch=1, rows=4096, cols=50176, g="bf16"),
        # an early convolution's update
        dict(name="muon 192x576", op="muon", count=1, rows=192, cols=576, p="fp32", g="fp32", nesterov=True),
        # the four 1024 -> 1024 convolutions at the end of the network
        dict(name="muon 4x1024x9216", op="muon", count=4, rows=1024, cols=9216, p="fp32", g="bf16", nesterov=True),
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "orthogonalize", "muon"])
    if op == "linear":
        m, k = _spread(rng, 1, 8192), _spread(rng, 64, 50176)
        n = _spread(rng, 16, 4096)
        while m * n * k > 8192 * 4096 * 4096:
            m = (m + 1) // 2
        x = rng.choice(["fp32", "bf16", "fp16", "int8"])
        return dict(op=op, m=m, k=k, n=n, x=x, out=rng.choice(["fp32", "bf16", "fp16"]), bias=rng.random() < 0.5,
                    quantized=x == "int8")
    rows, cols = _spread(rng, 16, 4096), _spread(rng, 16, 9216)
    count = rng.choice([1, 1, 2, 3, 5])
    while count * rows * cols > 4 * 1024 * 9216:
        count, cols = (count + 1) // 2, (cols + 1) // 2
    g = rng.choice(["fp32", "bf16", "fp16"])
    if op == "orthogonalize":
        return dict(op=op, batch=count, rows=rows, cols=cols, g=g)
    return dict(op=op, count=count, rows=rows, cols=cols, p=rng.choice(["fp32", "bf16"]), g=g, nesterov=rng.random() < 0.7)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows_i8(t):
    """t (rows, k) as 8-bit integers and a scale for each row, rows at a stride of a multiple of 64 bytes."""
    k = t.shape[1]
    top = t.abs().amax(1, keepdim=True).clamp_min(1e-30)
    q = torch.zeros(t.shape[0], (k + 63) // 64 * 64, dtype=torch.int8, device=t.device)
    q[:, :k] = torch.round(t * (127.0 / top)).to(torch.int8)
    return q[:, :k], (top / 127.0).squeeze(1)


def _features(m, k, gen):
    """What the layers meet: activations behind a leaky ReLU, of another size from image to image."""
    x = torch.nn.functional.leaky_relu(torch.randn(m, k, generator=gen, device="cuda"), 0.1)
    return x * torch.exp(0.5 * torch.randn(m, 1, generator=gen, device="cuda"))


def _gradients(batch, rows, cols, gen):
    """Weight gradients: a few strong directions over a floor of noise."""
    rank = min(16, rows, cols)
    u = torch.randn(batch, rows, rank, generator=gen, device="cuda")
    v = torch.randn(batch, rank, cols, generator=gen, device="cuda")
    strength = torch.logspace(0, -1.5, rank, device="cuda")
    noise = torch.randn(batch, rows, cols, generator=gen, device="cuda")
    return 1e-3 * (torch.matmul(u * strength, v) + 0.1 * noise)


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        w, w_scale = _rows_i8(torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k))
        x, x_scale = _features(m, k, gen), None
        if case["quantized"]:
            x, x_scale = _rows_i8(x)
        else:
            x = x.to(DTYPES[case["x"]])
        bias = torch.randn(n, generator=gen, device="cuda") if case["bias"] else None
        return dict(op="linear", x=x, x_scale=x_scale, w=w, w_scale=w_scale, bias=bias, out=DTYPES[case["out"]])
    if case["op"] == "orthogonalize":
        g = _gradients(case["batch"], case["rows"], case["cols"], gen).to(DTYPES[case["g"]])
        return dict(op="orthogonalize", g=g)
    count, rows, cols = case["count"], case["rows"], case["cols"]
    g = _gradients(count, rows, cols, gen).to(DTYPES[case["g"]])
    buf = 5 * _gradients(count, rows, cols, gen)
    bound = 1 / math.sqrt(cols)           # what a fresh convolution or linear layer starts with
    p = (bound * (2 * torch.rand(count, rows, cols, generator=gen, device="cuda") - 1)).to(DTYPES[case["p"]])
    return dict(op="muon", p=list(p.unbind(0)), g=list(g.unbind(0)), buf=list(buf.unbind(0)), lr=0.02, momentum=0.95,
                weight_decay=0.01, nesterov=case["nesterov"])


def _linear(s):
    if s["x_scale"] is None:
        x = s["x"].double()               # a quotient next to a border between two whole numbers needs 64 bits
        top = x.abs().amax(1, keepdim=True)
        q = torch.where(top > 0, torch.round(x * 127 / top), 0.0).float()
        x_scale = (top.float() / 127).squeeze(1)
    else:
        q, x_scale = s["x"].float(), s["x_scale"]
    y = torch.matmul(q, s["w"].float().t()) * x_scale[:, None] * s["w_scale"]
    return (y if s["bias"] is None else y + s["bias"]).to(s["out"])


def _newton_schulz(g):
    """(batch, rows, cols) in 32 bits."""
    a, b, c = COEFFS
    norm = g.double().square().sum((1, 2), keepdim=True).sqrt()
    x = (g / (norm + EPS)).float()
    wide = x.shape[1] <= x.shape[2]
    x = x if wide else x.transpose(1, 2).contiguous()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x if wide else x.transpose(1, 2)


def _muon(s):
    g = torch.stack(s["g"]).float()
    buf = s["momentum"] * torch.stack(s["buf"]) + g
    update = _newton_schulz(g + s["momentum"] * buf if s["nesterov"] else buf)
    rows, cols = g.shape[1:]
    step = s["lr"] * math.sqrt(max(1.0, rows / cols))
    p = torch.stack(s["p"]).float() * (1 - s["lr"] * s["weight_decay"]) - step * update
    p = p.to(s["p"][0].dtype)
    torch._foreach_copy_(s["p"], list(p.unbind(0)))
    torch._foreach_copy_(s["buf"], list(buf.unbind(0)))
    return {"p": s["p"], "buf": s["buf"]}


def run(state):
    s = state
    if own:
        import yolo_amd

        if s["op"] == "linear":
            return yolo_amd.linear_i8(s["x"], s["w"], s["w_scale"], bias=s["bias"], x_scale=s["x_scale"], out_dtype=s["out"])
        if s["op"] == "orthogonalize":
            return yolo_amd.orthogonalize(s["g"], steps=STEPS, coeffs=COEFFS, eps=EPS)
        yolo_amd.muon_step(s["p"], s["g"], s["buf"], lr=s["lr"], momentum=s["momentum"], weight_decay=s["weight_decay"],
                           nesterov=s["nesterov"], steps=STEPS, coeffs=COEFFS, eps=EPS)
        return {"p": s["p"], "buf": s["buf"]}
    if s["op"] == "linear":
        return _linear(s)
    if s["op"] == "orthogonalize":
        return _newton_schulz(s["g"].float()).to(torch.bfloat16)
    return _muon(s)


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2, "int8": 1}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        scales = 4 * (n + (m if case["quantized"] else 0) + (n if case["bias"] else 0))
        return {"bytes": m * k * size[case["x"]] + n * k + m * n * size[case["out"]] + scales, "flops": 2 * m * n * k}
    count = case["batch"] if case["op"] == "orthogonalize" else case["count"]
    short, long = sorted((case["rows"], case["cols"]))
    # XX' is symmetric: half a product. Either every step forms it and applies its polynomial, or one XX' is formed,
    # the steps run on symmetric short x short matrices alone (four products a step, two in the last) and one product applies them.
    stepwise = STEPS * (3 * short * short * long + short ** 3)
    at_once = 3 * short * short * long + (4 * STEPS - 3) * short ** 3
    flops = count * min(stepwise, at_once)
    numbers = count * short * long
    if case["op"] == "orthogonalize":
        return {"bytes": numbers * (size[case["g"]] + 2), "flops": flops}
    return {"bytes": numbers * (size[case["g"]] + 8 + 2 * size[case["p"]]), "flops": flops}


def _exact_polar(g):
    a, b, c = COEFFS
    out = torch.empty_like(g)
    for i in range(g.shape[0]):
        x = g[i] / (torch.linalg.vector_norm(g[i]) + EPS)
        tall = x.shape[0] > x.shape[1]
        x = x.t().contiguous() if tall else x
        for _ in range(STEPS):
            w = x @ x.t()
            x = a * x + (b * w + c * (w @ w)) @ x
        out[i] = x.t() if tall else x
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        if case["quantized"]:
            values = s["x"].double() * s["x_scale"].double()[:, None]
        else:
            x = s["x"].double()
            top = x.abs().max(1).values[:, None]
            values = torch.round(127 * x / top) * (top / 127)
        y = values @ (s["w"].double() * s["w_scale"].double()[:, None]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "orthogonalize":
        return _exact_polar(s["g"].double())
    g, buf, p = (torch.stack(s[name]).double() for name in ("g", "buf", "p"))
    buf = s["momentum"] * buf + g
    update = _exact_polar(g + s["momentum"] * buf) if case["nesterov"] else _exact_polar(buf)
    scale = max(1.0, case["rows"] / case["cols"]) ** 0.5
    p = p * (1 - s["lr"] * s["weight_decay"]) - s["lr"] * scale * update
    return {"p": list(p), "buf": list(buf)}
