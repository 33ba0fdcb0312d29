"""Muon's state: what loading a state dict does, hooks of the user's among it, how momenta lie, and what is refused before any
of it is made.  All but the steps of channels-last weights runs without a GPU."""
import math

import pytest
import torch

from yolo_amd import Muon


def _pair(dtype=torch.bfloat16):
    weights = [torch.nn.Parameter(torch.zeros(3, 5, dtype=dtype)), torch.nn.Parameter(torch.zeros(4, 2))]
    first, second = Muon(weights), Muon(weights, lr=1.0)
    for i, p in enumerate(weights):
        first.state[p]["momentum_buffer"] = torch.full(p.shape, 1.0 + 2.0 ** -20 + i)
    return weights, first, second


def test_a_pre_hook_decides_what_is_loaded():
    weights, first, second = _pair()

    def clear(optim, state_dict):
        state = {k: {"momentum_buffer": torch.zeros_like(v["momentum_buffer"])} for k, v in state_dict["state"].items()}
        return {**state_dict, "state": state}

    second.register_load_state_dict_pre_hook(clear)
    second.load_state_dict(first.state_dict())
    for p in weights:
        assert not second.state[p]["momentum_buffer"].any() and second.state[p]["momentum_buffer"].dtype == torch.float32
    assert first.state[weights[0]]["momentum_buffer"].any()


def test_hooks_run_in_order_and_once():
    weights, first, second = _pair()
    calls = []

    def twice(optim, state_dict):
        calls.append("pre")
        state = {k: {"momentum_buffer": 2 * v["momentum_buffer"]} for k, v in state_dict["state"].items()}
        return {**state_dict, "state": state}

    def after(optim):
        calls.append("post")
        for i, p in enumerate(weights):
            m = optim.state[p]["momentum_buffer"]
            assert m.dtype == torch.float32 and torch.equal(m, torch.full(p.shape, 2 * (1.0 + 2.0 ** -20 + i)))
            m.mul_(0.5)                                   # what a post-hook does stays

    second.register_load_state_dict_pre_hook(twice)
    second.register_load_state_dict_post_hook(after)
    for _ in range(2):
        second.load_state_dict(first.state_dict())
        for i, p in enumerate(weights):
            assert torch.equal(second.state[p]["momentum_buffer"], torch.full(p.shape, 1.0 + 2.0 ** -20 + i))
    assert calls == ["pre", "post"] * 2


def test_a_refused_state_dict_leaves_no_hooks_behind():
    weights, first, second = _pair()
    bad = first.state_dict()
    bad["param_groups"] = []
    for _ in range(2):
        try:
            second.load_state_dict(bad)
            raise AssertionError("loaded")
        except ValueError:
            pass
    second.load_state_dict(first.state_dict())
    for p in weights:
        assert torch.equal(second.state[p]["momentum_buffer"], first.state[p]["momentum_buffer"])
        assert second.state[p]["momentum_buffer"].data_ptr() != first.state[p]["momentum_buffer"].data_ptr()
    assert not second._optimizer_load_state_dict_pre_hooks and not second._optimizer_load_state_dict_post_hooks


@pytest.mark.parametrize("what", ["transposed", "float64", "sparse", "one axis", "every second row"])
def test_a_step_that_is_refused_changes_nothing(what):
    """Every weight is looked at before the first momentum is made (without a GPU the step itself is refused after that)."""
    fine = torch.nn.Parameter(torch.ones(4, 6))
    bad = {"transposed": lambda: torch.zeros(6, 4).t(), "float64": lambda: torch.zeros(4, 6, dtype=torch.float64),
           "every second row": lambda: torch.zeros(8, 6)[::2]}.get(what, lambda: torch.zeros(4, 6))()
    bad = torch.nn.Parameter(bad)
    optim = Muon([fine])
    if what == "one axis":
        bad = torch.nn.Parameter(torch.zeros(6))
    optim.add_param_group(dict(params=[bad]))
    fine.grad, bad.grad = torch.ones_like(fine), torch.ones_like(bad)
    if what == "sparse":
        bad.grad = torch.ones(4, 6).to_sparse()
    word = {"float64": "float64", "sparse": "sparse", "one axis": "two or more axes"}.get(what, "outermost")
    with pytest.raises(ValueError, match=word):
        optim.step()
    assert not any(optim.state.values()) and torch.equal(fine.detach(), torch.ones(4, 6))


def test_momenta_lie_as_their_weights_do():
    weights = [torch.nn.Parameter(torch.randn(8, 3, 5, 5).to(memory_format=torch.channels_last)), torch.nn.Parameter(torch.randn(8, 3, 5, 5))]
    first, second = Muon(weights), Muon(weights)
    momenta = [torch.randn(8, 3, 5, 5) for _ in weights]
    for p, m in zip(weights, momenta):
        first.state[p]["momentum_buffer"] = m
    second.load_state_dict(first.state_dict())
    for p, m in zip(weights, momenta):
        got = second.state[p]["momentum_buffer"]
        assert got.stride() == p.stride() and torch.equal(got, m)


def test_a_momentum_is_not_laid_out_anew_in_a_capture(monkeypatch):
    """Every replay would copy the old one again."""
    p = torch.nn.Parameter(torch.zeros(8, 3, 5, 5))
    p.grad = torch.ones_like(p)
    optim = Muon([p])
    held = optim.state[p]["momentum_buffer"] = torch.ones(8, 3, 5, 5).to(memory_format=torch.channels_last)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        optim.step()
    assert optim.state[p]["momentum_buffer"] is held


def _exact(p, g, m, lr, momentum, wd):
    """The step in 64 bits: (weight, momentum, size of the update)."""
    a, b, c = 3.4445, -4.7750, 2.0315
    m = momentum * m.double() + g.double()
    x = (g.double() + momentum * m).reshape(g.shape[0], -1)
    x = x / (x.norm() + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(5):
        w = x @ x.t()
        x = a * x + (b * w + c * w @ w) @ x
    x = x.t() if tall else x
    step = lr * math.sqrt(max(1.0, p.shape[0] / (p.numel() / p.shape[0])))
    return (1 - lr * wd) * p.double() - step * x.reshape(p.shape), m, step * x.norm().item()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,layout", [((64, 3, 7, 7), torch.channels_last), ((192, 64, 3, 3), torch.channels_last),
                                          ((300, 8, 2, 3), torch.channels_last), ((20, 6, 1, 1), torch.channels_last),
                                          ((40, 5, 2, 3, 4), torch.channels_last_3d)])
@pytest.mark.parametrize("grad_layout", ["same", "contiguous"])
def test_channels_last_weights(dev, shape, layout, grad_layout):
    """The columns of a weight's matrix in another order: the update's columns in that order.  Bounds: 1e-4 of the update's
    norm is its contract; decay, step, their products and the difference round to 2^-22 of the weight and the update;
    momenta round three times (0.95, its product, the sum)."""
    gen = torch.Generator().manual_seed(sum(shape))
    new = lambda scale: (scale * torch.randn(shape, generator=gen))  # noqa: E731
    p0, g0 = [new(0.1), new(0.1)], [[new(1e-2), new(1e-2)] for _ in range(3)]
    weights = [torch.nn.Parameter(p0[0].to(dev).to(memory_format=layout)), torch.nn.Parameter(p0[1].to(dev))]
    optim = Muon(weights, lr=0.05, weight_decay=0.1)
    strides = [p.stride() for p in weights]
    want = [(p, torch.zeros(shape), 0.0) for p in p0]
    for turn, grads in enumerate(g0):
        for p, g in zip(weights, grads):
            p.grad = g.to(dev)
            if grad_layout == "same":
                p.grad = torch.empty_like(p).copy_(p.grad)
        versions = [p._version for p in weights]
        optim.step()
        assert all(p._version > v for p, v in zip(weights, versions))
        for i, (p, g) in enumerate(zip(weights, grads)):
            # from what the step before left
            wp, wm, size = _exact(want[i][0], g, want[i][1], 0.05, 0.95, 0.1)
            m = optim.state[p]["momentum_buffer"]
            assert p.stride() == strides[i]
            assert all(m.is_contiguous(memory_format=f) == p.is_contiguous(memory_format=f) for f in (torch.contiguous_format, layout))
            bound = 2.0 ** -24 * (3 * 0.95 * want[i][1].double().abs() + g.double().abs()) * 1.0001
            assert bool(((m.cpu().double() - wm).abs() <= bound).all())
            err = (p.detach().cpu().double() - wp).norm().item()
            assert err <= 2.0 ** -22 * (wp.norm().item() + size) + 1e-4 * size, turn
            want[i] = (p.detach().cpu().contiguous(), m.cpu().contiguous(), size)
        if turn == 0:                                     # a network moved to the other layout between two steps
            for p in weights:
                p.data = p.data.contiguous() if p.stride() != weights[1].stride() else p.data.to(memory_format=layout)
            strides = [p.stride() for p in weights]
        if turn == 1:
            state = optim.state_dict()
            optim = Muon(weights)
            optim.load_state_dict(state)


@pytest.mark.gpu
def test_captured_steps_of_channels_last_weights(dev):
    gen = torch.Generator().manual_seed(9)
    nets = [torch.nn.Conv2d(16, 40, 3, bias=False).to(dev, memory_format=torch.channels_last) for _ in range(2)]
    nets[1].load_state_dict(nets[0].state_dict())
    weights = [n.weight for n in nets]
    optims = [Muon([w], lr=0.02) for w in weights]
    grads = [torch.empty_like(w) for w in weights]

    def new():
        g = torch.randn(weights[0].shape, generator=gen).to(dev)
        for w, into in zip(weights, grads):
            into.copy_(g)
            w.grad = into

    new()
    for optim in optims:
        optim.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optims[1].step()
    for turn in range(4):
        new()
        optims[0].step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(weights[0].detach(), weights[1].detach()), turn


@pytest.mark.parametrize("shape", [(1, 5), (5,), (1, 1), (3, 4), (5, 3)])
def test_a_momentum_of_another_shape_is_not_loaded(shape):
    weights, first, second = _pair()
    second.load_state_dict(first.state_dict())
    before = [second.state[p]["momentum_buffer"].clone() for p in weights]
    first.state[weights[0]]["momentum_buffer"] = torch.ones(shape)
    with pytest.raises(ValueError, match="momentum of shape"):
        second.load_state_dict(first.state_dict())
    assert all(torch.equal(second.state[p]["momentum_buffer"], b) for p, b in zip(weights, before))
