"""Muon's state without a GPU: what loading a state dict does, hooks of the user's among it."""
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
