"""Preference and policy tuning: refusals and host logic beside those of the operators' own tests."""
from __future__ import annotations

from contextlib import nullcontext

import pytest
import torch

from molt_b200 import _native

A, B, C, D, E = (0x10000 * i for i in range(1, 6))   # addresses that are only checked


def test_counted_adamw_needs_a_count(native_library):
    for skipped in (None, E + 4):
        rc = native_library.molt_adamw_step_counted(A, B, C, D, 4, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, skipped, 0)
        assert rc == _native.E_VALUE and b"skipped is NULL or not 8-byte aligned" in native_library.molt_last_error()
    for change, word in (((A, B, C, D, 3), b"multiple of 4"), ((None, B, C, D, 4), b"NULL"), ((A + 4, B, C, D, 4), b"16-byte aligned")):
        rc = native_library.molt_adamw_step_counted(*change, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, E, 0)
        assert rc == _native.E_VALUE and word in native_library.molt_last_error()


def _model(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(3, 4), torch.nn.Linear(4, 2))


def test_hooks_of_parameters_take_part_in_a_recording():
    """Both kinds of tensor hooks, several on one parameter, a shared parameter, hooks taken off again: the gradients inside
    are those of a backward pass outside, hooks run in the same order and get the parameter itself."""
    from molt_b200.qlora_step import leaves_of_its_own

    def triple(p):
        p.grad.mul_(3)

    x = torch.randn(5, 3)
    runs = []
    for inside in (False, True):
        model = _model()
        model.add_module("again", model[1])                       # the same parameters under two names
        weight, bias, other = model[0].weight, model[0].bias, model[1].weight
        told = []
        weight.register_hook(lambda g: torch.full_like(g, 7.0))
        weight.register_hook(lambda g: g * 2)
        weight.register_hook(lambda g: g * 0).remove()
        bias.register_post_accumulate_grad_hook(lambda p: told.append(p is bias))
        bias.register_post_accumulate_grad_hook(triple)
        bias.register_post_accumulate_grad_hook(lambda p: told.append("gone")).remove()
        other.register_hook(lambda g: told.append("other"))
        for p in model.parameters():
            p.grad = torch.zeros_like(p)
        grads = [p.grad for p in model.parameters()]
        with leaves_of_its_own(model) if inside else nullcontext():
            model[1](model[0](x)).square().sum().backward()
        assert all(p.grad is g for p, g in zip(model.parameters(), grads))
        assert told == ["other", True] and bool((weight.grad == 14).all())
        runs.append([g.clone() for g in grads])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_hook_that_takes_the_gradient_away_does_so_in_a_recording():
    """The optimizer inside the backward pass: the hook uses the parameter, and drops its gradient."""
    from molt_b200.qlora_step import leaves_of_its_own

    model = _model()
    weight = model[0].weight
    before = weight.detach().clone()

    def step(p):
        with torch.no_grad():
            p.sub_(p.grad, alpha=0.1)
        p.grad = None

    weight.register_post_accumulate_grad_hook(step)
    with leaves_of_its_own(model):
        model(torch.randn(5, 3)).square().sum().backward()
    assert weight.grad is None and not torch.equal(weight.detach(), before)


def test_gradients_made_in_a_recording_belong_to_the_parameters():
    """A parameter that had no gradient has the recorded one afterwards, as after a backward pass without stand-ins."""
    from molt_b200.qlora_step import leaves_of_its_own

    model, plain = _model(), _model()
    kept = model[0].weight.grad = torch.ones_like(model[0].weight)
    plain[0].weight.grad = torch.ones_like(kept)
    x = torch.randn(5, 3)
    with leaves_of_its_own(model):
        model(x).square().sum().backward()
    plain(x).square().sum().backward()
    assert model[0].weight.grad is kept
    assert all(torch.equal(p.grad, q.grad) for p, q in zip(model.parameters(), plain.parameters()))


class _Recording:
    """Stands in for a CUDA graph: what runs inside is run."""

    def replay(self):
        raise AssertionError("nothing is replayed here")


@pytest.fixture
def host_step(monkeypatch, native_library):
    from molt_b200.data_parallel import GradArena
    from molt_b200.qlora_step import QLoRAStep

    monkeypatch.setattr(torch.cuda, "CUDAGraph", _Recording)
    monkeypatch.setattr(torch.cuda, "graph", lambda graph: nullcontext())
    step = object.__new__(QLoRAStep)
    step.model, step.world, step._graph, step._static_loss, step.graph_launches = _model(), 1, None, None, 0
    step.arena = GradArena(step.model.parameters())

    class Objective:
        def loss(self, model, world, layer_done, tokens, targets):
            if targets.shape != tokens.shape:
                raise ValueError("not for this objective")
            return (model(tokens) * targets.sum()).sum()

    step.objective = Objective()
    return step


def test_recording_writes_into_the_arena_after_gradients_were_dropped(host_step):
    """``zero_grad()`` drops the gradients by default: the recorded backward pass must fill the arena all the same."""
    step = host_step
    step.model.zero_grad()
    step._capture(torch.ones(5, 3), torch.ones(5, 3))
    assert all(p.grad is view for p, view in zip(step.arena.params, step.arena.views))
    assert all(bool(view.any()) for view in step.arena.views)


def test_recording_that_failed_leaves_none_behind(host_step):
    """Inputs that the objective refuses: the next step records anew instead of replaying nothing."""
    step = host_step
    with pytest.raises(ValueError, match="not for this objective"):
        step._capture(torch.ones(5, 3), torch.ones(4, 3))
    assert step._graph is None and step._static_loss is None
    step._capture(torch.ones(5, 3), torch.ones(5, 3))
    assert isinstance(step._graph, _Recording) and step._static_loss is not None


def test_no_stream_is_named_for_a_device_that_is_not_cuda(monkeypatch):
    """A host tensor must not reach a kernel by way of the current device's stream."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 40 + index, raising=False)
    for device in (torch.device("cpu"), "cpu", torch.device("meta")):
        with pytest.raises(ValueError, match="cuda"):
            _native.stream_handle(device)
    assert [_native.stream_handle(d) for d in (None, "cuda", torch.device("cuda:1"), "cuda:2")] == [40, 40, 41, 42]
