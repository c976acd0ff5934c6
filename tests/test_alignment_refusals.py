"""Refusals of the entry points for preference and policy tuning: every one of them is made on the host, before any
launch, so no device is needed (the addresses below are never followed)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from molt_b200 import _native
from molt_b200.core.errors import CapabilityError

A, B, C, D, E = (0x7000_0000 + 0x100_0000 * i for i in range(5))   # addresses that nothing reads


def _strides(*values):
    return (ctypes.c_int64 * len(values))(*values)


def _refused(code, expected, word):
    message = _native.library().molt_last_error()
    assert code == expected, (code, message)
    assert word.encode() in message, message


@pytest.mark.parametrize("change,expected,word", [
    ({"rows": -1}, _native.E_VALUE, "shape"), ({"vocab": 0}, _native.E_VALUE, "shape"),
    ({"rows": (1 << 27) + 1}, _native.E_CAPABILITY, "2^27"), ({"vocab": (1 << 30) + 1}, _native.E_CAPABILITY, "2^30"),
    ({"dtype": 2}, _native.E_CAPABILITY, "bf16 or fp32"), ({"temperature": 0.0}, _native.E_VALUE, "temperature"),
    ({"temperature": -1.0}, _native.E_VALUE, "temperature"), ({"temperature": float("nan")}, _native.E_VALUE, "temperature"),
    ({"temperature": float("inf")}, _native.E_VALUE, "temperature"), ({"temperature": 1e-39}, _native.E_VALUE, "temperature"),
    ({"temperature": 1e38}, _native.E_VALUE, "temperature"), ({"ids": B + 4}, _native.E_VALUE, "aligned"),
    ({"logits": None}, _native.E_VALUE, "NULL"), ({"ids": None}, _native.E_VALUE, "NULL"),
    ({"logprob": None}, _native.E_VALUE, "NULL"), ({"stride": 99}, _native.E_VALUE, "overlap"),
    ({"logits": A + 1}, _native.E_VALUE, "aligned"), ({"grad": None}, _native.E_VALUE, "NULL"),
    ({"grad": C + 1}, _native.E_VALUE, "aligned"), ({"grad_stride": 99}, _native.E_VALUE, "overlap"),
    ({"grad_stride": 0}, _native.E_VALUE, "overlap"), ({"grad": A + 2}, _native.E_VALUE, "overlaps"),
    ({"grad": A, "grad_stride": 104}, _native.E_VALUE, "overlaps"), ({"grad": A + 2 * 50}, _native.E_VALUE, "overlaps"),
    ({"grad": A - 2 * 300}, _native.E_VALUE, "overlaps"), ({"groups": (-1, 0)}, _native.E_VALUE, "group_rows"),
    ({"groups": (2, 99)}, _native.E_VALUE, "groups"), ({"groups": (2, -200)}, _native.E_VALUE, "groups"),
    ({"grad": A, "groups": (2, 300)}, _native.E_VALUE, "overlaps"), ({"grad": A + 2 * 700, "groups": (1, 300)}, _native.E_VALUE, "overlaps"),
    ({"grad": A + 2 * 100, "stride": 200, "grad_stride": 200, "groups": (2, 500)}, _native.E_VALUE, "overlaps")])
def test_token_logprob_refusals(native_library, change, expected, word):
    call = dict(logits=A, dtype=_native.DTYPE_BF16, stride=100, ids=B, temperature=1.0, logprob=D, grad=C, grad_stride=100,
                rows=4, vocab=100, groups=(0, 0))
    call.update(change)
    c = call
    lib = native_library
    _refused(lib.molt_token_logprob_grad(c["logits"], c["dtype"], c["stride"], *c["groups"], c["ids"], None, c["temperature"], c["logprob"],
                                         c["grad"], c["grad_stride"], c["rows"], c["vocab"], 0), expected, word)
    if "logprob" not in change:
        _refused(lib.molt_token_logprob_bwd(c["logits"], c["dtype"], c["stride"], *c["groups"], c["ids"], E, E, c["temperature"], c["grad"],
                                            c["grad_stride"], c["rows"], c["vocab"], 0), expected, word)
    if not set(change) & {"grad", "grad_stride"}:
        _refused(lib.molt_token_logprob_fwd(c["logits"], c["dtype"], c["stride"], *c["groups"], c["ids"], c["temperature"], c["logprob"], None,
                                            c["rows"], c["vocab"], 0), expected, word)


def test_token_logprob_stats_are_aligned(native_library):
    lib = native_library
    _refused(lib.molt_token_logprob_fwd(A, 0, 100, 0, 0, B, 1.0, D, E + 4, 4, 100, 0), _native.E_VALUE, "stats")
    _refused(lib.molt_token_logprob_bwd(A, 0, 100, 0, 0, B, E + 4, E, 1.0, C, 100, 4, 100, 0), _native.E_VALUE, "stats")


def test_token_logprob_of_no_rows_is_no_launch(native_library):
    lib = native_library
    before = lib.molt_launch_count()
    assert lib.molt_token_logprob_fwd(None, 0, 0, 0, 0, None, 1.0, None, None, 0, 10, 0) == 0
    assert lib.molt_token_logprob_grad(None, 0, 0, 0, 0, None, None, 1.0, None, None, 0, 0, 10, 0) == 0
    assert lib.molt_token_logprob_bwd(None, 0, 0, 0, 0, None, None, None, 1.0, None, 0, 0, 10, 0) == 0
    assert lib.molt_launch_count() == before


@pytest.mark.parametrize("change,expected,word", [
    ({"batch": 0}, _native.E_VALUE, "no sequence"), ({"batch": -1}, _native.E_VALUE, "negative"),
    ({"seq": -1}, _native.E_VALUE, "negative"), ({"batch": 1 << 31}, _native.E_CAPABILITY, "2^31"),
    ({"seq": (1 << 25) + 1}, _native.E_CAPABILITY, "2^25"),
    ({"low": -0.1}, _native.E_VALUE, "clip_low"), ({"low": 1.1}, _native.E_VALUE, "clip_low"),
    ({"high": -0.1}, _native.E_VALUE, "clip_high"), ({"high": float("inf")}, _native.E_VALUE, "clip_high"),
    ({"high": float("nan")}, _native.E_VALUE, "clip_high"), ({"kl": float("nan")}, _native.E_VALUE, "kl_coef"),
    ({"reduction": 2}, _native.E_VALUE, "reduction"), ({"lp": None}, _native.E_VALUE, "NULL"), ({"old": None}, _native.E_VALUE, "NULL"),
    ({"adv": None}, _native.E_VALUE, "NULL"), ({"loss": None}, _native.E_VALUE, "NULL"), ({"stats": None}, _native.E_VALUE, "NULL"),
    ({"unit": None}, _native.E_VALUE, "NULL"), ({"weight": None}, _native.E_VALUE, "NULL"), ({"ws": None}, _native.E_VALUE, "workspace"),
    ({"ws": E + 4}, _native.E_VALUE, "workspace"), ({"ws_bytes": 8}, _native.E_VALUE, "workspace"),
    ({"strides": (15, 16, 16, 16, 16)}, _native.E_VALUE, "logprob"), ({"strides": (16, 16, 16, 16, 15)}, _native.E_VALUE, "mask"),
    ({"strides": (16, 16, 16, 15, 16)}, _native.E_VALUE, "advantage"), ({"strides": (16, 16, 16, -1, 16), "per_token": 0},
                                                                        _native.E_VALUE, "advantage")])
def test_policy_loss_refusals(native_library, change, expected, word):
    c = dict(lp=A, old=B, ref=C, adv=D, per_token=1, mask=None, strides=(16,) * 5, batch=600, seq=16, low=0.2, high=0.2, kl=0.1,
             reduction=0, unit=A + 0x1000, weight=A + 0x2000, loss=A + 0x3000, stats=A + 0x4000, ws=E, ws_bytes=1 << 20)
    c.update(change)
    rc = native_library.molt_policy_loss_fwd(c["lp"], c["old"], c["ref"], c["adv"], c["per_token"], c["mask"],
                                             _strides(*c["strides"]), c["batch"], c["seq"], c["low"], c["high"], c["kl"],
                                             c["reduction"], c["unit"], c["weight"], c["loss"], c["stats"], c["ws"],
                                             c["ws_bytes"], 0)
    _refused(rc, expected, word)


def test_policy_backward_refusals(native_library):
    lib = native_library
    _refused(lib.molt_policy_loss_bwd(None, B, C, D, 2, 2, 0), _native.E_VALUE, "NULL")
    _refused(lib.molt_policy_loss_bwd(A, B, C, D, -2, 2, 0), _native.E_VALUE, "negative")
    assert lib.molt_policy_loss_bwd(None, None, None, None, 0, 5, 0) == 0
    assert lib.molt_policy_loss_bwd(None, None, None, None, 5, 0, 0) == 0


@pytest.mark.parametrize("change,expected,word", [
    ({"pairs": 0}, _native.E_VALUE, "no pair"), ({"pairs": -2}, _native.E_VALUE, "no pair"), ({"seq": -1}, _native.E_VALUE, "negative"),
    ({"beta": 0.0}, _native.E_VALUE, "beta"), ({"beta": float("nan")}, _native.E_VALUE, "beta"),
    ({"beta": float("inf")}, _native.E_VALUE, "beta"), ({"smoothing": -0.1}, _native.E_VALUE, "smoothing"),
    ({"smoothing": 1.1}, _native.E_VALUE, "smoothing"), ({"smoothing": 0.1, "kind": 1}, _native.E_VALUE, "smoothing"),
    ({"kind": 3}, _native.E_VALUE, "kind"), ({"lp": None}, _native.E_VALUE, "NULL"), ({"rewards": None}, _native.E_VALUE, "NULL"),
    ({"loss": None}, _native.E_VALUE, "NULL"), ({"ws": None}, _native.E_VALUE, "workspace"), ({"ws": E + 4}, _native.E_VALUE, "workspace"),
    ({"ws_bytes": 8}, _native.E_VALUE, "workspace"), ({"strides": (7, 8, 8)}, _native.E_VALUE, "logprob"),
    ({"strides": (8, 7, 8)}, _native.E_VALUE, "ref_logprob"), ({"strides": (8, -1, 8), "per_token": 0}, _native.E_VALUE, "ref_logprob"),
    ({"strides": (8, 8, 7)}, _native.E_VALUE, "mask")])
def test_preference_loss_refusals(native_library, change, expected, word):
    c = dict(lp=A, ref=B, per_token=1, mask=C, strides=(8, 8, 8), pairs=200, seq=8, beta=0.1, smoothing=0.0, kind=0, average=0,
             grad=D, rewards=D + 0x1000, loss=D + 0x2000, ws=E, ws_bytes=1 << 20)
    c.update(change)
    rc = native_library.molt_preference_loss_fwd(c["lp"], c["ref"], c["per_token"], c["mask"], _strides(*c["strides"]), c["pairs"],
                                                 c["seq"], c["beta"], c["smoothing"], c["kind"], c["average"], c["grad"],
                                                 c["rewards"], c["loss"], c["ws"], c["ws_bytes"], 0)
    _refused(rc, expected, word)


def test_preference_backward_refusals(native_library):
    lib = native_library
    _refused(lib.molt_preference_loss_bwd(None, 0, None, B, C, 2, 2, 0), _native.E_VALUE, "NULL")
    _refused(lib.molt_preference_loss_bwd(A, 1, B, C, D, 2, 2, 0), _native.E_VALUE, "mask")
    _refused(lib.molt_preference_loss_bwd(A, 2, B, C, D, -2, 2, 0), _native.E_VALUE, "pair")
    assert lib.molt_preference_loss_bwd(None, 0, None, None, None, 0, 2, 0) == 0


def _items(*rows):
    return (ctypes.c_int64 * (4 * len(rows)))(*[v for row in rows for v in row])


F32, BF16 = _native.DTYPE_F32, _native.DTYPE_BF16


@pytest.mark.parametrize("rows,expected,word", [
    ([(A, B, 8, 3)], _native.E_CAPABILITY, "bf16 or fp32"), ([(A, B, -1, F32)], _native.E_VALUE, "count"),
    ([(0, B, 8, F32)], _native.E_VALUE, "NULL"), ([(A, 0, 8, F32)], _native.E_VALUE, "NULL"),
    ([(A + 2, B, 8, F32)], _native.E_VALUE, "aligned"), ([(A, B + 1, 8, BF16)], _native.E_VALUE, "aligned"),
    ([(A, B, 1 << 43, F32)], _native.E_VALUE, "count"),
    ([(A, A, 8, F32), (A, A, 8, F32)], _native.E_VALUE, "overlaps"),            # one tensor twice, in place
    ([(A, B, 8, F32), (C, B + 28, 8, F32)], _native.E_VALUE, "overlaps"),       # two outputs share an element
    ([(A, B, 8, F32), (B + 16, C, 8, F32)], _native.E_VALUE, "overlaps"),       # an output over another's gradient
    ([(A, A + 4, 8, F32)], _native.E_VALUE, "overlaps"),                        # an output shifted over its own gradient
    ([(A, B, 64, BF16), (C, B + 126, 8, BF16)], _native.E_VALUE, "overlaps"),
    ([(C, D, 4, F32), (A, B, 100, F32), (A + 40, B + 40, 1, F32)], _native.E_VALUE, "overlaps")])
def test_clip_refusals(native_library, rows, expected, word):
    rc = native_library.molt_clip_grads(_items(*rows), len(rows), 0, 1.0, E, D + 0x10_0000, 1 << 20, 0)
    _refused(rc, expected, word)


@pytest.mark.parametrize("change,expected,word", [
    ({"count": 0}, _native.E_VALUE, "no gradient"), ({"items": None}, _native.E_VALUE, "no gradient"), ({"kind": 2}, _native.E_VALUE, "norm"),
    ({"scale": float("nan")}, _native.E_VALUE, "max_norm"), ({"max_norm": -1.0}, _native.E_VALUE, "max_norm"),
    ({"max_norm": float("nan")}, _native.E_VALUE, "max_norm"), ({"result": None}, _native.E_VALUE, "workspace"),
    ({"ws": None}, _native.E_VALUE, "workspace"), ({"ws": B + 4}, _native.E_VALUE, "workspace"),
    ({"ws_bytes": 8}, _native.E_VALUE, "workspace")])
def test_grad_norm_refusals(native_library, change, expected, word):
    c = dict(items=_items((A, 0, 8, F32)), count=1, kind=0, scale=1.0, max_norm=1.0, result=C, ws=B, ws_bytes=1 << 20)
    c.update(change)
    rc = native_library.molt_grad_norm(c["items"], c["count"], c["kind"], c["scale"], c["max_norm"], c["result"], c["ws"],
                                       c["ws_bytes"], 0)
    _refused(rc, expected, word)


def test_clipped_adamw_needs_the_norm(native_library):
    rc = native_library.molt_adamw_step_clipped(A, B, C, D, 4, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, 0)
    _refused(rc, _native.E_VALUE, "clip is NULL")
    rc = native_library.molt_adamw_step_clipped(A, B, C, D, 3, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, E, 0)
    _refused(rc, _native.E_VALUE, "multiple of 4")


def test_host_tensors_are_refused(native_library):
    from molt_b200 import kernels

    lp = torch.zeros(2, 4)
    with pytest.raises(CapabilityError):
        kernels.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(CapabilityError):
        kernels.token_logprobs_with_grad(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(CapabilityError):
        kernels.clipped_policy_loss(lp, lp, lp)
    with pytest.raises(CapabilityError):
        kernels.preference_loss(lp)
    with pytest.raises(CapabilityError):
        kernels.global_grad_norm([lp])
    with pytest.raises(CapabilityError):
        kernels.clip_grad_norm(lp, 1.0)
    with pytest.raises(CapabilityError):
        kernels.global_grad_norm([lp], norm_type=1.0)
    with pytest.raises(ValueError):
        kernels.global_grad_norm([])
    with pytest.raises(ValueError):
        kernels.clip_grad_norm([lp], -1.0)
    with pytest.raises(ValueError):
        kernels.global_grad_norm([torch.zeros(4, 4)[:, :2]])


def test_step_driver_arguments_are_checked_on_the_host():
    from molt_b200.data_parallel import GradArena, ParamArena
    from molt_b200.qlora_step import CrossEntropy, PolicyObjective, PreferenceObjective, QLoRAStep, LLAMA3_8B, frozen_head_logprobs

    with pytest.raises(ValueError):
        QLoRAStep(LLAMA3_8B, torch.device("cpu"), max_grad_norm=-1.0)
    state = ParamArena(GradArena([torch.nn.Parameter(torch.zeros(4))]))
    with pytest.raises(ValueError):
        state.step(max_norm=float("nan"))
    assert state.steps == 0
    assert [o.grad_scale(4) for o in (CrossEntropy(), PolicyObjective(), PreferenceObjective())] == [1.0, 0.25, 0.25]
    hidden, head, ids = torch.zeros(3, 8), torch.zeros(16, 8), torch.zeros(3, dtype=torch.int64)
    for bad in ((hidden[0], head, ids), (hidden, head[:, :4], ids), (hidden, head, ids[:2])):
        with pytest.raises(ValueError):
            frozen_head_logprobs(*bad)
    with pytest.raises(CapabilityError):
        frozen_head_logprobs(hidden, head, ids)


class _HostStep:
    """A step driver without a device: model, optimizer and graph are stand-ins that record what they are given."""

    def __new__(cls):
        from molt_b200.qlora_step import CrossEntropy, QLoRAStep

        class Optimizer:
            def step(self, grad_scale, max_norm):
                return None

        step = object.__new__(QLoRAStep)
        step.guard = step.shadows = step.max_grad_norm = step._graph = None
        step.cuda_graph, step._eager_steps, step.steps, step.status_interval, step.world = False, 0, 0, 0, 1
        step.objective, step.optimizer = CrossEntropy(), Optimizer()
        step._forward_backward = lambda *inputs: inputs
        return step


def test_step_takes_tokens_and_targets_by_name():
    step = _HostStep()
    assert step.run(tokens=1, targets=2) == (1, 2)
    assert step.run(1, targets=2) == (1, 2)
    assert step.run(1, 2, 3, None) == (1, 2, 3, None)


def test_captured_step_keeps_no_graph_of_its_inputs():
    """Log-probabilities handed over with their graph: the held copies must not take part in it."""
    step = _HostStep()
    weight = torch.nn.Parameter(torch.ones(3))
    step._hold(torch.zeros(3, dtype=torch.int64), weight * 2, None)
    step._stage(torch.ones(3, dtype=torch.int64), weight * 3, None)
    tokens, old, mask = step._static_inputs
    assert tokens.tolist() == [1, 1, 1] and old.tolist() == [3, 3, 3] and mask is None
    assert old.grad_fn is None and not old.requires_grad


def _graph_nodes(tensor):
    seen, todo = set(), [tensor.grad_fn]
    while todo:
        node = todo.pop()
        if node is not None and node not in seen:
            seen.add(node)
            todo += [following for following, _ in node.next_functions]
    return seen


def test_recording_shares_no_node_with_an_eager_graph():
    """A graph that the caller keeps (log-probabilities not detached, say) shares its leaves' accumulation nodes, and the
    stream they were made on, with every later graph of the same leaves; a recording has leaves of its own."""
    from molt_b200.data_parallel import GradArena
    from molt_b200.qlora_step import leaves_of_its_own

    model = torch.nn.Sequential(torch.nn.Linear(3, 4), torch.nn.Linear(4, 2))
    model[1].weight.requires_grad_(False)
    model[1].bias = model[1].bias
    arena = GradArena(model.parameters())
    before = list(model.parameters())
    x = torch.randn(5, 3)
    kept = model(x).square().sum()
    with leaves_of_its_own(model):
        inside = list(model.parameters())
        assert all(a.data_ptr() == b.data_ptr() and a.requires_grad == b.requires_grad for a, b in zip(inside, before))
        assert all(vars(a) == vars(b) and (a is not b) == b.requires_grad for a, b in zip(inside, before))
        loss = model(x).square().sum()
        assert not _graph_nodes(loss) & _graph_nodes(kept)
        loss.backward()
    got = arena.flat.clone()
    assert all(a is b for a, b in zip(model.parameters(), before))
    arena.zero()
    kept.backward()
    assert bool(got.any()) and torch.equal(got, arena.flat)
    with pytest.raises(KeyError):
        with leaves_of_its_own(model):
            raise KeyError
    assert all(a is b for a, b in zip(model.parameters(), before))


def test_frozen_head_logprobs_needs_one_cuda_device():
    """Sizes that the GEMM kernel takes: a host pointer must not reach it."""
    from molt_b200.qlora_step import frozen_head_logprobs

    hidden, head, ids = torch.zeros(4, 64).bfloat16(), torch.zeros(128, 64).bfloat16(), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(CapabilityError):
        frozen_head_logprobs(hidden, head, ids)
    for bad in ((hidden, head.to("meta"), ids), (hidden.to("meta"), head, ids.to("meta")), (hidden, head, ids.to("meta"))):
        with pytest.raises(ValueError):
            frozen_head_logprobs(*bad)
