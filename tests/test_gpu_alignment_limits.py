"""Preference and policy tuning at the limits of the numbers: NaN in kept tokens, probabilities of zero, norms beyond fp32."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# one block, a block per part of a row, a warp per row
POLICY_SIZES = [(3, 5), (300, 100), (2048, 33)]


@pytest.mark.parametrize("batch,seq", POLICY_SIZES)
@pytest.mark.parametrize("where", ["logprobs", "old_logprobs"])
@pytest.mark.parametrize("masked", [False, True])
def test_policy_loss_keeps_a_nan_beside_an_advantage_of_zero(native_library, batch, seq, where, masked):
    """NaN times zero is NaN in loss and gradient; an infinite ratio times zero is zero, and so is what the mask leaves out."""
    from molt_b200.kernels import clipped_policy_loss

    given = {"logprobs": torch.full((batch, seq), -1.0, device="cuda"), "old_logprobs": torch.full((batch, seq), -1.5, device="cuda")}
    mask = torch.ones(batch, seq, dtype=torch.bool, device="cuda")
    mask[0, 0] = not masked
    given[where][0, 0] = float("nan")
    given["logprobs"][1, 1] = 400.0                       # a ratio of infinity
    leaf = given["logprobs"].requires_grad_()
    for reduction in ("token", "sequence"):
        got = clipped_policy_loss(leaf, given["old_logprobs"], torch.zeros(batch, device="cuda"), mask, reduction=reduction)
        (grad,) = torch.autograd.grad(got.loss, leaf)
        assert math.isnan(float(got.loss.detach())) != masked and math.isnan(float(grad[0, 0])) != masked
        grad[0, 0] = 0.0
        assert not bool(grad.any())
        if masked:
            assert float(got.loss.detach()) == 0.0
        assert float(got.clip_fraction) == 0.0


@pytest.mark.parametrize("pairs,seq", [(2, 3), (400, 40), (1100, 7)])     # one block, a block per row, a warp per row
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
def test_preference_loss_of_sequences_without_probability(native_library, pairs, seq, smoothing):
    """A kept token of probability zero in the rejected sequence: -ln sig(inf) = 0, and with smoothing infinite; in the chosen
    one the other way round.  The slope has its limits 0, beta e and -beta (1 - e).  Other pairs keep their share."""
    from molt_b200.kernels import preference_loss

    beta = 0.5
    one = -(1 - smoothing) * math.log(0.5) - smoothing * math.log(0.5)          # a pair with h = 0
    for side in ("rejected", "chosen"):
        lp = torch.full((2 * pairs, seq), -1.0, device="cuda")
        lp[pairs if side == "rejected" else 0, seq - 1] = -math.inf
        leaf = lp.requires_grad_()
        got = preference_loss(leaf, beta=beta, label_smoothing=smoothing)
        (grad,) = torch.autograd.grad(got.loss, leaf)
        against = smoothing if side == "rejected" else 1.0 - smoothing          # the factor of the infinite term
        want = math.inf if against else one * (pairs - 1) / pairs
        # the loss is summed in 64 bits and rounded once, the logarithm above is off by 2^-53
        assert float(got.loss.detach()) == pytest.approx(want, rel=2.0 ** -23, abs=0.0)
        slope = (beta * smoothing if side == "rejected" else -beta * (1.0 - smoothing)) / pairs
        for row, sign in ((0, 1.0), (pairs, -1.0)):
            assert torch.equal(grad[row], grad[row, :1].expand(seq))
            assert float(grad[row, 0]) == pytest.approx(sign * slope, rel=2.0 ** -23, abs=0.0)
        at = got.rejected_rewards if side == "rejected" else got.chosen_rewards
        assert float(at[0]) == -math.inf and bool(at[1:].isfinite().all())


@pytest.mark.parametrize("values", [[3e38, 3e38], [3.3e38] * 5000, [-3e38, 1.0, 2e38, 0.0, 1e-30]], ids=["two", "many", "mixed"])
def test_clipping_by_a_norm_beyond_fp32(native_library, values):
    """Finite gradients whose norm no fp32 value can hold.  The norm is reported as fp32's largest value; the coefficient
    comes from the norm in 64 bits: off by half a step of its own, 2^-150 where it is subnormal, 2^-24 of it where not.  The
    norm itself is off by 2^-20 at most (squares in 64 bits throughout here, so far less), the product by one rounding."""
    from molt_b200.kernels import clip_grad_norm, global_grad_norm

    top = torch.finfo(torch.float32).max
    grad = torch.tensor(values, device="cuda")
    exact = grad.double()
    norm = exact.norm()
    assert float(norm) > top
    assert float(global_grad_norm([grad])) == top
    for max_norm in (1.0, 1e30, 3e38):
        out = torch.empty_like(grad)
        assert float(clip_grad_norm([grad], max_norm, out=[out])) == top
        limit = float(torch.tensor(max_norm).float())
        coefficient = limit / float(norm)
        step = max(2.0 ** -150, coefficient * 2.0 ** -24)
        bound = exact.abs() * (step + coefficient * 2.0 ** -20) + 2.0 ** -150
        assert bool(((out.double() - exact * coefficient).abs() <= bound).all())
    out = torch.empty_like(grad)
    clip_grad_norm([grad], math.inf, out=[out])
    assert torch.equal(out, grad)
    for bad in (math.inf, math.nan):                       # these are still told apart
        assert not math.isfinite(float(global_grad_norm([grad, torch.tensor([bad], device="cuda")])))


def test_clipped_optimizer_step_with_a_norm_beyond_fp32(native_library):
    """Two gradients of 3e38 clipped to 1e15 (1e15 / sqrt(2) each, whose squares fp32 holds).  The first AdamW step from
    moments of zero moves a parameter by lr g / (|g| + eps): 16 roundings of 2^-24 at most, eps is below 2^-70 of |g|."""
    from molt_b200.data_parallel import GradArena, ParamArena

    p = torch.nn.Parameter(torch.zeros(2, device="cuda"))
    grads = GradArena([p])
    opt = ParamArena(grads, lr=0.5)
    grads.views[0].fill_(3e38)
    norm = opt.step(max_norm=1e15)
    assert math.isfinite(float(norm))
    assert bool(((p.detach() + 0.5).abs() <= 0.5 * 16 * 2.0 ** -24).all())


@pytest.mark.parametrize("bad_at", [(0,), (2,), (0, 1, 3), (5,)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_step_left_out_does_not_count(native_library, bad_at, bad):
    """A run with steps whose norm is not finite, against one that never saw them: the same moments, and parameters that
    differ only where a bias correction formed on the device is rounded to fp32 another way than the host's (2^-23 of it, and
    so at most 2^-22 of a step's change for both).  A change is below 4 lr: m / sqrt(v) of six random gradients is below 1.1
    by Cauchy and Schwarz, and the weight decay adds 0.1 |p|.  A parameter is rounded twice a step, from values that may then
    differ: 2^-23 of it each time."""
    from molt_b200.data_parallel import GradArena, ParamArena

    def arena():
        gen = torch.Generator(device="cuda").manual_seed(3)
        params = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen)) for n in (1000, 5)]
        return GradArena(params), params

    lr, gen = 1e-2, torch.Generator(device="cuda").manual_seed(4)
    batches = [torch.randn(1005, device="cuda", generator=gen) for _ in range(6)]
    runs = []
    for seen in (range(6), [i for i in range(6) if i not in bad_at]):
        grads, params = arena()
        opt = ParamArena(grads, lr=lr, weight_decay=0.1)
        for i in seen:
            grads.views[0].copy_(batches[i][:1000])
            grads.views[1].copy_(batches[i][1000:])
            if i in bad_at and len(seen) == 6:
                grads.views[1][2] = bad
            # the last step of all is made without a limit
            opt.step(max_norm=None if i == 5 and i not in bad_at else 0.5)
        runs.append((opt, torch.cat([p.detach() for p in params]), opt.exp_avg.clone(), opt.exp_avg_sq.clone()))
    (_, p, m, v), (_, q, n, w) = runs
    assert torch.equal(m, n) and torch.equal(v, w)
    assert float((p - q).abs().max()) <= 6 * (4 * lr * 2.0 ** -22 + 2 * 2.0 ** -23 * float(q.abs().max()))


def test_steps_left_out_are_counted_on_the_device(native_library):
    from molt_b200.data_parallel import GradArena, ParamArena

    grads = GradArena([torch.nn.Parameter(torch.ones(8, device="cuda"))])
    opt = ParamArena(grads)
    for value in (1.0, math.nan, math.inf, 1.0):
        grads.views[0].fill_(value)
        opt.step(max_norm=1.0)
    assert opt.steps == 4 and opt.skipped.dtype == torch.int64 and opt.skipped.tolist() == [2]


def test_captured_step_runs_the_hooks_of_its_parameters(native_library):
    """A weight that is trained beside the adapters, its gradient scaled by a hook: the captured steps give the eager ones'."""
    from molt_b200.qlora_step import CrossEntropy, DecoderShape, QLoRAStep

    shape = DecoderShape(layers=1, hidden=128, heads=4, kv_heads=2, head_dim=32, intermediate=256, vocab=512, rope_theta=1e4,
                         rank=8, alpha=16.0, nested_absmax=True, seq_len=32, micro_batch=2)

    class WithBias(CrossEntropy):
        def loss(self, model, world, layer_done, tokens, targets):
            return super().loss(model, world, layer_done, tokens, targets) + (model.bias * tokens.float().mean(0)).sum()

    runs = []
    for graph in (False, True):
        step = QLoRAStep(shape, torch.device("cuda"), lr=1e-3, objective=WithBias(), cuda_graph=graph)
        bias = step.model.bias = torch.nn.Parameter(torch.zeros(32, device="cuda"))
        bias.grad = torch.zeros_like(bias)
        bias.register_hook(lambda g: g * 3)
        gen = torch.Generator(device="cuda").manual_seed(6)
        grads = []
        for _ in range(5):
            tokens = torch.randint(0, 512, (2, 32), device="cuda", generator=gen)
            bias.grad.zero_()
            step.run(tokens, tokens.roll(-1, 1))
            grads.append(bias.grad.clone())
            assert torch.equal(grads[-1], 3 * tokens.float().mean(0))
        assert (step.replayed_launches > 0) == graph
        runs.append(torch.stack(grads))
    assert torch.equal(*runs)


def test_step_records_again_after_inputs_that_were_refused(native_library):
    """The third step, which is the recorded one, is given an odd number of sequences; the fourth is right again."""
    from molt_b200.qlora_step import DecoderShape, PreferenceObjective, QLoRAStep

    shape = DecoderShape(layers=1, hidden=128, heads=4, kv_heads=2, head_dim=32, intermediate=256, vocab=512, rope_theta=1e4,
                         rank=8, alpha=16.0, nested_absmax=True, seq_len=32, micro_batch=2)
    runs = []
    for graph in (False, True):
        step = QLoRAStep(shape, torch.device("cuda"), lr=1e-3, objective=PreferenceObjective(), cuda_graph=graph)
        gen = torch.Generator(device="cuda").manual_seed(7)
        losses = []
        for i in range(5):
            tokens = torch.randint(0, 512, (2, 32), device="cuda", generator=gen)
            if i == 2:
                with pytest.raises(ValueError, match="chosen sequences"):
                    step.run(tokens[:1], tokens[:1])
            losses.append(step.run(tokens, tokens.roll(-1, 1)).clone())
        assert (step.replayed_launches > 0) == graph
        runs.append((torch.stack(losses), step.optimizer.flat.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_dual_tensors_are_refused(native_library):
    """Nothing here has a forward-mode derivative: a tangent must not be dropped without a word, with or without grad mode,
    and for the losses' other arguments neither."""
    import torch.autograd.forward_ad as fwd

    from molt_b200 import kernels
    from molt_b200.qlora_step import frozen_head_logprobs

    logits, ids = torch.randn(4, 64, device="cuda"), torch.randint(0, 64, (4,), device="cuda")
    lp, adv = torch.randn(4, 6, device="cuda"), torch.randn(4, device="cuda")
    hidden, head = torch.randn(4, 64, device="cuda").bfloat16(), torch.randn(64, 64, device="cuda").bfloat16()
    calls = [(logits, lambda d: kernels.token_logprobs(d, ids)), (logits, lambda d: kernels.token_logprobs_with_grad(d, ids)),
             (adv, lambda d: kernels.token_logprobs_with_grad(logits, ids, d)),
             (lp, lambda d: kernels.clipped_policy_loss(d, lp, adv)), (lp, lambda d: kernels.clipped_policy_loss(lp, d, adv)),
             (adv, lambda d: kernels.clipped_policy_loss(lp, lp, d)),
             (lp, lambda d: kernels.clipped_policy_loss(lp, lp, adv, ref_logprobs=d)),
             (lp, lambda d: kernels.preference_loss(d)), (lp, lambda d: kernels.preference_loss(lp, d)),
             (lp, lambda d: kernels.global_grad_norm([adv, d])), (lp, lambda d: kernels.clip_grad_norm([d, adv], 1.0)),
             (hidden, lambda d: frozen_head_logprobs(d, head, ids)), (head, lambda d: frozen_head_logprobs(hidden, d, ids))]
    for primal, call in calls:
        for tracked in (False, True):
            for mode in (torch.enable_grad, torch.no_grad):
                with fwd.dual_level(), mode():
                    dual = fwd.make_dual(primal.clone().requires_grad_(tracked and primal is not head), torch.ones_like(primal))
                    with pytest.raises(NotImplementedError):
                        call(dual)
                    call(primal.clone())                  # a tensor without a tangent is welcome inside the level
