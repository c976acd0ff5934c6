"""Preference and policy tuning through the framework's own paths: the frozen head, the step driver, the optimizer."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_BF16 = 2.0 ** -8


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _close(got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound).max()):.3g} bounds"


@pytest.mark.parametrize("rows,width,vocab,chunk", [(300, 256, 1024, 128), (5, 64, 512, 8192), (70, 128, 1000, 33), (1, 64, 64, 1)])
def test_frozen_head_logprobs(native_library, rows, width, vocab, chunk):
    """Against 64 bits on the bf16 logits that the head GEMM gives.  A gradient row is (one-hot - p) / T rounded to bf16,
    times the head (fp32 accumulation: another 2^-12 of the terms covers it), rounded to bf16, scaled and rounded again."""
    from molt_b200.qlora_step import dense_gemm, frozen_head_logprobs

    gen = _gen(rows + vocab)
    hidden = torch.randn(rows, width, device="cuda", generator=gen).bfloat16().requires_grad_()
    head = (torch.randn(vocab, width, device="cuda", generator=gen) * 0.2).bfloat16()
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    if rows > 3:
        ids[1], ids[3] = -100, vocab
    weight = torch.randn(rows, device="cuda", generator=gen)
    temperature = 0.8
    parts = [hidden.detach()[i:i + chunk] for i in range(0, rows, chunk)]
    logits = torch.cat([dense_gemm(head, p, False) if vocab % 64 == 0 else p @ head.t() for p in parts]).double()
    kept = (ids >= 0) & (ids < vocab)
    at = ids.clamp(0, vocab - 1)[:, None]
    lsm = torch.log_softmax(logits / temperature, -1)
    want = torch.where(kept, lsm.gather(1, at)[:, 0], 0.0)
    lp = frozen_head_logprobs(hidden, head, ids, chunk, temperature)
    _close(lp.detach(), want, 2.0 ** -24 * (200 + 8 * want.abs()))
    (grad,) = torch.autograd.grad(lp, hidden, weight)
    row = (torch.zeros_like(lsm).scatter_(1, at, 1.0) - lsm.exp()) / temperature * kept[:, None]
    exact = row @ head.double()
    size = row.abs() @ head.double().abs()
    w = weight.double().abs()[:, None]
    _close(grad, exact * weight.double()[:, None], w * (size * (HALF_BF16 + 2 ** -12) + exact.abs() * 2.1 * HALF_BF16) * 1.01 + 1e-30)
    with torch.no_grad():   # scoring alone sums in another order: held to the same bound, not to the same bits
        scored = frozen_head_logprobs(hidden, head, ids, chunk, temperature)
    assert not scored.requires_grad
    _close(scored, want, 2.0 ** -24 * (200 + 8 * want.abs()))
    with pytest.raises(ValueError):
        frozen_head_logprobs(hidden, head.detach().requires_grad_(), ids)
    with pytest.raises(ValueError):
        frozen_head_logprobs(hidden, head, ids[:-1] if rows > 1 else ids.repeat(2))
    with pytest.raises(ValueError):
        frozen_head_logprobs(hidden, head, ids, chunk=0)


def _arena(sizes, seed):
    from molt_b200.data_parallel import GradArena, ParamArena

    gen = _gen(seed)
    params = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen)) for n in sizes]
    grads = GradArena(params)
    return params, grads, ParamArena(grads, lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


@pytest.mark.parametrize("max_norm", [0.05, 1e6, 0.0])
def test_clipped_optimizer_step_equals_clipping_first(native_library, max_norm):
    """The norm, and the step against one on gradients that were clipped beforehand.  The two gradients differ by 4 roundings
    at most (coefficient, its product with the scale, the products with the gradient: 2^-22 relatively), so do the
    moments, and the quotient m / sqrt(v) by twice that and its own 4 roundings: below 2^-19 of lr |m| / sqrt(v), where the
    bias-corrected quotient of three steps is below 4; three steps add up to 2^-15 * lr / 4 < lr 2^-16, and each rounds the
    parameter itself twice."""
    from molt_b200.kernels import clip_grad_norm

    params, grads, fused = _arena([1000, 77, 4096], 1)
    others, other_grads, plain = _arena([1000, 77, 4096], 1)
    for step in range(3):
        for g in (grads, other_grads):
            gen = _gen(10 + step)
            for view in g.views:
                view.normal_(0.0, 0.3, generator=gen)
        want = 0.5 * torch.cat([v.double() for v in grads.views]).norm()
        kept = grads.flat.clone()
        norm = fused.step(grad_scale=0.5, max_norm=max_norm)
        assert torch.equal(grads.flat, kept)                      # the gradients themselves stay
        _close(norm, want, want * 2 ** -20)
        other_grads.flat.mul_(0.5)
        clip_grad_norm(other_grads.flat, max_norm)
        plain.step()
        for a, b in zip(params, others):
            a, b = a.detach(), b.detach()
            assert float((a - b).abs().max()) <= 1e-2 * 2 ** -16 + float(b.abs().max()) * 2 ** -22
    assert params[0].grad is grads.views[0]
    with pytest.raises(ValueError):
        fused.step(max_norm=-1.0)
    assert fused.step() is None


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_optimizer_leaves_out_a_step_without_a_finite_norm(native_library, bad):
    params, grads, opt = _arena([100, 3], 2)
    grads.flat.fill_(0.25)
    opt.step(max_norm=1.0)
    before = [t.clone() for t in (opt.flat, opt.exp_avg, opt.exp_avg_sq)]
    grads.views[1][2] = bad
    norm = opt.step(max_norm=1.0)
    assert not math.isfinite(float(norm))
    assert all(torch.equal(a, b) for a, b in zip(before, (opt.flat, opt.exp_avg, opt.exp_avg_sq)))


def _shape(seq=32, batch=4):
    from molt_b200.qlora_step import DecoderShape

    return DecoderShape(layers=2, hidden=128, heads=4, kv_heads=2, head_dim=32, intermediate=256, vocab=512, rope_theta=1e4,
                        rank=8, alpha=16.0, nested_absmax=True, seq_len=seq, micro_batch=batch)


def _batch(shape, which, seed):
    gen = _gen(seed)
    size = (shape.micro_batch, shape.seq_len)
    tokens = torch.randint(0, shape.vocab, size, device="cuda", generator=gen)
    targets = torch.roll(tokens, -1, dims=1)
    mask = torch.rand(*size, device="cuda", generator=gen) < 0.7
    targets = torch.where(mask, targets, -100)
    near = -math.log(shape.vocab) + 0.3 * torch.randn(*size, device="cuda", generator=gen)
    if which == "policy":
        return tokens, targets, near, torch.randn(shape.micro_batch, device="cuda", generator=gen), mask, near - 0.1
    return tokens, targets, mask, near


def _objective(which):
    from molt_b200.qlora_step import PolicyObjective, PreferenceObjective

    return PolicyObjective(kl_coef=0.1, reduction="sequence") if which == "policy" else PreferenceObjective(beta=0.2)


def _torch_loss(which, lp, batch):
    if which == "policy":
        _, _, old, adv, mask, ref = batch
        r = torch.exp(lp - old)
        each = -torch.minimum(r * adv[:, None], r.clamp(0.8, 1.2) * adv[:, None]) + 0.1 * (torch.exp(ref - lp) - (ref - lp) - 1)
        return ((each * mask).sum(1) / mask.sum(1)).mean()
    _, _, mask, ref = batch
    s = ((lp - ref) * mask).sum(1)
    half = len(s) // 2
    return -torch.nn.functional.logsigmoid(0.2 * (s[:half] - s[half:])).mean()


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_step_gradients_match_plain_torch_behind_the_hidden_states(native_library, which):
    """The adapters' gradients of one step against head, log-softmax and loss in plain torch on the same hidden states.
    The two differ by bf16 roundings of logits, their gradients and the hidden gradient; 3e-2 relative Frobenius is what the
    decoder's gradients are held to elsewhere."""
    from molt_b200 import _native
    from molt_b200.qlora_step import QLoRAStep

    shape = _shape()
    step = QLoRAStep(shape, torch.device("cuda"), lr=0.0, objective=_objective(which), max_grad_norm=1.0)
    batch = _batch(shape, which, 5)
    loss = step.run(*batch)
    got = step.arena.flat.clone()
    assert float(step.grad_norm) == pytest.approx(float(got.double().norm()), rel=1e-5)
    step.arena.zero()
    hidden = step.model.hidden_states(batch[0])
    logits = (hidden.float() @ step.model.head.float().t()).view(*batch[0].shape, -1)
    lp = torch.log_softmax(logits, -1).gather(-1, batch[1].clamp(min=0)[..., None])[..., 0]
    want = _torch_loss(which, torch.where(batch[1] >= 0, lp, 0.0), batch)
    want.backward()
    assert abs(float(loss) - float(want)) < 2e-2 * max(1.0, abs(float(want)))
    plain = step.arena.flat
    assert float(plain.norm()) > 0
    assert float((got - plain).norm() / plain.norm()) < 3e-2
    with torch.no_grad():
        scored = step.model.logprobs(batch[0], batch[1])
    assert scored.shape == batch[0].shape and not bool(scored[batch[1] < 0].any())
    assert _native.read_status() == 0


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_captured_step_equals_the_eager_one(native_library, which):
    from molt_b200.qlora_step import QLoRAStep

    shape = _shape()
    runs = []
    for graph in (False, True):
        step = QLoRAStep(shape, torch.device("cuda"), lr=5e-3, objective=_objective(which), max_grad_norm=0.5, cuda_graph=graph)
        losses, norms = [], []
        for i in range(5):
            losses.append(step.run(*_batch(shape, which, i)).clone())
            norms.append(step.grad_norm.clone())
        runs.append((torch.stack(losses), torch.stack(norms), step.optimizer.flat.clone()))
        if graph:
            assert step.replayed_launches > 0
            with pytest.raises(ValueError):
                step.run(*_batch(shape, which, 0)[:2])
            with pytest.raises(ValueError):
                step.run(*_batch(_shape(16), which, 0))
    for a, b in zip(*runs):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


def test_default_step_still_takes_tokens_and_targets(native_library):
    from molt_b200.qlora_step import CrossEntropy, QLoRAStep

    shape = _shape()
    first = QLoRAStep(shape, torch.device("cuda"), lr=5e-3)
    second = QLoRAStep(shape, torch.device("cuda"), lr=5e-3, objective=CrossEntropy(), max_grad_norm=1e9)
    gen = _gen(0)
    tokens = torch.randint(0, shape.vocab, (4, 32), device="cuda", generator=gen)
    for _ in range(3):
        a, b = first.run(tokens, tokens.roll(-1, 1)), second.run(tokens, tokens.roll(-1, 1))
        assert torch.equal(a, b)
    assert torch.equal(first.optimizer.flat, second.optimizer.flat)   # a norm below the limit changes no bit
    assert first.grad_norm is None and float(second.grad_norm) > 0


def test_policy_step_in_the_static_microbatch_runner(native_library):
    """The loss captured by the micro-batch runner: replayed loss and gradients equal the eager ones."""
    from molt_b200.kernels import clipped_policy_loss, token_logprobs
    from molt_b200.training import StaticCudaMicrobatch

    gen = _gen(8)
    weight = torch.nn.Parameter(torch.randn(700, 32, device="cuda", generator=gen))
    x = torch.randn(6, 20, 32, device="cuda", generator=gen)
    ids = torch.randint(0, 700, (6, 20), device="cuda", generator=gen)
    old = -6 + torch.randn(6, 20, device="cuda", generator=gen)
    adv = torch.randn(6, 20, device="cuda", generator=gen)

    def build(x, ids, old, adv):
        return clipped_policy_loss(token_logprobs(x @ weight.t(), ids), old, adv).loss

    runner = StaticCudaMicrobatch(build, (x, ids, old, adv), [weight])
    loss = runner.replay(x, ids, old, adv).clone()
    grad = weight.grad.clone()
    runner.close()
    weight.grad = None
    eager = build(x, ids, old, adv)
    eager.backward()
    assert torch.equal(loss, eager.detach()) and torch.equal(grad, weight.grad)


def test_step_captured_while_the_caller_keeps_graphs_of_the_model(native_library):
    """Old log-probabilities taken from the model itself and handed over with their graph, before and after the capture."""
    from molt_b200.qlora_step import QLoRAStep

    shape = _shape()
    runs = []
    for graph in (False, True):
        step = QLoRAStep(shape, torch.device("cuda"), lr=5e-3, objective=_objective("policy"), max_grad_norm=0.5, cuda_graph=graph)
        losses, kept = [], []
        for i in range(5):
            tokens, targets, _, advantages, mask, ref = _batch(shape, "policy", i)
            kept.append(step.model.logprobs(tokens, targets))
            assert kept[-1].requires_grad
            losses.append(step.run(tokens, targets, kept[-1], advantages, mask, ref).clone())
        assert (step.replayed_launches > 0) == graph
        assert all(t is None or t.grad_fn is None for t in step._static_inputs)
        runs.append((torch.stack(losses), step.optimizer.flat.clone()))
    for a, b in zip(*runs):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


@pytest.mark.parametrize("form", ["transposed", "columns", "offset head", "offset hidden"])
def test_frozen_head_logprobs_of_a_head_that_is_no_dense_matrix(native_library, form):
    """Strides and offsets that the head's GEMM kernel does not take; bounds as for the dense head, on the plain product's logits."""
    from molt_b200.qlora_step import frozen_head_logprobs

    gen = _gen(31)
    rows, width, vocab = 9, 64, 128
    hidden = torch.randn(rows * width + 1, device="cuda", generator=gen).bfloat16()
    hidden = hidden[form == "offset hidden":][:rows * width].view(rows, width).requires_grad_()
    dense = (torch.randn(vocab, width, device="cuda", generator=gen) * 0.2).bfloat16()
    if form == "transposed":
        head = dense.t().contiguous().t()
    elif form == "columns":
        head = torch.cat([dense, dense], 1)[:, width:]
    elif form == "offset head":
        head = torch.cat([dense.new_zeros(1), dense.flatten()])[1:].view(vocab, width)
    else:
        head = dense
    assert torch.equal(head, dense)
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    logits = (hidden.detach() @ head.t()).double()
    lsm = torch.log_softmax(logits, -1)
    want = lsm.gather(1, ids[:, None])[:, 0]
    lp = frozen_head_logprobs(hidden, head, ids)
    _close(lp.detach(), want, 2.0 ** -24 * (200 + 8 * want.abs()))
    (grad,) = torch.autograd.grad(lp.sum(), hidden)
    row = torch.zeros_like(lsm).scatter_(1, ids[:, None], 1.0) - lsm.exp()
    exact = row @ dense.double()
    _close(grad, exact, (row.abs() @ dense.double().abs() * (HALF_BF16 + 2 ** -12) + exact.abs() * 2.1 * HALF_BF16) * 1.01 + 1e-30)
