"""Token log-probabilities, the policy and preference losses and gradient clipping against plain 64-bit forms.

Tolerances.  u = 2^-24 is half a step of fp32.  A rounding to bf16 adds ``finfo.eps / 2`` = 2^-8 of the value.

* log-probability: the exponents t = (x - M) / T are off by at most 4u |t| (difference, constant, product), so S by
  4u E[|t|] <= 4u ln V relatively, plus 2^-22 for each exp2 (4u), plus the sums: no thread adds more than V / 256 + 24 terms
  one after the other in a row that is split over at least 256 threads (u each).  ln S adds 4u |ln S|, the target's
  difference 3u |x_t - M| / T.
* gradient w (1[v=t] - p) / T: p's exponent off as above; |t| p <= 1, so absolutely |w| / T times the bound of the
  log-probability covers p and 1 - p; the product and one rounding to the result's type come on top.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _exact_logprobs(logits, ids, temperature):
    """Log-probabilities, the softmax and the bound of a log-probability's error, in 64 bits."""
    x = logits.double()
    x = (x - x.amax(-1, keepdim=True)) / temperature      # first: ln S is far below the last bit of the type's lowest value
    vocab = x.shape[-1]
    kept = (ids >= 0) & (ids < vocab)
    total = torch.logsumexp(x, -1)
    target = x.gather(-1, ids.clamp(0, vocab - 1)[..., None])[..., 0]
    lp = torch.where(kept, target - total, torch.zeros_like(total))
    bound = U * (vocab / 256 + 24 + 4 + 4 * math.log(vocab) + 4 * total.abs() + 3 * target.abs())
    return lp, torch.exp(x - total[..., None]), kept, torch.where(kept, bound, torch.zeros_like(bound))


def _exact_grad(probs, ids, kept, weight, temperature):
    onehot = torch.zeros_like(probs)
    vocab = probs.shape[-1]
    onehot.scatter_(-1, ids.clamp(0, vocab - 1)[..., None], 1.0)
    return torch.where(kept[..., None], (onehot - probs) * (weight.double() / temperature)[..., None], torch.zeros_like(probs))


def _close(got, want, bound):
    got, off = got.double(), (got.double() - want).abs()
    assert got.shape == want.shape
    bad = ~((off <= bound) | (got == want))
    assert not bool(bad.any()), f"{int(bad.sum())} values off, by up to {float((off / bound)[bad].max()):.3g} bounds"


def _check_grad(got, want, lp_bound, weight, temperature, dtype):
    bound = (weight.double().abs() / temperature * (lp_bound + 8 * U))[..., None] + want.abs() * (torch.finfo(dtype).eps / 2 + 4 * U)
    _close(got, want, bound + 1e-38)


LOGIT_CASES = [(1, 1), (1, 2), (3, 7), (5, 8), (2, 31), (4, 513), (4, 1000), (33, 4099), (300, 129), (7, 32001), (3, 50257),
               (2, 151936), (160, 20000)]


@pytest.mark.parametrize("rows,vocab", LOGIT_CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["plain", "wide", "shifted"])
def test_token_logprobs_forward_and_gradients(native_library, rows, vocab, dtype, layout):
    """All three forms: alone, with autograd, in one pass (beside the logits and over them)."""
    from molt_b200.kernels import token_logprobs, token_logprobs_with_grad

    gen = _gen(rows * 1000 + vocab)
    temperature = {"plain": 1.0, "wide": 0.6, "shifted": 1.7}[layout]
    pad, first = {"plain": (0, 0), "wide": (24, 8), "shifted": (5, 3)}[layout]   # columns around the logits
    store = (torch.randn(rows, vocab + pad, device="cuda", generator=gen) * 3).to(dtype)
    logits = store[:, first:first + vocab]
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    if rows > 2:
        ids[1], ids[2] = -100, vocab + 3
    weight = torch.randn(rows, device="cuda", generator=gen)
    want, probs, kept, bound = _exact_logprobs(logits, ids, temperature)
    want_grad = _exact_grad(probs, ids, kept, weight, temperature)

    _close(token_logprobs(logits, ids, temperature), want, bound)
    leaf = logits.detach().requires_grad_()
    lp = token_logprobs(leaf, ids, temperature)
    _close(lp.detach(), want, bound)
    (grad,) = torch.autograd.grad(lp, leaf, weight)
    assert grad.dtype == dtype
    _check_grad(grad, want_grad, bound, weight, temperature, dtype)

    lp, grad = token_logprobs_with_grad(logits, ids, weight, temperature)
    _close(lp, want, bound)
    _check_grad(grad, want_grad, bound, weight, temperature, dtype)
    lp, grad = token_logprobs_with_grad(logits, ids, temperature=temperature)
    _check_grad(grad, _exact_grad(probs, ids, kept, torch.ones_like(weight), temperature), bound, torch.ones_like(weight),
                temperature, dtype)
    other = torch.full((rows, vocab + 3), 7.0, dtype=dtype, device="cuda")      # rows that begin on another alignment
    token_logprobs_with_grad(logits, ids, weight, temperature, out=other[:, 1:vocab + 1])
    _check_grad(other[:, 1:vocab + 1], want_grad, bound, weight, temperature, dtype)
    assert bool((other[:, 0] == 7).all()) and bool((other[:, vocab + 1:] == 7).all())
    before = store.clone()
    lp, grad = token_logprobs_with_grad(logits, ids, weight, temperature, out=logits)
    assert grad.data_ptr() == logits.data_ptr()
    _close(lp, want, bound)
    _check_grad(logits, want_grad, bound, weight, temperature, dtype)
    assert torch.equal(store[:, :first], before[:, :first]) and torch.equal(store[:, first + vocab:], before[:, first + vocab:])


@pytest.mark.parametrize("vocab", [5, 1000, 40001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs_of_masked_and_broken_rows(native_library, vocab, dtype):
    from molt_b200.kernels import token_logprobs, token_logprobs_with_grad

    gen = _gen(vocab)
    lowest, inf = torch.finfo(dtype).min, float("inf")
    logits = torch.randn(10, vocab, device="cuda", generator=gen).to(dtype)
    ids = torch.full((10,), vocab - 1, device="cuda")
    logits[0, : vocab - 1] = -inf                        # only the target is left: log-probability 0, gradient 0
    logits[1, : vocab // 2] = lowest                     # masked by the type's lowest value
    logits[2, :] = lowest                                # nothing but it: uniform
    logits[3, vocab - 1] = -inf                          # the target itself is masked: -inf, gradient one-hot - p
    logits[4, 0] = float("nan")
    logits[5, 0] = inf
    logits[6, :] = -inf
    logits[7, :] = float("nan")
    ids[7] = -100                                        # an ignored row may hold anything
    logits[8, vocab - 1] = -lowest                       # the largest finite value beside ordinary ones
    logits[9, ::2] = -inf
    ids[9] = 1
    for temperature in (1.0, 0.05):
        want, probs, kept, bound = _exact_logprobs(logits, ids, temperature)
        # the lowest value over a small temperature is outside fp32, not outside the definition
        leaf = logits.detach().requires_grad_()
        lp = token_logprobs(leaf, ids, temperature)
        grad = torch.autograd.grad(lp, leaf, torch.ones(10, device="cuda"))[0]
        lp2, grad2 = token_logprobs_with_grad(logits, ids, temperature=temperature)
        for got, g in ((lp.detach(), grad), (lp2, grad2)):
            for row in (0, 1, 2, 3, 8, 9):
                _close(got[row], want[row], bound[row] if math.isfinite(float(bound[row])) else torch.zeros_like(bound[row]))
            assert bool(got[[4, 5, 6]].isnan().all()) and float(got[7]) == 0.0
            assert bool(g[[4, 5, 6]].isnan().all()) and not bool(g[7].any())
            one = torch.ones(10, device="cuda")
            want_grad = _exact_grad(probs, ids, kept, one, temperature)
            limit = torch.full_like(bound, U * (vocab / 256 + 60))
            for row in (0, 1, 2, 3, 8, 9):
                _check_grad(g[row:row + 1], want_grad[row:row + 1], limit[row:row + 1], one[row:row + 1], temperature, dtype)


def test_token_logprobs_shapes_strides_and_offsets(native_library):
    from molt_b200.kernels import token_logprobs, token_logprobs_with_grad

    gen = _gen(5)
    logits = torch.randn(3, 6, 77, device="cuda", generator=gen, requires_grad=True)
    ids = torch.randint(0, 77, (3, 6), device="cuda", generator=gen)
    # next-token scoring: all positions but the last, the ids but the first
    lp = token_logprobs(logits[:, :-1], ids[:, 1:])
    want = torch.log_softmax(logits.detach().double()[:, :-1], -1).gather(-1, ids[:, 1:, None])[..., 0]
    assert lp.shape == (3, 5)
    _close(lp.detach(), want, torch.full_like(want, 200 * U))
    (grad,) = torch.autograd.grad(lp.sum(), logits)      # the incoming gradient is an expanded scalar
    assert grad.shape == logits.shape and not bool(grad[:, -1].any())
    assert float(grad.double().sum(-1).abs().max()) < 1e-5
    one = logits.detach()[0, 0]
    scalar = token_logprobs(one, ids[0, 0])
    assert scalar.shape == ()
    _close(scalar, torch.log_softmax(one.double(), -1)[ids[0, 0]], torch.tensor(200 * U, device="cuda"))
    # one row for all ids, columns that are not neighbours, no rows
    shared = torch.randn(1, 300, device="cuda", generator=gen)
    many = torch.arange(40, device="cuda")
    want = torch.log_softmax(shared.double(), -1)[0, :40]
    _close(token_logprobs(shared.expand(40, 300), many), want, torch.full_like(want, 200 * U))
    turned = torch.randn(300, 4, device="cuda", generator=gen).t()
    want = torch.log_softmax(turned.double(), -1)[torch.arange(4), many[:4]]
    _close(token_logprobs(turned, many[:4]), want, torch.full_like(want, 200 * U))
    empty = torch.empty(0, 11, device="cuda", requires_grad=True)
    lp = token_logprobs(empty, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert lp.shape == (0,) and torch.autograd.grad(lp.sum(), empty)[0].shape == (0, 11)
    # rows more than 2^31 elements apart
    step = (1 << 30) + 8
    wide = torch.empty(4 * step + 1024, dtype=torch.bfloat16, device="cuda").as_strided((5, 1000), (step, 1))
    wide.copy_(torch.randn(5, 1000, device="cuda", generator=gen))
    near = wide.clone()
    a, g = token_logprobs_with_grad(wide, many[:5], out=wide)
    b, h = token_logprobs_with_grad(near, many[:5])
    assert torch.equal(a, b) and torch.equal(g, h)


GROUPED = {
    "all but the last": lambda x: x[:, :-1],
    "every second": lambda x: x[:, ::2],
    "batch last": lambda x: x.transpose(0, 1),
    "one batch for all": lambda x: x[:1].expand(5, -1, -1),
    "one row per batch": lambda x: x[:, :1].expand(-1, 4, -1),
    "inner columns": lambda x: x[1:, 1:-1, 3:-2],
    "four dimensions": lambda x: x[:, :-1].unflatten(1, (2, -1))[:, :, :2],     # three strides: a copy
    "a row each": lambda x: x[:, 2],
}


@pytest.mark.parametrize("form", GROUPED)
@pytest.mark.parametrize("vocab", [37, 5000, 40000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_token_logprobs_of_rows_in_groups(native_library, form, vocab, dtype):
    from molt_b200.kernels import token_logprobs, token_logprobs_with_grad

    gen = _gen(vocab + len(form))
    store = (torch.randn(3, 7, vocab, device="cuda", generator=gen) * 2).to(dtype)
    logits = GROUPED[form](store)
    shape, width = logits.shape[:-1], logits.shape[-1]
    ids = torch.randint(0, width, shape, device="cuda", generator=gen)
    ids.view(-1)[1] = -100
    weight = torch.randn(shape, device="cuda", generator=gen)
    flat, w = ids.reshape(-1), weight.reshape(-1)
    want, probs, kept, bound = _exact_logprobs(logits.reshape(-1, width), flat, 0.7)
    want_grad = _exact_grad(probs, flat, kept, w, 0.7)
    assert token_logprobs(logits, ids, 0.7).shape == shape
    _close(token_logprobs(logits, ids, 0.7).reshape(-1), want, bound)
    leaf = logits.detach().requires_grad_()
    lp = token_logprobs(leaf, ids, 0.7)
    _close(lp.detach().reshape(-1), want, bound)
    (grad,) = torch.autograd.grad(lp, leaf, weight)
    assert grad.shape == logits.shape
    _check_grad(grad.reshape(-1, width), want_grad, bound, w, 0.7, dtype)
    lp, grad = token_logprobs_with_grad(logits, ids, weight, 0.7)
    assert lp.shape == shape and grad.shape == logits.shape
    _close(lp.reshape(-1), want, bound)
    _check_grad(grad.reshape(-1, width), want_grad, bound, w, 0.7, dtype)


def test_token_logprobs_make_no_copy_of_a_slice(native_library):
    from molt_b200.kernels import token_logprobs

    logits = torch.zeros(4, 65, 40000, device="cuda", dtype=torch.bfloat16)
    ids = torch.zeros(4, 64, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    token_logprobs(logits[:, :-1], ids)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20


def _check_all_forms(logits, ids, temperature, out=None):
    from molt_b200.kernels import token_logprobs, token_logprobs_with_grad

    weight = torch.linspace(-2.0, 2.0, len(ids), device="cuda")
    want, probs, kept, bound = _exact_logprobs(logits, ids, temperature)
    want_grad = _exact_grad(probs, ids, kept, weight, temperature)
    leaf = logits.detach().requires_grad_()
    lp = token_logprobs(leaf, ids, temperature)
    _close(lp.detach(), want, bound)
    _check_grad(torch.autograd.grad(lp, leaf, weight)[0], want_grad, bound, weight, temperature, logits.dtype)
    lp, grad = token_logprobs_with_grad(logits, ids, weight, temperature, out=out)
    _close(lp, want, bound)
    _check_grad(grad, want_grad, bound, weight, temperature, logits.dtype)


# Vectors of 16 bytes around the borders of the batches (512 vectors per block) and of the ring (5 batches), and of the
# small blocks (512 vectors); the elements behind them; 3 rows are spread over many blocks, 700 are not.
BORDERS = [1, 63, 64, 511, 512, 513, 1023, 1024, 1025, 2559, 2560, 2561, 3073, 3136, 5119, 5120, 5121, 5632, 8192]


@pytest.mark.parametrize("vectors", BORDERS)
@pytest.mark.parametrize("rows,dtype", [(3, torch.bfloat16), (3, torch.float32), (700, torch.bfloat16)])
def test_token_logprobs_at_the_borders_of_their_blocks(native_library, vectors, rows, dtype):
    gen = _gen(vectors)
    per = 16 // dtype.itemsize
    for extra in (0, per - 1):
        vocab = vectors * per + extra
        logits = (torch.randn(rows, vocab, device="cuda", generator=gen) * 2).to(dtype)
        ids = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        ids[0], ids[1] = vocab - 1, 0
        _check_all_forms(logits, ids, 0.9)


@pytest.mark.parametrize("temperature", [1e-30, 1e-4, 1e4, 1e30])
@pytest.mark.parametrize("vocab", [900, 60_000])
def test_token_logprobs_at_extreme_temperatures(native_library, temperature, vocab):
    gen = _gen(vocab)
    for dtype in (torch.bfloat16, torch.float32):
        logits = (torch.randn(5, vocab, device="cuda", generator=gen) * 4).to(dtype)
        _check_all_forms(logits, torch.randint(0, vocab, (5,), device="cuda", generator=gen), temperature)


@pytest.mark.parametrize("rows,vocab,dtype", [(2, 700_001, torch.bfloat16), (2, 1_300_000, torch.float32), (70_000, 5, torch.float32),
                                              (66_000, 131, torch.bfloat16)])
def test_token_logprobs_of_long_rows_and_many_rows(native_library, rows, vocab, dtype):
    gen = _gen(rows)
    logits = torch.empty(rows, vocab, dtype=dtype, device="cuda").normal_(0.0, 3.0, generator=gen)
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    ids[-1] = -1
    _check_all_forms(logits, ids, 1.0)


def test_token_logprobs_with_every_id_ignored_and_in_inference_mode(native_library):
    from molt_b200.kernels import token_logprobs, token_logprobs_with_grad

    logits = torch.full((5, 9000), float("nan"), device="cuda", requires_grad=True)
    ids = torch.full((5,), -100, device="cuda")
    lp = token_logprobs(logits, ids)
    lp.sum().backward()
    assert not bool(lp.any()) and not bool(logits.grad.any())
    with torch.inference_mode():
        x = torch.zeros(5, 9000, device="cuda")
        lp, grad = token_logprobs_with_grad(x, ids + 101, out=x)
        _close(lp, torch.full((5,), -math.log(9000), device="cuda", dtype=torch.float64), torch.full((5,), 200 * U, device="cuda"))
        assert grad is x and float(grad[0, 1]) == pytest.approx(1 - 1 / 9000, rel=1e-6)
        _close(token_logprobs(torch.zeros(5, 9000, device="cuda"), ids + 101), lp.double(), torch.full((5,), 400 * U, device="cuda"))


@pytest.mark.parametrize("rows,vocab", [(3, 151936), (40, 40000)])
def test_token_logprobs_replayed_as_graphs(native_library, rows, vocab):
    """Rows spread over clusters of blocks, recorded once and replayed on other logits and ids, ignored ones among them."""
    from molt_b200.kernels import token_logprobs, token_logprobs_with_grad

    gen = _gen(rows)
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(rows, dtype=torch.int64, device="cuda")
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_logprobs(x, ids), token_logprobs_with_grad(x, ids, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scored = token_logprobs(x, ids)
        lp, _ = token_logprobs_with_grad(x, ids, out=out)
    for step in range(3):
        x.normal_(0.0, 2.0, generator=gen)
        ids.random_(0, vocab, generator=gen)
        ids[step] = -100
        graph.replay()
        want = token_logprobs_with_grad(x, ids)
        assert torch.equal(lp, want[0]) and torch.equal(out, want[1]) and torch.equal(scored, token_logprobs(x, ids))


def test_token_logprobs_refusals(native_library):
    from molt_b200.core.errors import CapabilityError
    from molt_b200.kernels import token_logprobs, token_logprobs_with_grad

    logits, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(CapabilityError):
        token_logprobs(logits.half(), ids)
    for bad in (ids[:3], ids.int(), ids.cpu(), ids[:, None]):
        with pytest.raises(ValueError):
            token_logprobs(logits, bad)
    for temperature in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            token_logprobs(logits, ids, temperature)
    for weight in (torch.ones(3, device="cuda"), torch.ones(4, device="cuda").bfloat16(), torch.ones(4)):
        with pytest.raises(ValueError):
            token_logprobs_with_grad(logits, ids, weight)
    shared = torch.zeros(100, device="cuda")
    for out in (logits.bfloat16(), logits[:3], torch.zeros(8, 4, device="cuda").t(), torch.zeros(4, 8, device="cuda", requires_grad=True),
                torch.zeros(1, 8, device="cuda").expand(4, 8)):
        with pytest.raises(ValueError):
            token_logprobs_with_grad(logits, ids, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        token_logprobs_with_grad(shared[:32].view(4, 8), ids, out=shared[4:36].view(4, 8))
    leaf = logits.clone().requires_grad_()
    lp = token_logprobs(leaf, ids)
    token_logprobs_with_grad(leaf.detach(), ids, out=leaf.detach())      # overwrites what the backward pass needs
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()


def test_token_logprob_gradient_against_differences(native_library):
    """f = sum w l: its slope along v from central differences of the kernel's own forward pass.  l is off by < 100u = 6e-6
    per row, the step is 2^-4 and |f'''| <= 2 |w| / T^3 for |v| <= 1, so the quotient is off by < 12 * 6e-6 / 2^-3 + 12 * 2 * 2^-8 / 6."""
    from molt_b200.kernels import token_logprobs

    gen = _gen(11)
    x = torch.randn(12, 211, device="cuda", generator=gen)
    ids = torch.randint(0, 211, (12,), device="cuda", generator=gen)
    w = torch.rand(12, device="cuda", generator=gen)
    v = torch.rand(12, 211, device="cuda", generator=gen) * 2 - 1
    leaf = x.clone().requires_grad_()
    (grad,) = torch.autograd.grad(token_logprobs(leaf, ids, 1.0), leaf, w)
    h = 2.0 ** -4
    slope = (w.double() * (token_logprobs(x + h * v, ids).double() - token_logprobs(x - h * v, ids).double())).sum() / (2 * h)
    assert abs(float(slope - (grad.double() * v).sum())) < 12 * 6e-6 / 2 ** -3 + 12 * 2 * 2 ** -8 / 6


# ---- policy loss ---------------------------------------------------------------------------------------------------
# A token's ratio is off by 2^-22 (exp) + |d| u, its products by u each; k and 1 - exp(e) by less than 8u relatively (the
# difference e is off by u |e|, which moves k by 2u and 1 - exp(e) by (1 + |e|) u, |e| < 5): 16u = 2^-20 of the terms'
# magnitudes covers both.  Sums are held in 64 bits; every output is rounded once (u) and weights are rounded (u).
POLICY_CASES = [(1, 1), (1, 7), (3, 16), (4, 64), (5, 257), (2, 4099), (64, 100), (257, 31), (700, 33), (1, 70001), (2000, 1),
                (2047, 40), (2048, 40), (3001, 1), (2049, 1024), (2050, 1025), (12000, 17), (3, 513), (20, 512), (1, 1_300_000)]


def _policy_inputs(batch, seq, gen, per_token, ragged):
    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    lp = -3 * torch.rand(batch, seq, device="cuda", generator=gen)
    old, ref = lp + 0.25 * normal(batch, seq), lp + 0.5 * normal(batch, seq)
    adv = normal(batch, seq) if per_token else normal(batch)
    if batch > 1:
        adv[0] = 0.0
    mask = None
    if ragged:
        mask = torch.rand(batch, seq, device="cuda", generator=gen) < 0.7
        if batch > 2:
            mask[1] = False
        for t in (lp, old, ref):
            t[~mask] = float("nan")
            t.view(-1)[~mask.view(-1) & (torch.arange(batch * seq, device="cuda") % 3 == 0)] = float("inf")
        if per_token:
            adv[~mask] = float("nan")
    return lp, old, ref, adv, mask


def _exact_policy(lp, old, ref, adv, mask, low, high, kl_coef, reduction):
    mask = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask.bool()
    leaf = lp.detach().double().requires_grad_()
    at = mask.nonzero(as_tuple=True)
    x = leaf[at]
    a = (adv if adv.dim() == 2 else adv[:, None].expand_as(lp))[at].double()
    n = mask.sum(1).double()
    w = torch.ones_like(a) / max(1, len(a)) if reduction == "token" else 1 / (n[at[0]] * (n > 0).sum())
    r = torch.exp(x - old[at].double())
    taken = torch.minimum(r * a, torch.clamp(r, 1 - low, 1 + high) * a)
    e = (ref[at].double() if ref is not None else x.detach()) - x
    if ref is None:
        e = e.detach()
    k = torch.expm1(e) - e
    loss = (w * (kl_coef * k - taken)).sum()
    (grad,) = torch.autograd.grad(loss, leaf)
    with torch.no_grad():
        cut = (taken < r * a).double()
        size = w * (a.abs() * r.clamp(min=1 - low) + abs(kl_coef) * (k + torch.expm1(e).abs()))
        bound = torch.zeros_like(leaf)
        bound[at] = size * 2 ** -20
        return loss.detach(), (w * k).sum(), (w * cut).sum(), grad, bound, size.sum() * 2 ** -20


@pytest.mark.parametrize("batch,seq", POLICY_CASES)
@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("form", ["per-token,ref,ragged", "per-sequence,ragged", "per-token", "per-sequence,ref"])
def test_policy_loss_and_gradient(native_library, batch, seq, reduction, form):
    from molt_b200.kernels import clipped_policy_loss

    lp, old, ref, adv, mask = _policy_inputs(batch, seq, _gen(batch * 7 + seq), "per-token" in form, "ragged" in form)
    if "ref" not in form:
        ref = None
    kl = 0.05 if ref is not None else 0.0
    leaf = lp.clone().requires_grad_()
    got = clipped_policy_loss(leaf, old, adv, mask, ref, clip_low=0.2, clip_high=0.3, kl_coef=kl, reduction=reduction)
    loss, k, cut, grad, bound, total = _exact_policy(lp, old, ref, adv, mask, 0.2, 0.3, kl, reduction)
    _close(got.loss.detach(), loss, total + loss.abs() * U)
    _close(got.kl, k, 2 ** -20 * k)
    _close(got.clip_fraction, cut, 2 * U * cut)
    scale = torch.tensor(-2.5, device="cuda")
    (dlp,) = torch.autograd.grad(got.loss, leaf, scale)
    _close(dlp, grad * -2.5, 2.5 * (bound + grad.abs() * 4 * U) + 1e-38)
    if mask is not None:
        assert not bool(dlp[~mask].any())
    assert not got.kl.requires_grad and not got.clip_fraction.requires_grad
    with torch.no_grad():
        again = clipped_policy_loss(lp, old, adv, mask, ref, clip_low=0.2, clip_high=0.3, kl_coef=kl, reduction=reduction)
    assert all(torch.equal(x, y) for x, y in zip(again, [got.loss.detach(), got.kl, got.clip_fraction]))


def test_policy_loss_on_the_borders(native_library):
    """Ratios at the clamp's borders and beside them, decided as in 64 bits; advantages of zero beside ratios that
    overflow; clamps of width zero and one."""
    from molt_b200.kernels import clipped_policy_loss

    for low, high in ((0.2, 0.28), (0.0, 0.0), (1.0, 3.0)):
        edges = [math.log1p(high), math.log1p(-low) if low < 1 else -20.0, 0.0]
        steps = torch.arange(-8, 9, dtype=torch.float64) * 2.0 ** -27
        d = torch.cat([e + steps for e in edges]).float()[None].cuda().repeat(2, 1)
        adv = torch.tensor([1.5, -0.5], device="cuda")
        old = torch.zeros_like(d)
        leaf = d.clone().requires_grad_()
        got = clipped_policy_loss(leaf, old, adv, clip_low=low, clip_high=high)
        (grad,) = torch.autograd.grad(got.loss, leaf)
        x = d.double()
        cut = torch.stack([x[0] > math.log1p(high), (x[1] < math.log1p(-low)) if low < 1 else torch.zeros_like(x[1], dtype=torch.bool)])
        want = torch.where(cut, torch.zeros_like(x), -adv.double()[:, None] * torch.exp(x)) / x.numel()
        assert torch.equal(grad == 0, cut)
        _close(grad, want, want.abs() * 2 ** -20)
        _close(got.clip_fraction, cut.double().mean(), 2 * U)
    lp = torch.tensor([[0.0, 200.0]], device="cuda", requires_grad=True)
    got = clipped_policy_loss(lp, torch.zeros(1, 2, device="cuda"), torch.tensor([[1.0, 0.0]], device="cuda"))
    got.loss.backward()
    assert float(got.loss) == -0.5 and lp.grad.tolist() == [[-0.5, 0.0]]
    # a clipped token far outside keeps its finite loss
    lp = torch.tensor([[200.0]], device="cuda", requires_grad=True)
    got = clipped_policy_loss(lp, torch.zeros(1, 1, device="cuda"), torch.ones(1, device="cuda"), clip_high=0.5)
    got.loss.backward()
    assert float(got.loss) == -1.5 and float(lp.grad) == 0.0 and float(got.clip_fraction) == 1.0


def test_policy_loss_kl_of_near_and_far_policies(native_library):
    from molt_b200.kernels import clipped_policy_loss

    e = torch.cat([2.0 ** -torch.arange(0, 30).float(), torch.tensor([0.5, 0.4999999, 0.51, 1.0, 5.0, 40.0, 61.0, 88.0])])
    e = torch.cat([e, -e]).cuda()[:, None]
    zero = torch.zeros_like(e)
    for i in range(len(e)):
        leaf = zero[i:i + 1].clone().requires_grad_()
        got = clipped_policy_loss(leaf, zero[i:i + 1], torch.zeros(1, device="cuda"), ref_logprobs=e[i:i + 1], kl_coef=1.0)
        x = e[i, 0].double()
        # the series in 64 bits where the plain difference would lose digits
        k = x * x / 2 * (1 + x / 3 * (1 + x / 4 * (1 + x / 5 * (1 + x / 6)))) if abs(x) < 2 ** -8 else torch.expm1(x) - x
        _close(got.kl, k, k * 2 ** -20)
        got.loss.backward()
        _close(leaf.grad[0, 0], -torch.expm1(x), torch.expm1(x).abs() * 2 ** -20)


def test_policy_loss_without_tokens(native_library):
    from molt_b200.kernels import clipped_policy_loss

    for reduction in ("token", "sequence"):
        for shape, mask in (((3, 5), torch.zeros(3, 5, dtype=torch.bool, device="cuda")), ((3, 0), None)):
            lp = torch.full(shape, float("nan"), device="cuda", requires_grad=True)
            got = clipped_policy_loss(lp, lp.detach(), torch.ones(3, device="cuda"), mask, lp.detach(), kl_coef=1.0, reduction=reduction)
            got.loss.backward()
            assert [float(v) for v in got] == [0.0, 0.0, 0.0] and lp.grad.shape == shape and not bool(lp.grad.any())


def test_policy_loss_strides_masks_and_refusals(native_library):
    from molt_b200.core.errors import CapabilityError
    from molt_b200.kernels import clipped_policy_loss

    gen = _gen(3)
    lp, old, ref, adv, _ = _policy_inputs(6, 50, gen, True, False)
    mask = torch.rand(6, 50, device="cuda", generator=gen) < 0.5

    def gapped(t):   # the same values inside a wider tensor
        wide = torch.full((6, 61), 3, dtype=t.dtype, device="cuda")
        wide[:, 7:57] = t
        return wide[:, 7:57]

    want = clipped_policy_loss(lp, old, adv, mask, ref, kl_coef=0.1)
    got = clipped_policy_loss(gapped(lp), gapped(old), gapped(adv), gapped(mask), gapped(ref), kl_coef=0.1)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = clipped_policy_loss(lp.t().contiguous().t(), old, adv, mask.to(torch.uint8) * 200, ref, kl_coef=0.1)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    rows = clipped_policy_loss(lp, old, adv[:1].expand(6, 50), mask[:1].expand(6, 50), kl_coef=0.1)
    same = clipped_policy_loss(lp, old, adv[:1].repeat(6, 1), mask[:1].repeat(6, 1), kl_coef=0.1)
    assert all(torch.equal(a, b) for a, b in zip(rows, same))
    per_row = torch.randn(12, device="cuda", generator=gen)[::2]
    a, b = clipped_policy_loss(lp, old, per_row), clipped_policy_loss(lp, old, per_row.contiguous())
    assert torch.equal(a.loss, b.loss)
    with pytest.raises(CapabilityError):
        clipped_policy_loss(lp.double(), old, adv)
    for args in ((lp[0], old[0], adv[0]), (lp, old[:5], adv), (lp, old.bfloat16(), adv), (lp, old, adv[:, :3]), (lp, old, adv[0]),
                 (lp, old.cpu(), adv), (lp, old, adv, mask[:3]), (lp, old, adv, mask.float()), (lp, old, adv, None, ref[:2])):
        with pytest.raises(ValueError):
            clipped_policy_loss(*args)
    for kw in ({"reduction": "sum"}, {"clip_low": 1.5}, {"clip_high": -0.1}, {"kl_coef": float("nan")}):
        with pytest.raises(ValueError):
            clipped_policy_loss(lp, old, adv, **kw)


# ---- preference loss -----------------------------------------------------------------------------------------------
# The differences of a sequence are each off by u at most before they are added in 64 bits: s by 2u sum |lp - ref| (twice what
# is needed, for the rounding of the reward), the loss by its slope times the errors of both sums, and a rounding.
PAIR_CASES = [(1, 1), (2, 129), (3, 1000), (40, 77), (1, 100003), (600, 3), (1023, 50), (1024, 50), (1025, 1025), (5000, 9), (1, 700_001)]


@pytest.mark.parametrize("pairs,seq", PAIR_CASES)
@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("form", ["tokens,ragged", "sums", "none,ragged,average", "tokens,average"])
def test_preference_loss_and_gradient(native_library, pairs, seq, kind, smoothing, form):
    from molt_b200.kernels import preference_loss

    gen = _gen(pairs + 13 * seq)
    beta = 0.3
    lp = -2 * torch.rand(2 * pairs, seq, device="cuda", generator=gen)
    noise = 3 * torch.randn(2 * pairs, seq, device="cuda", generator=gen) / math.sqrt(seq)
    average = "average" in form
    ref = lp + noise if "tokens" in form else None
    mask = None
    if "ragged" in form:
        mask = torch.rand(2 * pairs, seq, device="cuda", generator=gen) < 0.8
        if pairs > 1:
            mask[1] = False
        lp[~mask] = float("nan")
        if ref is not None:
            ref[~mask] = float("inf")
    if "sums" in form:
        ref = lp.double().sum(1).float() + torch.randn(2 * pairs, device="cuda", generator=gen)
    kept = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask
    leaf = lp.double().requires_grad_()
    diff = torch.where(kept, leaf - (ref.double() if ref is not None and ref.dim() == 2 else 0.0), torch.zeros_like(leaf))
    n = kept.sum(1).clamp(min=1) if average else 1
    s = diff.sum(1) / n
    size = diff.detach().abs().sum(1) / n
    if "sums" in form:
        s, size = s - ref.double(), size + ref.double().abs()
    h = s[:pairs] - s[pairs:]
    ls = torch.nn.functional.logsigmoid
    each = {"sigmoid": -(1 - smoothing) * ls(beta * h) - smoothing * ls(-beta * h), "hinge": (1 - beta * h).clamp(min=0),
            "ipo": (h - 0.5 / beta) ** 2}[kind]
    loss = each.mean()
    (grad,) = torch.autograd.grad(loss, leaf)
    slope = {"sigmoid": beta, "hinge": beta, "ipo": 2 * (h.detach() - 0.5 / beta).abs() + 1e-3}[kind]
    curve = {"sigmoid": beta * beta, "hinge": 0.0, "ipo": 2.0}[kind]
    bound_h = 2 * U * (size[:pairs] + size[pairs:])

    got_leaf = lp.clone().requires_grad_()
    got = preference_loss(got_leaf, ref, mask, beta=beta, label_smoothing=smoothing, kind=kind, average=average)
    _close(got.loss.detach(), loss.detach(), (slope * bound_h).mean() + 2 * U * loss.detach().abs())
    for side, part in ((got.chosen_rewards, slice(0, pairs)), (got.rejected_rewards, slice(pairs, None))):
        _close(side, beta * s.detach()[part], beta * 2 * U * (size[part] + s.detach()[part].abs()))
    scale = torch.tensor(1.75, device="cuda")
    (dlp,) = torch.autograd.grad(got.loss, got_leaf, scale)
    share = (1.0 / n if average else torch.ones_like(s)) / pairs
    per_row = share * torch.cat([curve * bound_h, curve * bound_h])
    _close(dlp, torch.where(kept, grad, torch.zeros_like(grad)) * 1.75, 1.75 * (per_row[:, None] + grad.nan_to_num().abs() * 4 * U) + 1e-38)
    if mask is not None:
        assert not bool(dlp[~mask].any())
    assert not got.chosen_rewards.requires_grad and not got.rejected_rewards.requires_grad
    with torch.no_grad():
        again = preference_loss(lp, ref, mask, beta=beta, label_smoothing=smoothing, kind=kind, average=average)
    assert torch.equal(again.loss, got.loss.detach())


def test_preference_loss_far_margins_and_refusals(native_library):
    from molt_b200.core.errors import CapabilityError
    from molt_b200.kernels import preference_loss

    for margin in (-1e5, -900.0, 0.0, 900.0, 1e5):
        lp = torch.tensor([[margin], [0.0]], device="cuda", requires_grad=True)
        got = preference_loss(lp, beta=1.0)
        got.loss.backward()
        assert float(got.loss) == pytest.approx(max(-margin, 0.0) + math.log1p(math.exp(-abs(margin))), rel=1e-6, abs=0)
        slope = -1.0 / (1.0 + math.exp(margin)) if margin < 700 else -math.exp(-margin)
        assert float(lp.grad[0]) == pytest.approx(slope, rel=1e-6, abs=1e-40) and float(lp.grad[1]) == -float(lp.grad[0])
    # the hinge's corner has slope zero on the flat side
    lp = torch.tensor([[2.0], [0.0]], device="cuda", requires_grad=True)
    preference_loss(lp, beta=0.5, kind="hinge").loss.backward()
    assert lp.grad.tolist() == [[0.0], [0.0]]
    # no token at all: h = 0
    lp = torch.empty(4, 0, device="cuda", requires_grad=True)
    got = preference_loss(lp)
    got.loss.backward()
    assert float(got.loss) == pytest.approx(math.log(2.0), rel=1e-6) and lp.grad.shape == (4, 0)
    lp = torch.randn(4, 9, device="cuda")
    wide = torch.randn(4, 12, device="cuda")
    wide[:, 1:10] = lp
    assert torch.equal(preference_loss(wide[:, 1:10]).loss, preference_loss(lp).loss)
    with pytest.raises(CapabilityError):
        preference_loss(lp.bfloat16())
    for args in ((lp[:3],), (lp[:0],), (lp[0],), (lp, lp[:, :3]), (lp, lp[:2, 0]), (lp, None, torch.ones(4, 9, device="cuda")), (lp, lp.cpu())):
        with pytest.raises(ValueError):
            preference_loss(*args)
    for kw in ({"kind": "exo"}, {"beta": 0.0}, {"label_smoothing": 1.5}, {"label_smoothing": 0.1, "kind": "ipo"}):
        with pytest.raises(ValueError):
            preference_loss(lp, **kw)


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_loss_gradients_against_differences(native_library, which):
    """Central differences of the forward pass along a direction: the loss is O(1) and rounded to 2^-24, the step is 2^-6, so
    the quotient is off by 2^-24 * 4 / 2^-6 = 2^-16 * 1, and by h^2 / 6 |f'''| < 2^-12 / 6 * 4 (ratios below e^2, |v| <= 1)."""
    from molt_b200.kernels import clipped_policy_loss, preference_loss

    gen = _gen(21)
    lp = -torch.rand(6, 40, device="cuda", generator=gen)
    old = lp + 0.05 * torch.randn(6, 40, device="cuda", generator=gen)   # inside the clamp by more than the step
    old = lp + (old - lp).clamp(-0.1, 0.1)
    ref = lp + 0.5 * torch.randn(6, 40, device="cuda", generator=gen)
    adv = torch.rand(6, device="cuda", generator=gen)
    mask = torch.rand(6, 40, device="cuda", generator=gen) < 0.6
    v = torch.rand(6, 40, device="cuda", generator=gen) * 2 - 1
    if which == "preference":
        v = v / 6                                        # a sum over a sequence moves by less than the step

    def loss(x):
        if which == "policy":
            return clipped_policy_loss(x, old, adv, mask, ref, clip_low=0.4, clip_high=0.4, kl_coef=0.2, reduction="sequence").loss
        return preference_loss(x, ref, mask, beta=0.5, label_smoothing=0.1).loss

    leaf = lp.clone().requires_grad_()
    (grad,) = torch.autograd.grad(loss(leaf), leaf)
    h = 2.0 ** -6
    slope = (float(loss(lp + h * v)) - float(loss(lp - h * v))) / (2 * h)
    assert abs(slope - float((grad.double() * v).sum())) < 2 ** -16 + 2 ** -12 / 6 * 4


# ---- gradient norm and clipping ------------------------------------------------------------------------------------
# Eight squares at most are added in fp32 before the sum goes on in 64 bits: 10u relatively, halved by the root, and one
# rounding; 16u = 2^-20 covers norm and coefficient, the product adds u and a rounding to the tensor's type.
LISTS = [[1], [3], [8], [0, 5, 0], [1, 2, 3, 4, 5], [4096, 8192, 8193, 100_003], [1_000_003] * 3, [64] * 700, [17] * 1100, [300_000_000]]


def _grads(sizes, gen, dtypes):
    made = []
    for k, n in enumerate(sizes):
        g = torch.empty(n + 4, dtype=dtypes[k % len(dtypes)], device="cuda").normal_(0.0, 10.0 ** (k % 3 - 1), generator=gen)
        made.append(g[k % 4:k % 4 + n])                  # every alignment that the type allows
    return made


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16, torch.bfloat16)],
                         ids=["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("norm_type", [2.0, float("inf")])
def test_grad_norm_and_clipping(native_library, sizes, dtypes, norm_type):
    from molt_b200.kernels import clip_grad_norm, global_grad_norm

    grads = _grads(sizes, _gen(len(sizes) + sizes[0]), dtypes)
    per = torch.stack([g.double().abs().max() if norm_type != 2.0 else g.double().square().sum() for g in grads if g.numel()])
    want = per.max() if norm_type != 2.0 else per.sum().sqrt()
    got = global_grad_norm(grads, norm_type)
    assert got.shape == () and got.dtype == torch.float32
    _close(got, want, want * (2 ** -20 if norm_type == 2.0 else 0.0) + 1e-300)
    assert torch.equal(got, global_grad_norm(grads, norm_type))
    for max_norm in (float(want) * 0.37, float(want) * 3, 0.0):
        coefficient = min(1.0, max_norm / (float(want) + 1e-6))
        copies = [g.clone() for g in grads]
        outs = [torch.full_like(g, 9.0) for g in grads]
        norm = clip_grad_norm(grads, max_norm, norm_type, out=outs)
        assert torch.equal(norm, got) and all(torch.equal(g, c) for g, c in zip(grads, copies))
        norm = clip_grad_norm(copies, max_norm, norm_type)
        assert torch.equal(norm, got) and all(torch.equal(o, c) for o, c in zip(outs, copies))
        for g, o in list(zip(grads, outs))[:12]:
            want_o = g.double() * coefficient
            _close(o, want_o, want_o.abs() * (2 ** -20 + torch.finfo(g.dtype).eps / 2) + 1e-38)


def test_grad_norm_of_extreme_values(native_library):
    from molt_b200.kernels import clip_grad_norm, global_grad_norm

    for scale in (1e-30, 1e-24, 1e-19, 1e18, 1e25, 1e34):       # squares outside fp32, norms inside
        g = torch.randn(5000, device="cuda", generator=_gen(1)) * scale
        want = g.double().square().sum().sqrt()
        _close(global_grad_norm([g, g[:7].bfloat16()]), (want ** 2 + g[:7].bfloat16().double().square().sum()).sqrt(), want * 2 ** -20)
    mixed = [torch.full((9,), 1e30, device="cuda"), torch.full((9,), 1e-30, device="cuda"), torch.zeros(5, device="cuda")]
    _close(global_grad_norm(mixed), torch.tensor(3e30, device="cuda").double(), torch.tensor(3e30 * 2 ** -20, device="cuda").double())
    for bad in (float("nan"), float("inf"), -float("inf")):
        for dtype in (torch.float32, torch.bfloat16):
            for at in (0, 4999):
                g = torch.ones(5000, device="cuda", dtype=dtype)
                g[at] = bad
                for norm_type in (2.0, float("inf")):
                    norm = float(global_grad_norm([torch.ones(3, device="cuda"), g], norm_type))
                    assert math.isnan(norm) if math.isnan(bad) else norm == float("inf")
    zero = torch.zeros(100, device="cuda")
    assert float(clip_grad_norm([zero], 1.0)) == 0.0 and not bool(zero.any())
    nothing = torch.empty(0, 7, device="cuda")
    assert float(clip_grad_norm([nothing], 1.0)) == 0.0 and float(global_grad_norm([nothing, nothing], float("inf"))) == 0.0


def test_grad_norm_layouts_and_refusals(native_library):
    from molt_b200.core.errors import CapabilityError
    from molt_b200.kernels import clip_grad_norm, global_grad_norm

    gen = _gen(2)
    turned = torch.randn(30, 50, device="cuda", generator=gen).t()          # dense, in another order
    channels = torch.randn(2, 3, 4, 5, device="cuda", generator=gen).to(memory_format=torch.channels_last)
    want = (turned.double().square().sum() + channels.double().square().sum()).sqrt()
    copy = [turned.double() / want / 2, channels.double() / want / 2]
    _close(clip_grad_norm([turned, channels], 0.5), want, want * 2 ** -20)
    for t, c in zip((turned, channels), copy):
        _close(t, c, c.abs() * 2 ** -19 + 1e-6 * c.abs())
    matrix, flat = torch.randn(6, 7, device="cuda", generator=gen), torch.zeros(50, device="cuda")
    clip_grad_norm(matrix, 1e9, out=flat[3:45])             # contiguous outputs may have other shapes
    assert torch.equal(flat[3:45].view(6, 7), matrix) and not bool(flat[:3].any()) and not bool(flat[45:].any())
    a, b = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(CapabilityError):
        global_grad_norm([a.half()])
    with pytest.raises(CapabilityError):
        global_grad_norm([a, b.cpu()])
    for bad in ([torch.ones(4, 4, device="cuda")[:, :2]], [torch.ones(1, device="cuda").expand(4)]):
        with pytest.raises(ValueError):
            global_grad_norm(bad)
    for grads, out in (([a, b], [b]), ([a], [b.bfloat16()]), ([a], [b[:4]]), ([turned], [torch.empty(50, 30, device="cuda")])):
        with pytest.raises(ValueError):
            clip_grad_norm(grads, 1.0, out=out)
    for grads, out in (([a, a], None), ([a, b], [b, a]), ([a, a[4:]], None), ([a, b], [a, a])):
        with pytest.raises(ValueError, match="overlaps"):
            clip_grad_norm(grads, 1.0, out=out)
    _close(global_grad_norm([a, a]), torch.tensor(4.0).cuda().double(), torch.tensor(2 ** -18).cuda())   # reading twice is fine
    leaf = torch.ones(4, device="cuda", requires_grad=True)
    y = (leaf * a[:4]).sum()
    clip_grad_norm([a], 0.5)                               # overwrites what the backward pass needs
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# ---- together ------------------------------------------------------------------------------------------------------


def _policy_step(logits, ids, old, adv, mask, out):
    from molt_b200.kernels import clip_grad_norm, clipped_policy_loss, token_logprobs

    lp = token_logprobs(logits, ids, 0.9)
    loss = clipped_policy_loss(lp, old, adv, mask, old, kl_coef=0.1, reduction="sequence").loss
    (grad,) = torch.autograd.grad(loss, logits)
    return loss.detach(), clip_grad_norm([grad], 0.01, out=[out]), out


def test_run_together_eager_on_a_stream_and_as_a_graph(native_library):
    """Logits to clipped gradient against 64 bits; the same bits on another stream and from a captured graph that is
    replayed with other inputs, beside a second graph."""
    gen = _gen(31)
    batch, seq, vocab = 5, 33, 1537

    def inputs():
        logits = torch.randn(batch, seq, vocab, device="cuda", generator=gen).requires_grad_()
        ids = torch.randint(0, vocab, (batch, seq), device="cuda", generator=gen)
        old = torch.log_softmax(logits.detach() / 0.9, -1).gather(-1, ids[..., None])[..., 0] + 0.2 * torch.randn(
            batch, seq, device="cuda", generator=gen)
        mask = torch.rand(batch, seq, device="cuda", generator=gen) < 0.8
        mask[3] = False
        return [logits, torch.where(mask, ids, -100), old, torch.randn(batch, device="cuda", generator=gen), mask]

    first, second = inputs(), inputs()
    out = torch.empty(batch, seq, vocab, device="cuda")
    results = []
    for data in (first, second):
        loss, norm, got = (t.clone() for t in _policy_step(*data, out))
        logits, ids, old, adv, mask = data
        x = logits.detach().double().requires_grad_()
        lp = torch.log_softmax(x / 0.9, -1).gather(-1, ids.clamp(min=0)[..., None])[..., 0]
        r = torch.exp(lp - old.double())
        a = adv.double()[:, None]
        e = old.double() - lp
        each = -torch.minimum(r * a, r.clamp(0.8, 1.2) * a) + 0.1 * (torch.expm1(e) - e)
        n = mask.sum(1)
        want = (each * mask).sum(1)[n > 0].div(n[n > 0]).mean()
        (g,) = torch.autograd.grad(want, x)
        # log-probabilities are off by < 100u, which moves ratios, k and their slopes by < 100u of O(1) magnitudes
        assert abs(float(loss) - float(want)) < 400 * U * float((each.abs() * mask).max())
        assert float(norm) == pytest.approx(float(g.norm()), rel=400 * U)
        clipped = g * min(1.0, 0.01 / (float(g.norm()) + 1e-6))
        assert float((got.double() - clipped).norm()) < 800 * U * float(clipped.norm())
        results.append((loss, norm, got))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [t.clone() for t in _policy_step(*second, torch.empty_like(out))]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(again, results[1]))

    graphs = []
    for data in (first, second):
        held = [t.detach().clone() for t in data]
        held[0].requires_grad_()
        target = torch.empty_like(out)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _policy_step(*held, target)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            produced = _policy_step(*held, target)
        graphs.append((graph, held, produced))
    for swap in (False, True):
        for (graph, held, produced), data in zip(graphs, (second, first) if swap else (first, second)):
            with torch.no_grad():
                for h, d in zip(held, data):
                    h.copy_(d)
            graph.replay()
        for (graph, held, produced), want in zip(graphs, reversed(results) if swap else results):
            assert all(torch.equal(a, b) for a, b in zip(produced, want))


def test_two_streams_at_once(native_library):
    """The same operators in flight on two streams, each with its own scratch."""
    from molt_b200.kernels import clip_grad_norm, preference_loss, token_logprobs_with_grad

    def work(seed):
        gen = _gen(seed)
        logits = torch.randn(64, 30001, device="cuda", generator=gen).bfloat16()
        ids = torch.randint(0, 30001, (64,), device="cuda", generator=gen)
        pairs = torch.randn(64, 4001, device="cuda", generator=gen)
        grads = [torch.randn(100_003, device="cuda", generator=gen) for _ in range(5)]
        return logits, ids, pairs, grads

    def run(logits, ids, pairs, grads):
        lp, grad = token_logprobs_with_grad(logits, ids)
        got = preference_loss(pairs)
        outs = [torch.empty_like(g) for g in grads]
        return [lp, grad, got.loss, got.chosen_rewards, clip_grad_norm(grads, 1.0, out=outs), *outs]

    data = [work(1), work(2)]
    want = [run(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(4):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k] = run(*data[k])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
