"""How near the softmax losses come to their formulas in 64 bits: errors that
lie to one side, which a bound per element does not see.  U = 2^-24, half a
step of float32."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_losses import U, gen, L  # noqa: E402,F401  (L: the fixture)

pytestmark = pytest.mark.gpu

# v_exp_f32's mean error, measured over [-24, 0]: at most 8e-8
EXP = 8e-8


def wide_logits(rows, vocab, shift, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(rows, vocab, generator=g, device="cuda") * 2.5 + shift


def mean_error(grad, p, coef, y):
    """Each row's mean of (-grad_j / (coef p_j)) - 1 over the classes but y."""
    q = grad.double() / (-coef[:, None] * p) - 1.0
    q.scatter_(1, y[:, None], 0.0)
    return q.sum(1) / (q.shape[1] - 1)


# (rows, classes): a row a workgroup, a row by chunks; policy_loss: a row held whole and in part
SHAPES = [(200, 1000), (130, 50257), (3, 50257), (129, 100003), (2, 200003)]


@pytest.mark.parametrize("temperature", [0.7, 0.8, 1.0, 1.3])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_policy_gradient_errs_to_no_side(L, rows, vocab, temperature):  # noqa: F811
    z = wide_logits(rows, vocab, 0.0, rows)
    y = torch.randint(0, vocab, (rows,), generator=gen(1)).cuda()
    x = z.double() / temperature
    lse = torch.logsumexp(x, 1)
    lp = x.gather(1, y[:, None])[:, 0] - lse
    old = lp.float()
    out = L.policy_loss(z, y, old, torch.ones(rows, device="cuda"), clip_low=1.0, clip_high=1.0,
                        temperature=temperature)
    coef = -torch.exp(lp - old.double()) / temperature  # advantage 1, nothing clipped
    # one rounding each of the coefficient and of it over the row's sum, the
    # sum's and the log-probability's own errors (within U each), the exponentials'
    # mean; what is random in the classes leaves less than U / sqrt(vocab) * 50
    bound = 4 * U + EXP + 50 * U / math.sqrt(vocab)
    err = mean_error(out.grad, torch.exp(x - lse[:, None]), coef, y).abs()
    assert float(err.max()) <= bound, float(err.max())


@pytest.mark.parametrize("temperature", [0.7, 0.9, 1.0, 1.7])
@pytest.mark.parametrize("shift", [0.0, -60.0, 50.0, 400.0])
@pytest.mark.parametrize("rows,vocab", [(200, 1000), (300, 10007), (3, 50257)])
def test_logprob_gradient_errs_to_no_side(L, rows, vocab, shift, temperature):  # noqa: F811
    z = wide_logits(rows, vocab, shift, rows)
    y = torch.randint(0, vocab, (rows,), generator=gen(1)).cuda()
    _, lse = L.token_logprob(z, y, temperature=temperature)
    grad = L.token_logprob_grad(z, y, lse, torch.ones(rows, device="cuda"), temperature=temperature)
    x = z.double() / temperature
    # up to |lse| = 128 the probabilities are of the lse given, in 32 bits; beyond of the row itself
    own = torch.logsumexp(x, 1)
    base = torch.where(lse.abs() > 128, own, lse.double())
    coef = torch.full((rows,), 1.0 / temperature, dtype=torch.float64, device="cuda")
    err = mean_error(grad, torch.exp(x - base[:, None]), coef, y).abs()
    # as above, without a log-probability; the exponent's rounding is random
    # and at most half a step of 256: 2^-17
    bound = 3 * U + EXP + 50 * U / math.sqrt(vocab) + 2.0 ** -17 * 5 / math.sqrt(vocab) * (abs(shift) < 100)
    assert float(err.max()) <= bound, float(err.max())


# Errors of lse, with rows shifted so that it is about 0 and its own rounding does
# not hide them.  The sum's terms are off by random shares of U that average out,
# and by the exponentials' mean; its roundings in a tree are random too.  So the mean
# over the rows is within EXP + U, and one row's (a spread of a quarter of U and its
# own rounding, U / 2 up to 1) within 2 U of that.
def check_errors(lse, want):
    err = lse.double() - want
    assert float(want.abs().max()) <= 1.0
    assert float(err.mean().abs()) <= EXP + U, float(err.mean())
    assert float(err.pow(2).mean().sqrt()) <= EXP + 2 * U, float(err.pow(2).mean().sqrt())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.3])
@pytest.mark.parametrize("rows,vocab", [(400, 1000), (400, 50257), (300, 131072), (100, 131072)])
def test_lse_errs_to_no_side(L, rows, vocab, temperature, dtype):  # noqa: F811
    z = wide_logits(rows, vocab, 0.0, vocab)
    z -= torch.logsumexp(z.double() / temperature, 1, keepdim=True).float() * temperature
    if dtype == "bf16":
        z = z.bfloat16()
    want = torch.logsumexp(z.double() / temperature, 1)
    y = torch.randint(0, vocab, (rows,), generator=gen(1)).cuda()
    lp, lse = L.token_logprob(z, y, temperature=temperature)
    check_errors(lse, want)
    # logprob: the same lse, rounded where it is about 10
    exact = z.double().gather(1, y[:, None])[:, 0] / temperature - want
    err = lp.double() - exact
    step = exact.abs() * U
    assert bool((err.abs() <= step + EXP + 2 * U + 4 * U).all()), float(err.abs().max())


@pytest.mark.parametrize("rows,vocab,dim", [(400, 50257, 520), (300, 20011, 264), (16, 131072, 520), (130, 9000, 261)])
def test_head_lse_errs_to_no_side(L, rows, vocab, dim):  # noqa: F811
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    x = torch.randint(-2, 3, (rows, dim), generator=g, device="cuda").bfloat16()
    w = torch.randint(-2, 3, (vocab, dim), generator=g, device="cuda").bfloat16()
    scale = 0.8 * math.sqrt(dim)
    # four columns of every class take each row's lse off: whole numbers up to 256 are exact
    x[:, -4:], w[:, -4:] = 0.0, -1.0
    z = torch.mm(x.double(), w.double().t())
    off = torch.round(torch.logsumexp(z / scale, 1) * scale)
    x[:, -4:] = torch.stack([torch.floor((off + i) / 4) for i in range(4)], 1).bfloat16()
    z = torch.mm(x.double(), w.double().t())
    assert float((z - torch.round(z)).abs().max()) == 0.0
    y = torch.randint(0, vocab, (rows,), generator=gen(1)).cuda()
    _, lse = L.head_logprob(x, w, y, temperature=scale)
    check_errors(lse, torch.logsumexp(z / scale, 1))
