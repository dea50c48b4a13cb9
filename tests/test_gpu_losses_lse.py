"""token_logprob_grad with the lse of more classes than its logits hold (a
vocabulary split by class), at every size of lse."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_losses import DTYPES, HALF, TINY, U, L, close, make_target  # noqa: E402,F401  (L: the fixture)

pytestmark = pytest.mark.gpu


def shard_gradient(z64, y, lse, first, temperature):
    """The formula on classes first .. first + columns, in 64 bits; y counts all classes."""
    d = -torch.exp(z64 / temperature - lse[:, None])
    here = (y >= first) & (y < first + z64.shape[1])
    d[here.nonzero()[:, 0], y[here] - first] += 1.0
    return d / temperature


# one row a workgroup, and few long rows by chunks
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,cut", [(6, 3000, 1000), (300, 20001, 9001), (3, 120001, 60001), (5, 40000, 1)])
@pytest.mark.parametrize("shift", [0.0, 300.0, -300.0])
def test_classes_in_two_parts(L, dtype, rows, vocab, cut, shift):  # noqa: F811
    temperature = 0.9
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    z = (torch.randn(rows, vocab, generator=g, device="cuda") * 2.5 + shift).to(DTYPES[dtype])
    z[2, :cut] = float("-inf")  # all of a row's first part masked out
    y = make_target(rows, vocab).cuda()
    y[0], y[1] = 0, vocab - 1
    parts = [(z[:, :cut], 0), (z[:, cut:], cut)]
    own = []
    for part, first in parts:
        t = torch.where((y >= first) & (y < first + part.shape[1]), y - first, 0)
        own.append(L.token_logprob(part, t, temperature=temperature)[1].double())
    whole = torch.logsumexp(z.double() / temperature, 1)
    lse = torch.logaddexp(*own)
    # 64 bits from here on, but for the lse's rounding to 32 and its parts'
    close(lse, whole.cpu(), 8 * U * (whole.abs().cpu() + 20))
    lse = lse.float()
    for part, first in parts:
        here = (y >= first) & (y < first + part.shape[1])
        keep = here.nonzero()[:, 0]
        # rows whose class lies in this part
        rowsof = part[keep]
        got = L.token_logprob_grad(rowsof, y[keep] - first, lse[keep], torch.ones(len(keep), device="cuda"),
                                   temperature=temperature)
        want = shard_gradient(rowsof.double(), y[keep], lse[keep].double(), first, temperature).cpu()
        p = torch.exp(rowsof.double() / temperature - lse[keep].double()[:, None]).cpu()
        # the probability's exponent is off by U of its size and of the lse's,
        # taken twice where the row's own stands for the lse given; then one rounding
        logp = torch.where(p > 0, p.log().abs(), 0.0)
        rel = U * (4 * logp + 8) + 2 * U * lse[keep].abs().double().cpu()[:, None]
        tol = (p * rel + 2 * U) / temperature + want.abs() * HALF[got.dtype] * 1.01 + TINY[got.dtype]
        close(got, want, tol)


def test_the_rows_own_lse_beyond_32_bits(L):  # noqa: F811
    # masked with the type's lowest value throughout: the lse's 32 bits hold nothing of the classes' number
    for dtype in DTYPES.values():
        z = torch.full((3, 5000), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        y = torch.tensor([0, 7, 4999]).cuda()
        _, lse = L.token_logprob(z, y)
        d = L.token_logprob_grad(z, y, lse, torch.ones(3).cuda())
        share = torch.full((3, 5000), -1 / 5000, dtype=torch.float64)
        share[torch.arange(3), y.cpu()] += 1
        close(d, share, share.abs() * (HALF[dtype] + 8 * U) + U)
