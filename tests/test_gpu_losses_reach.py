"""The softmax losses at sizes that pick each of their kernels: what is noted
beside a case is the rule of dlr_losses.hip that it stands for.  Tolerances as in
test_gpu_losses.py."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_losses import (DTYPES, HALF, L, TINY, U, close, gen, lse_tol, make_target,  # noqa: E402,F401
                             ref_logprob)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------ head

HEADS = [
    (1, 131072, 520),   # 256 classes a workgroup; eight whole stages and a short one
    (1, 98304, 64),     # the fewest classes for that; one whole stage
    (16, 98309, 1000),  # the last tile nearly empty; 15 whole stages and a short one
    (9, 100003, 8),     # no whole stage
    (3, 20011, 1000),   # 64 classes a workgroup, four stages in flight, a short one
    (16, 9000, 256),    # as many stages as are in flight
    (2, 8200, 264),     # one more, short
    (7, 8000, 1016),    # few tiles: the dimension over four waves
    (17, 70001, 200),   # more than 16 rows: three whole stages and a short one
    (40, 50257, 584),
    (64, 8192, 520),    # few tiles of 64 rows
    (200, 32000, 648),
    (333, 50257, 584),  # two kinds of tiles, both with a short last stage
    (600, 30001, 136),  # no more whole stages than are in flight
    (700, 50257, 1000),
    (700, 30001, 328),
    (1500, 50257, 72),
    (2100, 1000, 520),
]


def seams(vocab):
    """Classes at the ends of tiles of 64 to 256, and of the whole."""
    at = {0, vocab - 1, vocab // 2}
    for tile in (64, 128, 256):
        for n in (1, vocab // tile // 3, vocab // tile):
            at |= {n * tile - 1, n * tile}
    return sorted(a for a in at if 0 <= a < vocab)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,dim", HEADS)
def test_head(L, rows, vocab, dim, dtype):  # noqa: F811
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + dim)
    x = torch.randint(-2, 3, (rows, dim), generator=g, device="cuda").to(DTYPES[dtype])
    w = torch.randint(-2, 3, (vocab, dim), generator=g, device="cuda").to(DTYPES[dtype])
    scale = 1.0 + math.sqrt(dim)
    z = torch.mm(x.double(), w.double().t()).cpu()  # whole numbers: exact, in 32 bits too
    e = lse_tol(vocab) + U * 36
    want_lse = torch.logsumexp(z / scale, 1)
    places = seams(vocab)
    first = None
    for at in range(0, len(places), max(1, min(rows, len(places)))):
        some = torch.tensor((places[at:] + places)[:len(places)])
        y = some.repeat(rows // len(places) + 1)[:rows].clone()
        if rows > 3:
            y[2] = -1
        lp, lse = L.head_logprob(x, w, y.cuda(), temperature=scale)
        want, want_l = ref_logprob(z, y, scale)
        close(lse, want_l, e + U * want_lse.abs())
        close(lp, want, e + U * want.abs())
        if first is not None:
            assert torch.equal(lse, first)
        first = lse


# -------------------------------------------------------------------- gradients

def residual(z64, y, lse, coef, temperature):
    # beyond |lse| = 128 the row's own softmax (64 bits of the lse of lowest values hold nothing of it either)
    p = torch.where(lse.abs()[:, None] > 128, torch.softmax(z64 / temperature, 1),
                    torch.exp(z64 / temperature - lse[:, None]))
    one = torch.zeros_like(p).scatter_(1, y.clamp(min=0)[:, None], 1.0)
    return (coef / temperature)[:, None] * (one - p), p


def check(L, z, y, temperature, over, same):  # noqa: F811
    """token_logprob_grad of the rows of z against the formula, into a tensor of its own and over the logits."""
    rows = z.shape[0]
    _, lse = L.token_logprob(z, y, temperature=temperature)
    g = torch.randn(rows, generator=gen(3)).cuda()
    g[rows // 2] = 0.0
    got = L.token_logprob_grad(z, y, lse, g, temperature=temperature)
    pick = torch.tensor(sorted({0, min(1, rows - 1), rows // 2, rows - 1})).cuda()
    z64, lse64 = z[pick].double(), lse[pick].double()
    coef = torch.where(y[pick] >= 0, g[pick].double(), 0.0)
    want, p = residual(z64, y[pick], lse64, coef, temperature)
    logp = torch.where(p > 0, p.log().abs(), 0.0)
    # p's exponent is off by 2^-24 of its size, and of z's and the lse's up to 128;
    # its factors by 2^-24 each; then one rounding to the gradient's type
    rel = U * (3 * logp + 8 + 2 * lse64.abs().clamp(max=128)[:, None])
    size = coef.abs()[:, None] / temperature
    tol = size * (p * rel + 2 * U * (want != 0)) + want.abs() * HALF[z.dtype] * 1.01 + TINY[z.dtype]
    close(got[pick], want.cpu(), tol.cpu())
    if over:
        assert L.token_logprob_grad(z, y, lse, g, temperature=temperature, out=z) is z
        close(z[pick], want.cpu(), tol.cpu())
        # by chunks and whole, rows beyond |lse| = 128 add their statistics in another order
        assert torch.equal(z, got) or not same


def make(rows, vocab, dtype, shift, pad=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + vocab)
    z = (torch.randn(rows, vocab + pad, generator=g, device="cuda") * 2.5 + shift).to(DTYPES[dtype])
    return z[:, :vocab], make_target(rows, vocab, ignore=(1,)).cuda()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("packs,tail", [(2049, 0), (2047, 3), (4096, 1), (12564, 1), (16384, 0), (16384, 3), (16385, 0),
                                        (257, 1), (1025, 2)])
@pytest.mark.parametrize("shift", [0.0, 250.0])
def test_gradient_of_many_rows(L, dtype, packs, tail, shift):  # noqa: F811
    # more than 256 rows: a row a workgroup, of 64 to 1,024 threads by its packs of 16 bytes
    vocab = packs * (4 if dtype == "f32" else 8) + tail
    z, y = make(259, vocab, dtype, shift, pad=1)
    check(L, z, y, 0.9, over=True, same=True)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,packs", [(1, 2048), (3, 9000), (256, 2048), (256, 2500), (40, 17001)])
@pytest.mark.parametrize("shift", [0.0, 250.0, -250.0])
def test_gradient_of_few_long_rows(L, dtype, rows, packs, shift):  # noqa: F811
    # by chunks into a tensor of its own, whole over the logits
    vocab = packs * (4 if dtype == "f32" else 8) + 3
    z, y = make(rows, vocab, dtype, shift, pad=5)
    if rows > 2:
        z[2, : vocab // 2] = float("-inf")
    check(L, z, y, 1.1, over=True, same=shift == 0.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_lowest_values_in_long_rows(L, dtype):  # noqa: F811
    # the lse's 32 bits hold nothing of the row: its own statistics, in every chunk and over the logits
    vocab = 40003
    z, y = make(3, vocab, dtype, 0.0)
    low = torch.finfo(z.dtype).min
    z[0, 100:] = low  # a few classes left
    z[2] = low        # none: uniform
    for over in (False, True):
        check(L, z, y, 1.0, over, same=False)
