"""The softmax losses against their formulas in 64 bits (on the CPU).

Tolerances, with u = 2^-24 (half a step of float32) and h = half a step of
the gradient's type, relative:

* lse: each term 2^((z - m) k) has a relative error of at most u (2 |d| + 3),
  d = (z - m) / temperature (k's rounding and the product's, then the
  exponential's unit in the last place); the mean of |d| under the softmax is
  at most ln vocab.  A thread adds ceil(vocab / 512) terms, then 6 + 16 joins
  of 3 roundings: ADDS.  So lse is off by u (2 ln vocab + 3 + ADDS), plus its
  own rounding u |lse|; logprob likewise.
* a gradient coef (1[j = y] - p_j): p_j off by a relative
  u (3 |x| + |z / temperature| + 8) + the error of lse, x = log p_j; coef by
  what its formula's derivative makes of logprob's error; then one rounding.
* preference: everything in 64 bits, one rounding at the end.
* head: products are exact in 32 bits, their sum over dim is off by at most
  dim u sum |x w|; with small whole numbers the logits are exact.
"""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}  # smallest steps, flushed 32-bit ones


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import distlr_amd.losses as losses
    return losses


@pytest.fixture(scope="module")
def dlr():
    import distlr_amd
    return distlr_amd


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def make_logits(rows, vocab, dtype, pad=0, seed=0, scale=2.5):
    """(device view with rows vocab + pad apart, 64-bit copy)."""
    z = (torch.randn(rows, vocab + pad, generator=gen(seed)) * scale).to(dtype)
    return z.cuda()[:, :vocab], z[:, :vocab].double()


def make_target(rows, vocab, seed=1, ignore=()):
    y = torch.randint(0, vocab, (rows,), generator=gen(seed))
    for r in ignore:
        if r < rows:
            y[r] = -100
    return y


def lse_tol(vocab):
    return U * (2 * math.log(vocab + 1) + 3 + math.ceil(vocab / 512) + 22 * 3)


def ref_logprob(z, y, temperature):
    x = z / temperature
    lse = torch.logsumexp(x, 1)
    lp = x.gather(1, y.clamp(min=0)[:, None])[:, 0] - lse
    return torch.where(y >= 0, lp, 0.0), torch.where(y >= 0, lse, 0.0)


def close(got, want, tol):
    got = got.detach().cpu().double()
    err = (got - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float(err.max()), got[bad][:4], want[bad][:4])


def check_grad(got, z, y, coef, coef_err, temperature, extra=0.0, lse=None):
    """got ~ coef / temperature (one_hot - softmax); coef is 0 in rows out."""
    x = z / temperature
    logp = x - (torch.logsumexp(x, 1, keepdim=True) if lse is None else lse[:, None])
    p = torch.exp(logp)
    c = (coef / temperature)[:, None]
    one = torch.zeros_like(p).scatter_(1, y.clamp(min=0)[:, None], 1.0)
    want = torch.where(c != 0, c * (one - p), 0.0)
    rel = U * (3 * logp.abs() + x.abs() + 8) + extra
    tol = c.abs() * p * torch.where(p > 0, rel, 0.0) + c.abs() * one * 2 * U
    tol = tol + (coef_err / temperature)[:, None] * (one - p).abs()
    tol = tol + want.abs() * (HALF[got.dtype] + 2 * U) * 1.01 + TINY[got.dtype]
    close(got, want, torch.where(c != 0, tol, 0.0))


SHAPES = [(1, 1, 0), (3, 1, 3), (2, 2, 0), (5, 7, 1), (4, 8, 0), (3, 9, 2), (1, 511, 0), (3, 513, 5), (17, 1000, 0),
          (2, 4097, 7), (3, 16389, 0), (2, 50257, 47), (260, 129, 0), (1, 131075, 0), (5, 262147, 3),
          (100, 65541, 1)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,pad", SHAPES)
def test_token_logprob(L, rows, vocab, pad, dtype):
    z, z64 = make_logits(rows, vocab, DTYPES[dtype], pad)
    y = make_target(rows, vocab, ignore=(1,))
    for temperature, yy in ((1.0, y.cuda()), (0.7, y.int().cuda())):
        lp, lse = L.token_logprob(z, yy, temperature=temperature)
        want_lp, want_lse = ref_logprob(z64, y, temperature)
        t = lse_tol(vocab)
        close(lse, want_lse, t + U * want_lse.abs())
        close(lp, want_lp, t + U * want_lp.abs())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,pad", SHAPES)
def test_token_logprob_grad(L, rows, vocab, pad, dtype):
    z, z64 = make_logits(rows, vocab, DTYPES[dtype], pad)
    y = make_target(rows, vocab, ignore=(1,))
    g = torch.randn(rows, generator=gen(5))
    g[2 % rows] = 0.0
    lse = ref_logprob(z64, y, 0.7)[1].float()
    before = z.clone()
    d = L.token_logprob_grad(z, y.cuda(), lse.cuda(), g.cuda(), temperature=0.7)
    assert d.dtype == z.dtype and d.shape == z.shape and torch.equal(z, before)
    check_grad(d, z64, y, torch.where(y >= 0, g.double(), 0.0), torch.zeros(rows).double(), 0.7, lse=lse.double())


def test_grad_over_the_logits_and_in_a_wider_tensor(L):
    for dtype in DTYPES.values():
        z, z64 = make_logits(9, 1003, dtype, 5)
        y = make_target(9, 1003, ignore=(4,)).cuda()
        lp, lse = L.token_logprob(z, y)
        g = torch.randn(9, generator=gen(2)).cuda()
        d = L.token_logprob_grad(z, y, lse, g)
        wide = torch.full((9, 1011), 7.0, dtype=dtype, device="cuda")
        got = L.token_logprob_grad(z, y, lse, g, out=wide[:, 3:1006])
        assert got.data_ptr() == wide[:, 3:].data_ptr() and torch.equal(wide[:, 3:1006], d)
        assert (wide[:, :3] == 7.0).all() and (wide[:, 1006:] == 7.0).all()
        whole = z._base if z._base is not None else z
        pad = whole[:, 1003:].clone()
        assert L.token_logprob_grad(z, y, lse, g, out=z) is z
        assert torch.equal(z, d) and torch.equal(whole[:, 1003:], pad)


def policy_inputs(rows, seed, lp):
    g = gen(seed)
    shift = 0.3 * torch.randn(rows, generator=g).double()
    for border in (math.log(0.8), math.log(1.3)):
        shift = torch.where((shift - border).abs() < 1e-3, border + 2e-3, shift)
    old = (lp - shift).float()
    ref = (lp + 0.5 * torch.randn(rows, generator=g).double()).float()
    adv = torch.randn(rows, generator=g)
    adv[:1] = 0.0 if rows > 2 else adv[:1]
    w = torch.rand(rows, generator=g) + 0.1
    return old, ref, adv, w


def ref_policy(lp, old, ref, adv, w, lo, hi, klc):
    """Per row in 64 bits: (loss, kl, clipped, d loss / d logprob * w), and
    |d loss / d logprob| without cancellation, for the tolerance."""
    old, adv, w = old.double(), adv.double(), w.double()
    r = torch.exp(lp - old)
    clipped = ((adv > 0) & (r > 1 + hi)) | ((adv < 0) & (r < 1 - lo))
    surrogate = torch.minimum(r * adv, r.clamp(1 - lo, 1 + hi) * adv)
    slope = torch.where(clipped, 0.0, -r * adv)
    size = (r * adv).abs()
    kl = torch.zeros_like(lp)
    if ref is not None:
        gap = ref.double() - lp
        kl = torch.expm1(gap) - gap
        slope = slope - klc * torch.expm1(gap)
        size = size + klc * torch.exp(gap)
    return klc * kl - surrogate, kl, clipped, slope * w, size


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,pad", SHAPES)
def test_policy_loss(L, rows, vocab, pad, dtype):
    z, z64 = make_logits(rows, vocab, DTYPES[dtype], pad)
    y = make_target(rows, vocab, ignore=(1,))
    tau, lo, hi, klc = 0.8, 0.2, 0.3, 0.05
    lp, _ = ref_logprob(z64, y, tau)
    old, ref, adv, w = policy_inputs(rows, 3, lp)
    if rows > 3:
        w[3] = 0.0
    used = (y >= 0) & (w != 0)
    loss, kl, clipped, coef, size = ref_policy(lp, old, ref, adv, w, lo, hi, klc)
    out = L.policy_loss(z, y.cuda(), old.cuda(), adv.cuda(), ref_logprob=ref.cuda(), weight=w.cuda(), clip_low=lo,
                        clip_high=hi, kl_coef=klc, temperature=tau)
    e = lse_tol(vocab)  # logprob's error before its rounding
    zero = torch.zeros_like(lp)
    close(out.logprob, torch.where(used, lp, zero), e + U * lp.abs())
    close(out.kl, torch.where(used, kl, zero), e * torch.expm1(ref.double() - lp).abs() + 2 * e * e + 2 * U * kl.abs())
    close(out.loss, torch.where(used, loss, zero), 2 * e * size + 2 * U * loss.abs() + 2 * U * kl)
    assert torch.equal(out.clipped.cpu(), clipped & used)
    check_grad(out.grad, z64, y, torch.where(used, coef, zero), w.double() * (2 * e * size) + 2 * U * coef.abs(), tau,
               extra=e)
    assert out.grad.dtype == z.dtype
    # the loss without its gradient, over the logits, and without the KL term
    alone = L.policy_loss(z, y.cuda(), old.cuda(), adv.cuda(), ref_logprob=ref.cuda(), weight=w.cuda(), clip_low=lo,
                          clip_high=hi, kl_coef=klc, temperature=tau, grad=False)
    assert alone.grad is None
    for a, b in zip(alone[:4], out[:4]):
        assert torch.equal(a, b)
    plain = L.policy_loss(z, y.cuda(), old.cuda(), adv.cuda(), clip_low=lo, clip_high=hi, temperature=tau)
    loss, kl, clipped, coef, size = ref_policy(lp, old, None, adv, torch.ones(rows), lo, hi, 0.0)
    used = y >= 0
    close(plain.loss, torch.where(used, loss, zero), 2 * e * size + 2 * U * loss.abs())
    assert (plain.kl == 0).all()
    check_grad(plain.grad, z64, y, torch.where(used, coef, zero), 2 * e * size + 2 * U * coef.abs(), tau, extra=e)
    same = L.policy_loss(z, y.cuda(), old.cuda(), adv.cuda(), ref_logprob=ref.cuda(), weight=w.cuda(), clip_low=lo,
                         clip_high=hi, kl_coef=klc, temperature=tau, out=z)
    assert same.grad is z and torch.equal(z, out.grad) and torch.equal(same.loss, out.loss)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [5, 700, 4100, 40001, 140003])
def test_masked_classes_infinities_and_nan(L, dtype, vocab):
    inf, nan = float("inf"), float("nan")
    rows = 8
    z, z64 = make_logits(rows, vocab, DTYPES[dtype])
    y = make_target(rows, vocab)
    edit = torch.zeros(rows, vocab)
    edit[1, :] = -inf          # all classes but one are masked out
    edit[1, y[1]] = 0.0
    edit[2, vocab // 2] = -inf
    y[2] = (vocab // 2 + 1) % vocab
    edit[3, y[3]] = -inf       # the given class is masked out
    edit[4, :] = -inf          # nothing left
    edit[5, 3 % vocab] = nan
    edit[6, 2] = inf
    y[0], edit[0, :] = -1, nan  # a row that takes no part holds anything
    y[7] = vocab               # out of range: NaN, nothing read
    z += edit.to(z.dtype).cuda()
    z64 = z64 + edit.double()
    lp, lse = (t.cpu() for t in L.token_logprob(z, y.cuda()))
    assert lp[0] == 0 and lse[0] == 0
    assert lp[1].abs() <= lse_tol(1) + 1e-6 and abs(lse[1] - z64[1, y[1]]) <= U * 4 * abs(float(z64[1, y[1]]))
    want, _ = ref_logprob(z64[2:3], y[2:3], 1.0)
    assert abs(lp[2] - want[0]) <= lse_tol(vocab) + U * abs(want[0])
    assert lp[3] == -inf and math.isfinite(lse[3])
    assert lse[4] == -inf and math.isnan(lp[4])
    assert math.isnan(lp[5]) and math.isnan(lse[5]) and math.isnan(lp[6]) and math.isnan(lp[7])
    g = torch.ones(rows)
    d = L.token_logprob_grad(z, y.cuda(), lse.cuda(), g.cuda()).cpu().double()
    assert (d[0] == 0).all() and d[1].abs().max() <= HALF[z.dtype] + 1e-5
    assert d[2, vocab // 2] == 0 and torch.isfinite(d[1:4]).all()
    assert abs(d[3, y[3]] - 1.0) <= HALF[z.dtype]
    assert torch.isnan(d[5]).all() and torch.isnan(d[7]).all()
    g[:] = 0.0  # nothing flows back: zeros, whatever the rows hold
    assert (L.token_logprob_grad(z, y.cuda(), lse.cuda(), g.cuda()) == 0).all()
    one = torch.ones(rows).cuda()
    out = L.policy_loss(z, y.cuda(), lp.cuda().nan_to_num(0, 0, 0), one, ref_logprob=one * -1, kl_coef=0.1)
    assert out.loss[0] == 0 and out.kl[0] == 0 and (out.grad[0] == 0).all() and not out.clipped[0]
    assert torch.isfinite(out.grad[1:3]).all() and torch.isfinite(out.loss[1:3]).all()
    for r in (4, 5, 6, 7):
        assert torch.isnan(out.loss[r]) and torch.isnan(out.logprob[r]) and torch.isnan(out.grad[r]).all()
    # the same rows out by weight
    w = one.clone()
    w[3:] = 0.0
    out = L.policy_loss(z, y.cuda(), one * -1, one, weight=w)
    assert (out.loss[3:] == 0).all() and (out.grad[3:] == 0).all() and torch.isfinite(out.grad).all()


def test_lowest_value_masks(L):
    # a mask by the type's lowest finite value, not -inf
    for dtype in DTYPES.values():
        z, z64 = make_logits(4, 2000, dtype)
        low = torch.finfo(dtype).min
        z[:, 100:1900] = low
        z64[:, 100:1900] = low
        y = torch.tensor([0, 1999, 50, 1900])
        lp, lse = L.token_logprob(z, y.cuda())
        want_lp, want_lse = ref_logprob(z64, y, 1.0)
        close(lp, want_lp, lse_tol(2000) + U * want_lp.abs())
        z[2] = low  # nothing but the lowest value: uniform
        lp, lse = L.token_logprob(z, y.cuda())
        assert abs(float(lp[2]) + math.log(2000)) <= lse_tol(2000) + U * 8
        d = L.token_logprob_grad(z, y.cuda(), lse, torch.ones(4).cuda())
        assert (d[0, 100:1900] == 0).all() and torch.isfinite(d[:2]).all()
        share = torch.full((2000,), -1 / 2000, dtype=torch.float64)
        share[50] += 1
        close(d[2], share, share.abs() * (HALF[dtype] + 8 * U) + U)


def test_logits_in_the_hundreds(L):
    # lse in 32 bits is too coarse there: the gradient takes the row's own statistics
    for dtype in DTYPES.values():
        z, z64 = make_logits(3, 1500, dtype, scale=3000.0)
        z64[1, 7:700] = z64[1].max()  # many equal maxima
        z.copy_(z64)
        y = torch.tensor([4, 8, 1000])
        lp, lse = L.token_logprob(z, y.cuda(), temperature=2.0)
        want, _ = ref_logprob(z64, y, 2.0)
        close(lp, want, lse_tol(1500) + 2 * U * want.abs())
        d = L.token_logprob_grad(z, y.cuda(), lse, torch.ones(3).cuda(), temperature=2.0)
        one = torch.ones(3).double()
        check_grad(d, z64, y, one, 0 * one, 2.0, extra=lse_tol(1500))


def test_rows_far_apart(L):
    # element offsets past 32 bits
    stride, vocab = (1 << 31) + 8, 1000
    store = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    z = store.as_strided((3, vocab), (stride, 1))
    small, z64 = make_logits(3, vocab, torch.bfloat16)
    z.copy_(small)
    y = make_target(3, vocab)
    lp, lse = L.token_logprob(z, y.cuda())
    a, b = L.token_logprob(small, y.cuda())
    assert torch.equal(lp, a) and torch.equal(lse, b)
    g = torch.ones(3).cuda()
    want = L.token_logprob_grad(small, y.cuda(), lse, g)
    assert torch.equal(L.token_logprob_grad(z, y.cuda(), lse, g, out=z), want)


def test_rows_that_share_memory(L):
    z, _ = make_logits(1, 777, torch.float16)
    y = make_target(5, 777).cuda()
    lp, lse = L.token_logprob(z.expand(5, 777), y)
    a, b = L.token_logprob(z.repeat(5, 1), y)
    assert torch.equal(lp, a) and torch.equal(lse, b)
    with pytest.raises(Exception):
        L.token_logprob_grad(z.expand(5, 777), y, lse, lp, out=z.expand(5, 777))


# ------------------------------------------------------------------ preference

def ref_preference(lp, ref, offsets, beta, mask=None, weight=None, average=False, eps=0.0, margin=0.0):
    """Plain loops in 64 bits."""
    lp = lp.double()
    ref = torch.zeros_like(lp) if ref is None else ref.double()
    P = (len(offsets) - 1) // 2
    keep = torch.ones(len(lp), dtype=torch.bool) if mask is None else mask
    grad = torch.zeros_like(lp)
    loss, rewards = [], [[], []]
    for p in range(P):
        spans, scale = [], []
        for q in (p, P + p):
            idx = [t for t in range(offsets[q], offsets[q + 1]) if keep[t]]
            spans.append(idx)
            scale.append(beta / max(1, len(idx)) if average else beta)
        r = [sum(((float(lp[t]) - float(ref[t])) for t in idx), 0.0) * s for idx, s in zip(spans, scale)]
        u = r[0] - r[1] - margin
        soft = math.log1p(math.exp(-abs(u)))
        loss.append((1 - eps) * (soft + max(-u, 0)) + eps * (soft + max(u, 0)))
        slope = (1 / (1 + math.exp(-u)) if u > -700 else 0.0) - (1 - eps)
        w = 1.0 if weight is None else float(weight[p])
        for sign, idx, s in ((1, spans[0], scale[0]), (-1, spans[1], scale[1])):
            for t in idx:
                grad[t] = sign * slope * w * s
        rewards[0].append(r[0])
        rewards[1].append(r[1])
    return (torch.tensor(loss).double(), torch.tensor(rewards[0]).double(), torch.tensor(rewards[1]).double(), grad)


LENGTHS = {
    "ones": [1, 1], "zero": [0, 3, 2, 0], "both-empty": [0, 0], "short": [5, 1, 7, 64, 65, 63],
    "long": [1000, 257, 4099, 256], "many": [(i * 37) % 19 for i in range(200)], "uneven": [9001, 3],
}


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_preference_loss(L, lengths, average):
    n = LENGTHS[lengths]
    front, behind = 3, 5  # tokens of no sequence, before and behind
    offsets = [front]
    for k in n:
        offsets.append(offsets[-1] + k)
    T, P = offsets[-1] + behind, len(n) // 2
    g = gen(len(n) + T)
    lp = -torch.rand(T, generator=g) * 6
    ref = lp + 0.3 * torch.randn(T, generator=g)
    lp[:front] = ref[T - behind:] = float("nan")  # not read
    mask = torch.rand(T, generator=g) < 0.7
    mask[offsets[1]:offsets[2]] = False  # a sequence whose mask leaves nothing
    w = torch.rand(P, generator=g)
    for kw in (dict(), dict(mask=mask), dict(mask=mask, weight=w, eps=0.1, margin=0.5)):
        want = ref_preference(lp, ref, offsets, 0.3, average=average, **kw)
        spoiled = lp.clone()
        if "mask" in kw:
            spoiled[~mask] = float("nan")
        dev = {k: v.cuda() for k, v in kw.items() if k in ("mask", "weight")}
        got = L.preference_loss(spoiled.cuda(), ref.cuda(), torch.tensor(offsets).cuda(), beta=0.3, average=average,
                                label_smoothing=kw.get("eps", 0.0), margin=kw.get("margin", 0.0), **dev)
        for a, b in zip(got, want):
            close(a, b, 1.01 * U * b.abs() + 1e-9)  # 64-bit sums of up to 9,001 terms below 2^4: 1e-9 and far less
        quiet = L.preference_loss(spoiled.cuda(), ref.cuda(), torch.tensor(offsets).cuda(), beta=0.3, average=average,
                                  label_smoothing=kw.get("eps", 0.0), margin=kw.get("margin", 0.0), grad=False, **dev)
        assert quiet.grad is None and all(torch.equal(a, b) for a, b in zip(quiet[:3], got[:3]))


def test_preference_without_a_reference_and_far_apart(L):
    offsets = [0, 2, 4, 6, 8]
    lp = torch.tensor([0.0, -1.0, -2000.0, 0.0, -3000.0, 0.0, -1.0, 0.0])
    want = ref_preference(lp, None, offsets, 1.0)
    got = L.preference_loss(lp.cuda(), None, torch.tensor(offsets).cuda(), beta=1.0)
    for a, b in zip(got, want):
        close(a, b, 1.01 * U * b.abs() + 1e-30)
    assert got.loss[0] == 0 and got.loss[1] == 1999.0  # -log sigma far out on both sides, no overflow


def test_preference_bad_offsets_and_no_pairs(L):
    lp = torch.randn(10).cuda()
    for bad in ([0, 5, 3, 8, 10], [-1, 2, 4, 6, 8], [0, 2, 4, 6, 11], [0, 1 << 62, 4, 6, 8]):
        out = L.preference_loss(lp, None, torch.tensor(bad).cuda(), beta=0.1)
        torch.cuda.synchronize()
        assert torch.isnan(out.loss).any()
    out = L.preference_loss(lp, lp, torch.tensor([4]).cuda(), beta=0.1)
    assert out.loss.shape == (0,) and (out.grad == 0).all() and out.grad.shape == (10,)
    empty = torch.empty(0).cuda()
    out = L.preference_loss(empty, empty, torch.tensor([0, 0, 0]).cuda(), beta=0.1)
    assert out.grad.shape == (0,) and abs(float(out.loss[0]) - math.log(2)) < 1e-7


# ------------------------------------------------------------------------ head

HEAD_SHAPES = [(1, 1, 1), (1, 300, 64), (2, 129, 8), (3, 128, 72), (16, 1000, 256), (17, 513, 200), (33, 257, 33),
               (65, 1025, 129), (130, 300, 520), (129, 128, 31), (257, 700, 64), (5, 5003, 1024), (300, 391, 96), (16, 9000, 72),
               (64, 64, 320), (100, 1100, 1000), (90, 9001, 136), (7, 77, 1016)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,dim", HEAD_SHAPES)
def test_head_logprob(L, rows, vocab, dim, dtype):
    t = DTYPES[dtype]
    g = gen(rows + vocab)
    # whole numbers: the logits are exact in 32 bits (|z| <= 4 dim < 2^24)
    x = torch.randint(-2, 3, (rows, dim), generator=g).to(t)
    w = torch.randint(-2, 3, (vocab, dim), generator=g).to(t)
    y = make_target(rows, vocab, ignore=(1,))
    scale = 1.0 + math.sqrt(dim)  # a temperature that keeps the softmax wide
    z64 = x.double() @ w.double().t()
    lp, lse = L.head_logprob(x.cuda(), w.cuda(), y.cuda(), temperature=scale)
    want_lp, want_lse = ref_logprob(z64, y, scale)
    e = lse_tol(vocab) + U * 3 * 12  # more joins than a row's
    close(lse, want_lse, e + U * want_lse.abs())
    close(lp, want_lp, e + U * want_lp.abs())
    # real numbers, rows apart and at odd places
    xs = torch.randn(rows, dim + 3, generator=g).to(t)
    ws = (torch.randn(vocab, dim + 5, generator=g) / math.sqrt(dim)).to(t)
    lp, lse = L.head_logprob(xs.cuda()[:, 1:dim + 1], ws.cuda()[:, 3:dim + 3], y.int().cuda())
    x64, w64 = xs[:, 1:dim + 1].double(), ws[:, 3:dim + 3].double()
    want_lp, want_lse = ref_logprob(x64 @ w64.t(), y, 1.0)
    e = e + 2 * dim * U * float((x64.abs() @ w64.abs().t()).max())
    close(lse, want_lse, e + U * want_lse.abs())
    close(lp, want_lp, e + U * want_lp.abs())


def test_head_rows_out_and_nan(L):
    x, w = torch.randn(70, 128).bfloat16(), torch.randn(300, 128).bfloat16()
    y = make_target(70, 300)
    want_lp, want_lse = (t.clone() for t in L.head_logprob(x.cuda(), w.cuda(), y.cuda()))
    x[5] = float("nan")   # NaN in a row that takes no part does no harm to it or its neighbours
    x[40] = float("nan")  # in one that does: NaN there only
    y[5], y[41] = -1, 300
    lp, lse = L.head_logprob(x.cuda(), w.cuda(), y.cuda())
    assert lp[5] == 0 and lse[5] == 0 and torch.isnan(lp[40]) and torch.isnan(lse[40]) and torch.isnan(lp[41])
    keep = torch.ones(70, dtype=torch.bool)
    keep[[5, 40, 41]] = False
    assert torch.equal(lp[keep], want_lp[keep]) and torch.equal(lse[keep], want_lse[keep])
    w[7] = float("inf")
    lp, _ = L.head_logprob(x.cuda(), w.cuda(), y.cuda())
    assert torch.isnan(lp[keep]).all()


def test_head_shared_hidden_rows_and_no_rows(L):
    x, w = torch.randn(1, 64).half().cuda(), torch.randn(500, 64).half().cuda()
    y = make_target(6, 500).cuda()
    a = L.head_logprob(x.expand(6, 64), w, y)
    b = L.head_logprob(x.repeat(6, 1), w, y)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    lp, lse = L.head_logprob(x[:0], w, y[:0])
    assert lp.shape == (0,) and lse.shape == (0,)


# ------------------------------------------------------------- the set together

def chain64(z, y, ref, offsets, w, beta):
    """The preference objective from the logits, 64 bits."""
    lp, _ = ref_logprob(z, y, 1.0)
    P = len(w)
    keep = (y >= 0).double()
    delta = (lp - ref) * keep
    s = torch.stack([delta[a:b].sum() for a, b in zip(offsets, offsets[1:])]) * beta
    return (w * torch.nn.functional.softplus(-(s[:P] - s[P:]))).sum()


def test_preference_step_against_differences(L):
    """Logits to their gradient through three calls, against the formula's
    derivative and against differences of the 64-bit objective."""
    g = gen(11)
    n, V = [4, 3, 5, 6], 37
    offsets = [0, 4, 7, 12, 18]
    T = 18
    z = torch.randn(T, V, generator=g) * 2
    y = make_target(T, V, ignore=(0, 5))
    x, wt = torch.randn(T, 16, generator=g).bfloat16(), torch.randn(V, 16, generator=g).bfloat16()
    ref, _ = L.head_logprob(x.cuda(), wt.cuda(), y.cuda())  # the reference model's score
    w = torch.tensor([0.7, 0.4])
    zc, yc, off = z.cuda(), y.cuda(), torch.tensor(offsets).cuda()
    lp, lse = L.token_logprob(zc, yc)
    out = L.preference_loss(lp, ref, off, beta=0.5, weight=w.cuda())
    grad = L.token_logprob_grad(zc, yc, lse, out.grad).cpu().double()
    z64 = z.double().requires_grad_(True)
    obj = chain64(z64, y, ref.cpu().double(), offsets, w.double(), 0.5)
    obj.backward()
    got = float((w * out.loss.cpu()).sum())
    # 18 log-probabilities, each off by lse_tol and weighed by at most
    # beta max(w) |d loss / d u| < 0.35; as much again in the slopes of the gradient
    e = 18 * lse_tol(V) * 0.35
    assert abs(got - float(obj.detach())) <= e
    close(grad, z64.grad, e)
    h = 1e-5
    for t, j in ((1, int(y[1])), (1, 3), (6, 20), (9, int(y[9])), (17, 0), (0, 4), (5, 5)):
        up, down = z.double().clone(), z.double().clone()
        up[t, j] += h
        down[t, j] -= h
        slope = (chain64(up, y, ref.cpu().double(), offsets, w.double(), 0.5)
                 - chain64(down, y, ref.cpu().double(), offsets, w.double(), 0.5)) / (2 * h)
        assert abs(float(slope) - float(grad[t, j])) <= e + 1e-9  # h^2 / 6 and 1e-16 / h are below 1e-9


def test_policy_gradient_against_differences(L):
    g = gen(12)
    T, V, tau, klc = 9, 23, 0.9, 0.2
    z = torch.randn(T, V, generator=g) * 2
    y = make_target(T, V, ignore=(2,))
    lp64, _ = ref_logprob(z.double(), y, tau)
    old, ref, adv, w = policy_inputs(T, 13, lp64)
    out = L.policy_loss(z.cuda(), y.cuda(), old.cuda(), adv.cuda(), ref_logprob=ref.cuda(), weight=w.cuda(),
                        kl_coef=klc, temperature=tau, clip_low=0.2, clip_high=0.3)

    def objective(zz):
        lp, _ = ref_logprob(zz, y, tau)
        loss = ref_policy(lp, old, ref, adv, w, 0.2, 0.3, klc)[0]
        return float((loss * w.double() * (y >= 0)).sum())

    h = 1e-6
    for t in range(T):
        for j in (int(y[t].clamp(min=0)), (t * 5) % V):
            up, down = z.double().clone(), z.double().clone()
            up[t, j] += h
            down[t, j] -= h
            slope = (objective(up) - objective(down)) / (2 * h)
            # logprob's error in coef and in p, float32's rounding; h^2 / 6 and 1e-16 / h are below 1e-9
            assert abs(slope - float(out.grad[t, j])) <= 4 * lse_tol(V) * (1 + abs(slope)) + 1e-9


def test_other_stream_and_same_bits(L):
    z, _ = make_logits(33, 5003, torch.bfloat16)
    y = make_target(33, 5003, ignore=(3,)).cuda()
    old, adv = torch.full((33,), -9.0).cuda(), torch.randn(33, generator=gen(1)).cuda()
    x, w = torch.randn(33, 256, generator=gen(1)).bfloat16().cuda(), torch.randn(5003, 256, generator=gen(2)).bfloat16().cuda()

    def step():
        lp, lse = L.token_logprob(z, y)
        pol = L.policy_loss(z, y, old, adv, clip_low=0.2, clip_high=0.2)
        pre = L.preference_loss(lp, None, off, beta=0.1)
        d = L.token_logprob_grad(z, y, lse, pre.grad)
        return [lp, lse, *pol, *pre, d, *L.head_logprob(x, w, y)]

    off = torch.tensor([0, 10, 16, 20, 33]).cuda()
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured_and_replayed(L):
    """One graph of the whole set, replayed on new inputs with eager work and
    synchronisations in between; a second graph of the same calls lives
    beside it."""
    T, V, Dm = 40, 3001, 128
    z = torch.empty(T, V, dtype=torch.bfloat16, device="cuda")
    x, w = torch.empty(T, Dm, dtype=torch.bfloat16, device="cuda"), torch.empty(V, Dm, dtype=torch.bfloat16, device="cuda")
    y = torch.empty(T, dtype=torch.int64, device="cuda")
    off = torch.tensor([0, 9, 20, 31, 40]).cuda()
    adv = torch.randn(T, generator=gen(4)).cuda()

    def fill(seed):
        g = gen(seed)
        z.copy_(torch.randn(T, V, generator=g) * 2)
        x.copy_(torch.randn(T, Dm, generator=g))
        w.copy_(torch.randn(V, Dm, generator=g) / 11)
        y.copy_(make_target(T, V, seed, ignore=(seed % T,)))

    def step():
        ref, _ = L.head_logprob(x, w, y)
        lp, lse = L.token_logprob(z, y)
        pre = L.preference_loss(lp, ref, off, beta=0.1)
        d = L.token_logprob_grad(z, y, lse, pre.grad)
        pol = L.policy_loss(z, y, lp, adv, ref_logprob=ref, kl_coef=0.1)
        return [ref, lp, *pre, d, *pol]

    fill(0)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for seed in range(1, 5):
        fill(seed)
        want = [t.clone() for t in step()]
        for gr, out in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_refusals_on_the_gpu(L, dlr):
    z, y, v = torch.zeros(3, 5).cuda(), torch.zeros(3, dtype=torch.int64).cuda(), torch.zeros(3).cuda()
    off = torch.tensor([0, 1, 3]).cuda()
    bad = [
        lambda: L.token_logprob(z.double(), y), lambda: L.token_logprob(z[0], y), lambda: L.token_logprob(z.t(), y),
        lambda: L.token_logprob(z, y[:2]), lambda: L.token_logprob(z, y.float()), lambda: L.token_logprob(z, y.cpu()),
        lambda: L.token_logprob(z[:, :0], y), lambda: L.token_logprob(z, y, temperature=0.0),
        lambda: L.token_logprob_grad(z, y, v.double(), v), lambda: L.token_logprob_grad(z, y, v, v[:2]),
        lambda: L.token_logprob_grad(z, y, v, v, out=z.half()), lambda: L.token_logprob_grad(z, y, v, v, out=z[:2]),
        lambda: L.token_logprob_grad(z[:2], y[:2], v[:2], v[:2], out=z[1:]),
        lambda: L.policy_loss(z, y, v, v, kl_coef=0.1), lambda: L.policy_loss(z, y, v, v, clip_low=2.0),
        lambda: L.policy_loss(z, y, v, v, weight=v[:1]), lambda: L.policy_loss(z, y, v, v, grad=False, out=z),
        lambda: L.preference_loss(v, v, off, beta=0.0), lambda: L.preference_loss(v, v, off[:2], beta=0.1),
        lambda: L.preference_loss(v, v[:2], off, beta=0.1), lambda: L.preference_loss(v, v, off.int(), beta=0.1),
        lambda: L.preference_loss(v, v, off, beta=0.1, mask=v), lambda: L.preference_loss(z, v, off, beta=0.1),
        lambda: L.preference_loss(v, v, off, beta=0.1, weight=v),
        lambda: L.head_logprob(z, z, y), lambda: L.head_logprob(z.half(), z.bfloat16(), y),
        lambda: L.head_logprob(z.half(), z.half()[:, :4].contiguous(), y),
        lambda: L.head_logprob(z.half(), z.half().t(), y), lambda: L.head_logprob(z.half(), z.half(), y[:1]),
        lambda: L.head_logprob(z.half(), z.half(), y, temperature=-1.0),
    ]
    for call in bad:
        with pytest.raises(dlr.DLRError) as e:
            call()
        assert e.value.code == dlr.E_ARG
    lp, lse = L.token_logprob(z[:0], y[:0])
    assert lp.shape == (0,)
    assert L.token_logprob_grad(z[:0], y[:0], v[:0], v[:0]).shape == (0, 5)
    assert L.policy_loss(z[:0], y[:0], v[:0], v[:0]).grad.shape == (0, 5)


@pytest.mark.parametrize("out", ["none", "half", "all", "all but the last", "all but the first 130"])
def test_head_long_calls_leave_out_the_rows_that_take_no_part(L, out):
    # from rows * vocab * dim = 6.4e10 on the rows that take part are picked first
    rows, vocab, dim = 700, 50001, 2048
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randint(-2, 3, (rows, dim), generator=g, device="cuda").bfloat16()
    w = torch.randint(-2, 3, (vocab, dim), generator=g, device="cuda").bfloat16()
    y = make_target(rows, vocab)
    keep = torch.ones(rows, dtype=torch.bool)
    if out == "half":
        keep = torch.rand(rows, generator=gen(4)) < 0.5
    elif out != "none":
        keep[:] = False
        keep[-1] = out == "all but the last"
        keep[:130] = out == "all but the first 130"
    y[~keep] = -7
    x[~keep.cuda()] = float("nan")
    scale = 60.0
    lp, lse = L.head_logprob(x, w, y.cuda(), temperature=scale)
    z = torch.mm(torch.nan_to_num(x).double(), w.double().t()).cpu()  # whole numbers: exact
    want_lp, want_lse = ref_logprob(z, y, scale)
    e = lse_tol(vocab) + U * 3 * 12
    close(lse, want_lse, torch.where(keep, e + U * want_lse.abs(), 0.0))
    close(lp, want_lp, torch.where(keep, e + U * want_lp.abs(), 0.0))


def test_captured_with_picked_rows(L):
    """A captured long call, its rows picked on the device: the mask changes
    between replays."""
    rows, vocab, dim = 640, 50001, 2048
    x = torch.randn(rows, dim, generator=gen(1)).bfloat16().cuda()
    w = (torch.randn(vocab, dim, generator=gen(2)) / 18).bfloat16().cuda()
    y = make_target(rows, vocab).cuda()
    L.head_logprob(x, w, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = L.head_logprob(x, w, y)
    for seed in range(4):
        new = make_target(rows, vocab, seed + 5)
        new[torch.rand(rows, generator=gen(seed)) < 0.3 * seed] = -1
        y.copy_(new)
        want = [t.clone() for t in L.head_logprob(x, w, y)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_class_of_probability_zero(L):
    # the given class is masked out for the policy: the KL estimate is inf, not NaN
    z, _ = make_logits(3, 50, torch.float32)
    y = torch.tensor([4, 5, 6]).cuda()
    z[1, 5] = float("-inf")
    v = torch.full((3,), -2.0).cuda()
    out = L.policy_loss(z, y, v, torch.ones(3).cuda(), ref_logprob=v, kl_coef=0.1)
    assert out.kl[1] == float("inf") and out.loss[1] == float("inf") and out.logprob[1] == float("-inf")
    assert torch.isfinite(out.grad[[0, 2]]).all() and torch.isfinite(out.kl[[0, 2]]).all()
    quiet = L.policy_loss(z, y, v, torch.ones(3).cuda(), ref_logprob=v)  # reported, but no term of the loss
    assert quiet.kl[1] == float("inf") and quiet.loss[1] == 0 and torch.isfinite(quiet.grad).all()


def test_the_current_device_and_the_last_error_stay(L, dlr):
    z, y = torch.zeros(3, 5).cuda(), torch.zeros(3, dtype=torch.int64).cuda()
    x = L._logits(z, y, 1.0)[2]
    import ctypes
    assert L.lib.dlr_token_logprob(99, None, ctypes.byref(x), None, 0, z.data_ptr(), z.data_ptr()) == -4
    assert torch.cuda.current_device() == 0
    torch.cuda.synchronize()  # the failed call's error is not reported again
    lp, _ = L.token_logprob(z, y)
    assert abs(float(lp[0]) + math.log(5)) < 1e-6


def test_targets_of_32_bits_and_strided_vectors(L):
    z, _ = make_logits(11, 300, torch.bfloat16)
    x, w = torch.randn(11, 64).bfloat16().cuda(), torch.randn(300, 64).bfloat16().cuda()
    y = make_target(11, 300, ignore=(2,)).cuda()
    v = torch.randn(5, 11, generator=gen(3)).cuda()

    def calls(y, v):
        lp, lse = L.token_logprob(z, y)
        g = L.token_logprob_grad(z, y, lse, v[0])
        p = L.policy_loss(z, y, v[1] - 6, v[2], ref_logprob=v[3] - 6, weight=v[4], kl_coef=0.1)
        q = L.preference_loss(v[0], v[1], torch.tensor([0, 3, 5, 7, 11]).cuda(), beta=0.1, weight=v[2][:2])
        return [lp, lse, g, *p, *q, *L.head_logprob(x, w, y)]

    apart = v.t().contiguous().t()  # the same vectors, 5 elements apart
    assert not apart[0].is_contiguous()
    wide = torch.stack([y, y], 1)[:, 0]
    for other in (calls(y.int(), v), calls(y, apart), calls(wide, v)):
        for a, b in zip(calls(y, v), other):
            assert torch.equal(a, b)


def test_many_short_rows_and_pairs(L):
    rows = 70003
    z, z64 = make_logits(rows, 5, torch.float32)
    y = make_target(rows, 5)
    lp, _ = L.token_logprob(z, y.cuda())
    want, _ = ref_logprob(z64, y, 1.0)
    close(lp, want, lse_tol(5) + U * want.abs())
    out = L.policy_loss(z, y.cuda(), lp, torch.ones(rows).cuda())
    close(out.loss, torch.full((rows,), -1.0).double(), torch.tensor(2 * lse_tol(5) + 4 * U).double())  # ratio 1
    P = 70001
    l = torch.randn(2 * P, generator=gen(1))
    got = L.preference_loss(l.cuda(), None, torch.arange(2 * P + 1).cuda(), beta=1.0)
    u = l[:P].double() - l[P:].double()
    want = torch.nn.functional.softplus(-u)
    close(got.loss, want, 1.01 * U * want + 1e-12)
    slope = torch.sigmoid(u) - 1
    close(got.grad, torch.cat([slope, -slope]), 1.01 * U * slope.abs().repeat(2) + 1e-12)


def test_two_calls_at_once(L):
    """On two streams, each with its own scratch memory."""
    args = []
    for seed in (1, 2):
        x = torch.randn(200, 512, generator=gen(seed)).bfloat16().cuda()
        w = (torch.randn(20011, 512, generator=gen(seed + 5)) / 9).bfloat16().cuda()
        args.append((x, w, make_target(200, 20011, seed).cuda()))
    want = [[t.clone() for t in L.head_logprob(*a)] for a in args]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(L.head_logprob(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for out in got[i] for a, b in zip(out, want[i]))


@pytest.mark.parametrize("rows,vocab,dim", [(333, 50257, 512), (600, 30001, 512), (700, 50257, 512)])
def test_head_tiles_of_two_kinds(L, rows, vocab, dim):
    # whole rounds of large tiles, the other classes by smaller ones; targets on both sides of the seam
    g = gen(rows)
    x = torch.randint(-2, 3, (rows, dim), generator=g).half()
    w = torch.randint(-2, 3, (vocab, dim), generator=g).half()
    y = make_target(rows, vocab, ignore=(7,))
    y[0], y[1] = 0, vocab - 1
    scale = 3 * math.sqrt(dim)
    lp, lse = L.head_logprob(x.cuda(), w.cuda(), y.cuda(), temperature=scale)
    want_lp, want_lse = ref_logprob((x.cuda().double() @ w.cuda().double().t()).cpu(), y, scale)
    e = lse_tol(vocab) + U * 3 * 12
    close(lse, want_lse, e + U * want_lse.abs())
    close(lp, want_lp, e + U * want_lp.abs())


def test_autograd_notices_a_gradient_written_over_the_logits(L):
    z = torch.randn(4, 9, device="cuda", requires_grad=True)
    h = z * 2.0
    loss = (h * h).sum()  # saves h
    y = make_target(4, 9).cuda()
    lp, lse = L.token_logprob(h, y)
    assert not lp.requires_grad
    L.token_logprob_grad(h.detach(), y, lse, torch.ones(4).cuda(), out=h.detach())
    with pytest.raises(RuntimeError):
        loss.backward()


def test_preference_with_an_impossible_sequence(L):
    # a token of probability 0 in the sequence that is not preferred: u = inf, loss 0, nothing flows back
    inf = float("inf")
    off = torch.tensor([0, 2, 4]).cuda()
    worse = torch.tensor([-1.0, -2.0, -inf, -1.0]).cuda()
    out = L.preference_loss(worse, None, off, beta=0.5)
    assert out.loss[0] == 0 and out.rejected_reward[0] == -inf and (out.grad == 0).all()
    out = L.preference_loss(-worse.flip(0) * -1, None, off, beta=0.5)  # in the preferred one: loss inf, slope -1
    assert out.loss[0] == inf and torch.equal(out.grad.cpu(), torch.tensor([-0.5, -0.5, 0.5, 0.5]))
    out = L.preference_loss(worse, None, off, beta=0.5, label_smoothing=0.1)
    assert out.loss[0] == inf
    out = L.preference_loss(worse, None, off, beta=0.5, label_smoothing=1.0)  # all weight on the other side
    assert out.loss[0] == inf


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [8192, 16388, 32776, 65543, 69632, 69647, 131075])
def test_long_rows_of_many(L, vocab, dtype):
    # more rows than go by chunks, on both sides of what a workgroup holds of a row
    rows, tau, lo, hi, klc = 131, 0.8, 0.2, 0.3, 0.05
    z, z64 = make_logits(rows, vocab, DTYPES[dtype], 1)
    y = make_target(rows, vocab, ignore=(1,))
    y[0], y[2], y[3] = vocab - 1, 0, min(vocab - 1, 69632)
    edit = torch.zeros(4, vocab)
    edit[2, vocab // 2:] = -math.inf  # nothing left in the second half
    edit[3, :] = -math.inf            # nothing but the given class
    edit[3, y[3]] = 0.0
    z[:4] += edit.to(z.dtype).cuda()
    pick = torch.tensor([0, 1, 2, 3, 64, 129, 130])
    z64 = z64[pick]
    z64[:4] += edit.double()
    some = y[pick]
    lp, lse = ref_logprob(z64, some, tau)
    e = lse_tol(vocab)
    got_lp, got_lse = L.token_logprob(z, y.cuda(), temperature=tau)
    close(got_lp[pick], lp, e + U * lp.abs())
    close(got_lse[pick], lse, e + U * lse.abs())
    old, ref, adv, w = policy_inputs(rows, 3, torch.full((rows,), -5.0, dtype=torch.float64))
    old[pick], ref[pick] = (lp + 0.2).float(), (lp - 0.3).float()
    used = (some >= 0) & (w[pick] != 0)
    loss, kl, clipped, coef, size = ref_policy(lp, old[pick], ref[pick], adv[pick], w[pick], lo, hi, klc)
    args = (y.cuda(), old.cuda(), adv.cuda())
    more = dict(ref_logprob=ref.cuda(), weight=w.cuda(), clip_low=lo, clip_high=hi, kl_coef=klc, temperature=tau)
    out = L.policy_loss(z, *args, **more)
    zero = torch.zeros_like(lp)
    close(out.logprob[pick], torch.where(used, lp, zero), e + U * lp.abs())
    close(out.loss[pick], torch.where(used, loss, zero), 2 * e * size + 2 * U * loss.abs() + 2 * U * kl)
    assert torch.equal(out.clipped.cpu()[pick], clipped & used)
    check_grad(out.grad[pick], z64, some, torch.where(used, coef, zero),
               w[pick].double() * (2 * e * size) + 2 * U * coef.abs(), tau, extra=e)
    same = L.policy_loss(z, *args, **more, out=z)
    assert same.grad is z and torch.equal(z, out.grad) and torch.equal(same.loss, out.loss)


def test_preference_bad_offsets_write_every_gradient(L):
    import ctypes
    inf = float("inf")
    for bad, want in (([-1, 2, 4, 6, 8], "nnggnngg00"), ([0, 2, 4, 6, 11], "ggnnggnnnn"),
                      ([0, 1 << 62, 4, 6, 8], "nnnnnnnn??"), ([3, 4, 5, 6, 20], "000gngnnnn")):
        lp, off = torch.randn(10).cuda(), torch.tensor(bad).cuda()
        out = torch.full((3, 2), inf).cuda()
        grad = torch.full((10,), inf).cuda()
        p = L._Preference(lp.data_ptr(), None, None, off.data_ptr(), None, 2, 10, 0.1, 0.0, 0.0, 0, 0)
        L._check(L.lib.dlr_preference_loss(0, L._stream(0), ctypes.byref(p), *(o.data_ptr() for o in out),
                                           grad.data_ptr()))
        g = grad.cpu()
        for token, kind in enumerate(want):
            v = float(g[token])
            assert {"n": math.isnan(v), "g": 0 < abs(v) < 0.1, "0": v == 0, "?": v != inf}[kind], (bad, token, v)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_rows_than_one_launch(L, dtype):
    # from 2^21 rows on a call is several launches; a row's results depend on the row alone
    rows, vocab, many = 1000, 9, (1 << 21) + 5
    times = many // rows + 1
    z, z64 = make_logits(rows, vocab, DTYPES[dtype])
    y = make_target(rows, vocab, ignore=(1,))
    lp, lse = L.token_logprob(z, y.cuda())
    want = ref_logprob(z64, y, 1.0)[0]
    close(lp, want, lse_tol(vocab) + U * want.abs())
    g = torch.randn(rows, generator=gen(5)).cuda()
    old, ref, adv, w = (t.cuda() for t in policy_inputs(rows, 3, want))

    def over(t):
        return t.repeat(times, *[1] * (t.dim() - 1))[:many]

    def all_of(z, y, lse, g, old, ref, adv, w):
        yield from L.token_logprob(z, y)
        yield L.token_logprob_grad(z, y, lse, g)
        yield from L.policy_loss(z, y, old, adv, ref_logprob=ref, weight=w, kl_coef=0.1)

    few = (z, y.cuda(), lse, g, old, ref, adv, w)
    for got, want in zip(all_of(*(over(t) for t in few)), all_of(*few)):
        assert torch.equal(got, over(want))
    yy = over(y.cuda())
    zz = over(z).contiguous()
    want = L.token_logprob_grad(z, y.cuda(), lse, g)
    assert torch.equal(L.token_logprob_grad(zz, yy, over(lse), over(g), out=zz), over(want))
    if dtype == "bf16":
        hidden = torch.randn(rows, 16, generator=gen(8)).bfloat16().cuda()
        head = torch.randn(vocab, 16, generator=gen(9)).bfloat16().cuda()
        e = 2 * (lse_tol(vocab) + U * 36 + 32 * U * float((hidden.double().abs() @ head.double().abs().t()).max()))
        for got, want in zip(L.head_logprob(over(hidden), head, yy), L.head_logprob(hidden, head, y.cuda())):
            close(got, over(want).cpu().double(), (e + 2 * U * over(want).abs()).cpu().double())


def test_head_of_more_logits_than_one_launch(L):
    # from 2^35 logits on a call is several runs of launches over one workspace
    rows, vocab, dim, scale = 8292, (1 << 22) + 77, 8, 4.0
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randint(-2, 3, (rows, dim), generator=g, device="cuda").bfloat16()
    w = torch.randint(-2, 3, (vocab, dim), generator=g, device="cuda").bfloat16()
    y = make_target(rows, vocab)
    y[torch.rand(rows, generator=gen(4)) < 0.5] = -1
    pick = torch.tensor([0, 1, 2, 4145, 4146, 4147, 8290, 8291])
    y[pick] = make_target(8, vocab, seed=9)
    lp, lse = L.head_logprob(x, w, y.cuda(), temperature=scale)
    z = torch.mm(x[pick.cuda()].double(), w.double().t()).cpu()  # whole numbers: exact
    want_lp, want_lse = ref_logprob(z, y[pick], scale)
    e = lse_tol(vocab) + U * 3 * 12
    close(lse[pick], want_lse, e + U * want_lse.abs())
    close(lp[pick], want_lp, e + U * want_lp.abs())
    out = (y < 0).cuda()
    assert (lp[out] == 0).all() and (lse[out] == 0).all() and (lse[~out] > 0).all() and (lp[~out] < 0).all()
