"""The gradient's tensor, given by the caller."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_losses import DTYPES, L, dlr, gen, make_target  # noqa: E402,F401  (L, dlr: fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", [(7, 1000), (300, 20001), (2, 70001)])
def test_a_gradient_beside_the_logits(L, dtype, rows, vocab):  # noqa: F811
    # logits and gradient are columns of one buffer
    both = (torch.randn(rows, 2 * vocab + 3, generator=gen(1)) * 2.5).to(DTYPES[dtype]).cuda()
    z, out, rest = both[:, :vocab], both[:, vocab:2 * vocab], both[:, 2 * vocab:].clone()
    keep = z.clone()
    y = make_target(rows, vocab, ignore=(1,)).cuda()
    lp, lse = L.token_logprob(z, y)
    g = torch.randn(rows, generator=gen(2)).cuda()
    want = L.token_logprob_grad(keep, y, lse, g)
    assert L.token_logprob_grad(z, y, lse, g, out=out) is out
    assert torch.equal(out, want) and torch.equal(z, keep) and torch.equal(both[:, 2 * vocab:], rest)
    want = L.policy_loss(keep, y, lp, g, weight=g)
    got = L.policy_loss(z, y, lp, g, weight=g, out=out)
    assert torch.equal(out, want.grad) and torch.equal(got.loss, want.loss)
    assert torch.equal(z, keep) and torch.equal(both[:, 2 * vocab:], rest)


def test_a_refused_call_leaves_the_tensors_version(L, dlr):  # noqa: F811
    z = torch.randn(6, 40, device="cuda")
    y, v = make_target(4, 40).cuda(), torch.zeros(4, device="cuda")
    calls = [lambda out, **kw: L.token_logprob_grad(z[:4], y, v, v, out=out, **kw),
             lambda out, **kw: L.policy_loss(z[:4], y, v, v, out=out, **kw)]
    for call in calls:
        for bad, kw in ((z[1:5], {}), (torch.empty(4, 40, device="cuda"), dict(temperature=0.0))):
            before = bad._version
            with pytest.raises(dlr.DLRError):
                call(bad, **kw)
            assert bad._version == before
        out = torch.empty(4, 40, device="cuda")
        before = out._version
        call(out)
        assert out._version == before + 1
