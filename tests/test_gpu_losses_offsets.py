"""preference_loss where the offsets descend (sequences would overlap) or leave
the tokens: the same answer on every call."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_losses import U, L, gen  # noqa: E402,F401  (L: the fixture)

pytestmark = pytest.mark.gpu


def all_nan(out):
    return all(bool(torch.isnan(t).all()) for t in out if t is not None)


@pytest.mark.parametrize("bad", [[0, 5, 3, 8, 10], [5, 2, 9], [0, 4, 3], [9, 10, 0], [0, 3, 6, 9, 8], [0, 0, 10, 9, 10],
                                 [2, 1, 1], [4, 6, 0, 10, 10], [1 << 62, 0, 10], [0, 10, -(1 << 62)]], ids=str)
@pytest.mark.parametrize("weighted", [False, True])
def test_descending_offsets_leave_nothing(L, bad, weighted):  # noqa: F811
    lp = torch.randn(10, generator=gen(1)).cuda()
    offsets = torch.tensor(bad).cuda()
    weight = torch.zeros(len(bad) // 2).cuda() if weighted else None
    out = L.preference_loss(lp, None, offsets, beta=0.1, weight=weight)
    assert all_nan(out)
    out = L.preference_loss(lp, None, offsets, beta=0.1, weight=weight, grad=False)
    assert all_nan(out) and out.grad is None


def packed(pairs, tokens, seed, before=0, behind=0):
    """Ascending offsets of 2 * pairs sequences, some of them empty."""
    cut = torch.randint(before, tokens - behind + 1, (2 * pairs + 1,), generator=gen(seed)).sort().values
    cut[0], cut[-1] = before, tokens - behind
    return cut


# up to 2,048 pairs each workgroup looks at the offsets, beyond a second launch does
PAIRS = [1, 2, 700, 2048, 2049, 5000, 40000]


@pytest.mark.parametrize("pairs", PAIRS)
def test_one_descent_anywhere(L, pairs):  # noqa: F811
    tokens = 3 * pairs + 40
    lp = torch.randn(tokens, generator=gen(2)).cuda()
    good = packed(pairs, tokens, 3)
    for at in {0, 1, pairs - 1, pairs, 2 * pairs - 1, int(torch.randint(0, 2 * pairs, (1,), generator=gen(4)))}:
        bad = good.clone()
        if bad[at] < tokens:
            bad[:at] = bad[:at].clamp(max=tokens - 1)
            bad[at] = tokens  # above the next one, unless every later one is the end
        if bool((bad[1:] >= bad[:-1]).all()):
            bad[at + 1] = bad[at] - 1
        out = L.preference_loss(lp, None, bad.cuda(), beta=0.1)
        assert all_nan(out), at


@pytest.mark.parametrize("pairs", PAIRS)
def test_ascending_offsets_of_many_pairs(L, pairs):  # noqa: F811
    tokens = 3 * pairs + 40
    lp, ref = (torch.randn(tokens, generator=gen(s)).cuda() for s in (5, 6))
    mask = (torch.rand(tokens, generator=gen(7)) < 0.7).cuda()
    for before, behind in ((0, 0), (7, 5)):
        offsets = packed(pairs, tokens, 8, before, behind).cuda()
        out = L.preference_loss(lp, ref, offsets, beta=0.5, mask=mask)
        delta = torch.where(mask, lp.double() - ref.double(), 0.0)
        n = offsets[1:] - offsets[:-1]
        owner = torch.repeat_interleave(torch.arange(2 * pairs, device="cuda"), n)
        inner = delta[before:tokens - behind]
        reward = torch.zeros(2 * pairs, dtype=torch.float64, device="cuda").index_add_(0, owner, inner) * 0.5
        u = reward[:pairs] - reward[pairs:]
        loss = torch.nn.functional.softplus(-u)
        slope = -torch.sigmoid(-u) * 0.5
        want = torch.zeros(tokens, dtype=torch.float64, device="cuda")
        want[before:tokens - behind] = torch.cat([slope, -slope])[owner] * mask[before:tokens - behind]
        # 64 bits and one rounding; sums in another order, 1e-12
        for got, exact in ((out.loss, loss), (out.chosen_reward, reward[:pairs]), (out.rejected_reward, reward[pairs:]),
                           (out.grad, want)):
            assert bool(((got.double() - exact).abs() <= 1.01 * U * exact.abs() + 1e-12).all())
        again = L.preference_loss(lp, ref, offsets, beta=0.5, mask=mask)
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_ascending_offsets_outside_the_tokens(L):  # noqa: F811
    # a pair with a sequence that leaves the tokens is NaN, the others are not; tokens of no sequence are 0
    lp = torch.randn(10, generator=gen(9)).cuda()
    for offsets, kinds in (([20, 30, 40], "0" * 10), ([-5, -3, -1], "0" * 10), ([-5, 3, 4], "nnnn000000"),
                           ([0, 3, 12], "n" * 10), ([1, 2, 3, 4, 5], "0gggg00000"),
                           # [-4, -2) is pair 0's and [-2, 3) pair 1's: both are NaN
                           ([-4, -2, 3, 5, 7], "nnnnnnn000")):
        out = L.preference_loss(lp, None, torch.tensor(offsets).cuda(), beta=0.1)
        for g, kind in zip(out.grad.tolist(), kinds):
            assert {"n": g != g, "0": g == 0, "g": 0 < abs(g) < 0.1}[kind], (offsets, out.grad)


@pytest.mark.parametrize("pairs", [5, 3000])
def test_captured_offsets_change_between_replays(L, pairs):  # noqa: F811
    # ascending, descending and ascending offsets through one graph, with eager work in between
    tokens = 3 * pairs + 40
    lp = torch.randn(tokens, generator=gen(10)).cuda()
    offsets = packed(pairs, tokens, 11).cuda()
    L.preference_loss(lp, None, offsets, beta=0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = L.preference_loss(lp, None, offsets, beta=0.1)
    for seed in range(6):
        new = packed(pairs, tokens, 20 + seed, seed % 3, seed % 2)
        if seed % 2:
            new[pairs] = tokens + 1 - new[pairs - 1]  # another place
            new[pairs + 1] = new[pairs] - 1
        offsets.copy_(new)
        want = [t.clone() for t in L.preference_loss(lp, None, offsets, beta=0.1)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(out, want)), seed
        assert all_nan(out) == bool(seed % 2)
