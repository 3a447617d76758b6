"""Routing where rounded values cannot tell what exact arithmetic chooses. Inputs are solved for in 64 bits so that two values that matter lie
within some 1e-5 of each other; the choice must be that of 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def group():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from nccl_b200 import Communicator, get_unique_id
    from nccl_b200.ops.ep import ExpertParallel
    torch.cuda.set_device(0)
    c, made = Communicator(1, 0, get_unique_id()), {}

    def get(experts):
        if experts not in made:
            made[experts] = ExpertParallel(c, min(experts, 256), 1, 128)   # as many as one rank serves
            made[experts].E = experts   # more of them are routed to in groups of more ranks
        return made[experts]

    yield get
    assert c.async_error() == 0
    for ep in made.values():
        ep.destroy()
    c.destroy()


def scores(l, score):
    return 1 / (1 + torch.exp(-l)) if score == "sigmoid" else torch.softmax(l, 1)


def group_sums(l, bias, score, groups, top2):
    v = (scores(l, score) + bias).view(l.shape[0], groups, -1)
    best = v.topk(min(2, v.shape[2]), dim=2).values
    return best.sum(2) if top2 else best[..., 0]


def best(v, n):
    return torch.sort(v, dim=1, descending=True, stable=True).indices[:, :n]


def chosen(l, bias, score, groups, keep, top2, topk):
    """Ids in 64 bits, equal values by index."""
    rank = scores(l, score) + bias
    T, E = l.shape
    if groups > 1:
        kept = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, best(group_sums(l, bias, score, groups, top2), keep), True)
        rank = torch.where(kept[..., None].expand(T, groups, E // groups).reshape(T, E), rank, -math.inf)
    return best(rank, topk)


def solve(l, at, difference, lo, hi):
    """Logits with column `at` moved so that the increasing difference(l) is zero, as fp32 holds them."""
    lo, hi = torch.full((l.shape[0],), lo, dtype=torch.float64), torch.full((l.shape[0],), hi, dtype=torch.float64)
    for _ in range(80):
        l[:, at] = (lo + hi) / 2
        up = difference(l) > 0
        hi, lo = torch.where(up, l[:, at], hi), torch.where(up, lo, l[:, at])
    return l.float()


def same(ep, logits, bias, want, topk, **rule):
    idx, w = ep.route(logits.float().cuda(), topk, bias=bias.float().cuda(), **rule)
    far = (idx.cpu() != want).any(1)
    assert not far.any(), "%d of %d tokens, the first %d: %s, not %s" % (int(far.sum()), far.numel(), int(far.nonzero()[0]), idx[far.cuda()][0].tolist(), want[far][0].tolist())
    assert torch.isfinite(w).all()


def test_sums_of_two_that_cancel(group):
    """0.80447046 and 0.80447167 exactly; fp32 makes 0.80447006 and 0.80446625 of them."""
    logits = torch.tensor([[-0.1875, -0.625, 2.4375, -0.125]])
    bias = torch.tensor([64.00180053710938, -63.999237060546875, 63.997711181640625, -64.58167266845703])
    same(group(4), logits, bias, torch.tensor([[2, 3]]), 2, score="sigmoid", groups=2, keep_groups=1, group_score="top2")


# experts and groups: a lane holds one expert of two groups, two of 32, 16 of 32, 60 of 17, 16 of three
@pytest.mark.parametrize("E,groups", [(4, 2), (64, 32), (512, 32), (1020, 17), (384, 3)])
@pytest.mark.parametrize("size", [1.0, 64.0, 1000.0])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("top2", [True, False])
def test_groups_next_to_each_other(group, E, groups, size, score, top2):
    """Groups 0 and 1 lie within 1e-5 of each other, the others behind. Two experts of a group count, with biases of either sign."""
    T, per = 600, E // groups
    g = torch.Generator().manual_seed(E + int(size))
    logits = torch.randn(T, E, generator=g).float().double()
    if score == "softmax":
        logits[:, 2:per] -= 6      # so that the leaders have shares that logits can move
        logits[:, per + 2:] -= 6
    bias = -torch.rand(E, generator=g) - 3 * size - 10
    for k in range(groups):
        first = size * (0.5 + torch.rand(1, generator=g).item()) * (1 if k % 2 == 0 or size == 1 else -1)
        bias[k * per], bias[k * per + 1] = first - (4.0 if k > 1 else 0.0), 0.01 * torch.randn(1, generator=g).item() - first
        if not top2:
            bias[k * per], bias[k * per + 1] = size + 0.01 * k - (4.0 if k > 1 else 0.0), -size
    bias = bias.float().double()
    delta = 1e-5 * (2 * torch.rand(T, generator=g).double() - 1)

    def difference(l):
        s = group_sums(l, bias, score, groups, top2)
        return s[:, 1] - s[:, 0] - delta

    logits = solve(logits, per, difference, -30.0, 30.0).double()
    s = group_sums(logits, bias, score, groups, top2)
    assert ((s[:, 0] - s[:, 1]).abs() < 2e-5).sum() > T // 3 and (s[:, :2].amin(1) > (s[:, 2:].amax(1) if groups > 2 else -math.inf)).all()
    topk = 2 if per > 1 else 1
    want = chosen(logits, bias, score, groups, 1, top2, topk)
    same(group(E), logits, bias, want, topk, score=score, groups=groups, keep_groups=1, group_score="top2" if top2 else "max")


def test_sums_beyond_fp32(group):
    """Two groups whose sums fp32 has no numbers for, above and below; a group without experts is behind both, however low they are."""
    ep = group(4)
    logits = torch.zeros(2, 4)
    rule = dict(score="sigmoid", groups=2, keep_groups=1, group_score="top2")
    same(ep, logits, torch.tensor([3.0e38, 2.0e38, 3.1e38, 3.0e38]), torch.tensor([[2, 3]] * 2), 2, **rule)
    same(ep, logits, torch.tensor([3.1e38, 3.0e38, 3.0e38, 2.0e38]), torch.tensor([[0, 1]] * 2), 2, **rule)
    same(ep, logits, torch.tensor([-3.1e38, -3.0e38, -3.0e38, -2.0e38]), torch.tensor([[3, 2]] * 2), 2, **rule)
    logits[0, :2] = -math.inf      # token 0 has no expert in group 0, token 1 none at all
    logits[1] = -math.inf
    same(ep, logits, torch.tensor([-3.1e38, -3.0e38, -3.0e38, -2.0e38]), torch.tensor([[3, 2], [-1, -1]]), 2, **rule)
    same(ep, logits, torch.tensor([1.0, 1.0, -3.0e38, -2.0e38]), torch.tensor([[3, 2], [-1, -1]]), 2, **rule)


@pytest.mark.parametrize("E,groups,keep", [(1020, 17, 16), (1020, 1, 1), (240, 1, 1), (32, 1, 1)])
def test_shares_of_many_experts(group, E, groups, keep):
    """One large share and many that fp32 loses one by one beside it: the large one's rank value is next to another's."""
    T = 800
    g = torch.Generator().manual_seed(E)
    logits = torch.full((T, E), -16.7, dtype=torch.float64)
    bias = (-0.5 - torch.arange(E) // (E // groups) / 128).double()   # groups and experts further apart than what is looked at
    bias[0], bias[E - 1] = 0.0, float(torch.tensor(1 - 5.6e-8 * E, dtype=torch.float32))
    delta = 4e-6 * (2 * torch.rand(T, generator=g).double() - 1)

    def difference(l):
        v = torch.softmax(l, 1) + bias
        return v[:, 0] - v[:, E - 1] - delta

    # (the share itself moves by no more than 1: where that does not reach, the two are as near as it gets)
    logits = solve(logits, 0, difference, -3.0, 3.0).double()
    want = chosen(logits, bias, "softmax", groups, keep, False, 3)[:, :2]
    idx, _ = group(E).route(logits.float().cuda(), 2, score="softmax", bias=bias.float().cuda(), groups=groups, keep_groups=keep)
    v = torch.softmax(logits, 1) + bias
    apart = (v[:, 0] - v[:, E - 1]).abs()
    assert ((apart < 1e-5) & (apart > 0)).sum() > T // 2
    far = (idx.cpu() != want).any(1)
    assert not far.any(), (int(far.sum()), float(apart[far].max()))
