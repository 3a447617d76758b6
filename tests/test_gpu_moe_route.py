"""Routing to experts against the formulas in 64 bits: choice and order exactly, weights and gradients to the rounding of fp32 (and of the
logits' type)."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24   # half a unit in the last place of fp32
HALF = {torch.float32: U32, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


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


def best_first(v):
    return torch.sort(v, dim=-1, descending=True, stable=True)


def reference(logits, topk, score, bias=None, groups=1, keep_groups=None, group_score="max", renormalize=True, scale=1.0):
    """(idx, weights, scores) in 64 bits on the CPU."""
    l = logits.cpu().double()
    l = torch.where(torch.isnan(l), -math.inf, l).clamp_max(torch.finfo(torch.float32).max)
    T, E = l.shape
    there = l > -math.inf
    if score == "sigmoid":
        s = 1 / (1 + torch.exp(-l))
    else:
        p = torch.where(there, torch.exp(l - torch.where(there, l, -1e300).amax(1, keepdim=True)), 0.0)
        s = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    v = (s if bias is None else s + bias.cpu().double())
    v = torch.where(there & ~torch.isnan(v), v, -math.inf)
    # without a bias the logits are the order (scores that 64 bits cannot tell apart included)
    rank = torch.where(v > -math.inf, l, -math.inf) if bias is None else v
    if groups > 1:
        best = best_first(v.view(T, groups, -1)).values
        of = best[..., 0].clone() if group_score == "top2" or bias is not None else best_first(rank.view(T, groups, -1)).values[..., 0]
        if group_score == "top2" and E // groups > 1:
            of = of + torch.where(best[..., 1] > -math.inf, best[..., 1], 0.0)
        kept = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, best_first(of).indices[:, :keep_groups or groups], True)
        rank = torch.where(kept[..., None].expand(T, groups, E // groups).reshape(T, E), rank, -math.inf)
    order = best_first(rank)
    taken, idx = order.values[:, :topk] > -math.inf, order.indices[:, :topk]
    if renormalize and score == "softmax":
        lk = torch.where(taken, l.gather(1, idx), -math.inf)
        x = torch.where(taken, torch.exp(lk - lk.amax(1, keepdim=True)), 0.0)
        w = x / x.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        w = torch.where(taken, s.gather(1, idx), 0.0)
        if renormalize:
            w = w / (w.sum(1, keepdim=True) + 1e-20)
    return torch.where(taken, idx, -1), scale * w, s


def weight_bound(logits, w):
    """exp is off by 2 units (4 half ones), its argument by half a unit of the difference; sums of up to 1024 terms are 5 additions in a tree
    over up to 32 in a row, then a division, a scale, and the same again for a renormalised sum: 64 half units and the range of the logits."""
    l = logits.cpu().double()
    l = torch.where(torch.isfinite(l), l, 0.0)
    return (64 + 2 * (l.amax() - l.amin()).clamp_max(200)) * U32 * w.abs() + 1e-37


CASES = [
    # tokens, experts, topk, score, bias, groups, keep, group score, renormalize, scale, dtype
    (1, 1, 1, "softmax", False, 1, 1, "max", True, 1.0, torch.float32),
    (1, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5, torch.float32),
    (5, 3, 3, "sigmoid", False, 1, 1, "max", False, 1.0, torch.bfloat16),
    (33, 60, 6, "softmax", False, 1, 1, "max", False, 1.0, torch.float16),
    (257, 64, 6, "softmax", True, 8, 3, "max", True, 16.0, torch.bfloat16),
    (100, 72, 5, "softmax", False, 24, 5, "top2", False, 1.0, torch.float32),
    (700, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5, torch.bfloat16),
    (64, 32, 4, "sigmoid", False, 32, 7, "top2", True, 1.0, torch.float16),
    (300, 96, 9, "sigmoid", False, 4, 2, "top2", False, 0.5, torch.float32),
    (41, 1000, 16, "softmax", True, 1, 1, "max", False, 1.0, torch.float32),
    (19, 1024, 16, "sigmoid", False, 32, 2, "max", True, 1.0, torch.bfloat16),
    (2000, 128, 8, "softmax", False, 1, 1, "max", True, 1.0, torch.bfloat16),
    (150, 60, 7, "sigmoid", True, 5, 2, "top2", True, 1.0, torch.float32),        # groups that leave lanes without experts
    (70, 1020, 12, "softmax", False, 17, 6, "top2", False, 1.0, torch.bfloat16),  # the most experts of one lane
    (90, 111, 5, "sigmoid", True, 3, 1, "max", True, 1.0, torch.float16),
]


@pytest.mark.parametrize("T,E,K,score,biased,groups,keep,gs,renorm,scale,dtype", CASES)
@pytest.mark.parametrize("masked", [False, True])
def test_choice_weights_and_gradient(group, T, E, K, score, biased, groups, keep, gs, renorm, scale, dtype, masked):
    ep = group(E)
    g = torch.Generator(device="cuda").manual_seed(T * 31 + E)
    logits = 2 * torch.randn(T, E, device="cuda", generator=g)
    if masked:
        logits = logits.masked_fill(torch.rand(T, E, device="cuda", generator=g) < 0.5, -math.inf)
        logits[::3, : E // 2] = math.nan
        logits[T // 2] = -math.inf       # a padding row
        logits[-1, E // 2] = math.inf
        logits[0] = torch.finfo(dtype).min if T > 1 else logits[0]   # all of them the lowest number: equal, by index
    logits = logits.to(dtype)
    bias = torch.randn(E, device="cuda", generator=g) * (0.2 if score == "sigmoid" else 0.5 / E) if biased else None
    rule = dict(score=score, renormalize=renorm, scale=scale)
    idx, w = ep.route(logits, K, bias=bias, groups=groups, keep_groups=keep, group_score=gs, **rule)
    want, ww, s = reference(logits, K, bias=bias, groups=groups, keep_groups=keep, group_score=gs, **rule)
    assert torch.equal(idx.cpu(), want)
    assert ((w.cpu().double() - ww).abs() <= weight_bound(logits, ww)).all()
    if masked and T > 2:   # (else one of the lines below wrote over it)
        assert (idx[T // 2] == -1).all() and (w[T // 2] == 0).all()

    dw = torch.randn(T, K, device="cuda", generator=g)
    d = ep.route_backward(dw, logits, idx, **rule)
    assert d.dtype == dtype
    taken, gk = want >= 0, scale * dw.cpu().double()
    gk = torch.where(taken, gk, 0.0)
    at, u = want.clamp_min(0), ww / scale
    sk = torch.where(taken, s.gather(1, at), 0.0)
    zero = torch.zeros(T, E, dtype=torch.float64)
    # the largest intermediate terms bound the rounding: shares of the sum over the entries, times the units of a weight
    if renorm and score == "softmax":
        ref = zero.scatter_add(1, at, u * (gk - (gk * u).sum(1, keepdim=True)))
        size = zero.scatter_add(1, at, u * (gk.abs() + (gk * u).abs().sum(1, keepdim=True)))
    else:
        big = gk.abs()
        if renorm:
            total = sk.sum(1, keepdim=True) + 1e-20
            big = torch.where(taken, (big + (gk * u).abs().sum(1, keepdim=True)) / total, 0.0)
            gk = torch.where(taken, (gk - (gk * u).sum(1, keepdim=True)) / total, 0.0)
        if score == "sigmoid":
            other = torch.where(taken, 1 / (1 + torch.exp(torch.where(taken, logits.cpu().double().gather(1, at), 0.0))), 0.0)
            ref, size = zero.scatter_add(1, at, gk * sk * other), zero.scatter_add(1, at, big * sk * other)
        else:
            ref = zero.scatter_add(1, at, gk * sk) - s * (gk * sk).sum(1, keepdim=True)
            size = zero.scatter_add(1, at, big * sk) + s * (big * sk).sum(1, keepdim=True)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps   # half of the smallest step of the type
    assert ((d.cpu().double() - ref).abs() <= HALF[dtype] * ref.abs() + 4 * weight_bound(logits, size) + tiny).all()


def test_values_next_to_a_border_are_ordered_as_exact_arithmetic_orders_them(group):
    """Pairs of experts whose score + bias differ by far less than fp32 resolves, and pairs that are the same."""
    ep = group(64)
    T = 400
    g = torch.Generator(device="cuda").manual_seed(11)
    logits = torch.randn(T, 64, device="cuda", generator=g)
    bias = torch.randn(64, device="cuda", generator=g).double()
    for t in range(T):   # expert 2i+1 of token t: a logit whose score makes up for the difference of the biases
        i = t % 32
        target = (torch.sigmoid(logits[t, 2 * i].double()) + bias[2 * i].float().double() - bias[2 * i + 1].float().double()).clamp(1e-3, 1 - 1e-3)
        logits[t, 2 * i + 1] = torch.log(target / (1 - target)).float()
    bias = bias.float()
    logits[1] = logits[1, 0]
    bias[10:14] = bias[10]
    logits[:, 10:14] = logits[:, 10:11]
    for rule in (dict(), dict(groups=32, keep_groups=5, group_score="top2"), dict(groups=16, keep_groups=3, group_score="max")):
        idx, w = ep.route(logits, 6, score="sigmoid", bias=bias, **rule)
        want, ww, _ = reference(logits, 6, "sigmoid", bias=bias, **rule)
        assert torch.equal(idx.cpu(), want)
        assert ((w.cpu().double() - ww).abs() <= weight_bound(logits, ww)).all()


def test_far_logits_keep_their_order(group):
    """Sigmoids that are all 1 in fp32, softmax shares that are all 0: the logits still order them."""
    ep = group(32)
    logits = (torch.arange(32, device="cuda", dtype=torch.float32) * 5 + 20).flip(0).repeat(3, 1)
    logits[1] = -logits[1]
    logits[2, 5] = 3e38
    for score in ("sigmoid", "softmax"):
        idx, w = ep.route(logits, 16, score=score)
        want, ww, _ = reference(logits, 16, score)
        assert torch.equal(idx.cpu(), want)
        assert torch.isfinite(w).all() and ((w.cpu().double() - ww).abs() <= (64 + 400) * U32 * ww + 1e-37).all()


def test_gradient_against_differences(group):
    ep = group(24)
    g = torch.Generator(device="cuda").manual_seed(3)
    logits, dw = torch.randn(4, 24, device="cuda", generator=g), torch.randn(4, 5, device="cuda", generator=g)
    for rule in (dict(score="softmax"), dict(score="softmax", renormalize=False, scale=3.0), dict(score="sigmoid", scale=2.5), dict(score="sigmoid", renormalize=False)):
        idx, _ = ep.route(logits, 5, **rule)
        d = ep.route_backward(dw, logits, idx, **rule).cpu().double()

        def value(l):
            s = torch.softmax(l, 1) if rule["score"] == "softmax" else torch.sigmoid(l)
            w = s.gather(1, idx.cpu())
            w = w / w.sum(1, keepdim=True) if rule.get("renormalize", True) else w
            return (rule.get("scale", 1.0) * w * dw.cpu().double()).sum(1)

        l, h = logits.cpu().double(), 1e-5
        for e in range(24):
            step = torch.zeros(24, dtype=torch.float64)
            step[e] = h
            slope = (value(l + step) - value(l - step)) / (2 * h)
            # central differences: h^2 / 6 of a third derivative (below 10 x the weights' gradients), and 2^-52 / h of rounding
            assert ((d[:, e] - slope).abs() <= 64 * U32 * 10 * dw.cpu().double().abs().sum(1) + 1e-8).all()


def test_indices_that_repeat_or_lie_outside(group):
    """An expert that is named twice gets both shares; -1 and what is no expert adds nothing."""
    ep = group(8)
    logits = torch.randn(3, 8, device="cuda")
    dw = torch.randn(3, 4, device="cuda")
    idx = torch.tensor([[2, 2, 5, -1], [7, 8, 1 << 40, 0], [-1, -1, -5, -1]], device="cuda")
    for rule in (dict(score="softmax"), dict(score="softmax", renormalize=False), dict(score="sigmoid"), dict(score="sigmoid", renormalize=False)):
        d = ep.route_backward(dw, logits, idx, **rule).cpu().double()
        l = logits.cpu().double().requires_grad_(True)
        s = torch.softmax(l, 1) if rule["score"] == "softmax" else torch.sigmoid(l)
        ok = ((idx >= 0) & (idx < 8)).cpu()
        w = s.gather(1, idx.cpu().clamp(0, 7)) * ok
        if rule.get("renormalize", True):
            w = w / w.sum(1, keepdim=True).clamp_min(1e-30)
        ref, = torch.autograd.grad((w * dw.cpu().double() * ok).sum(), l)
        assert ((d - ref).abs() <= 256 * U32 * dw.cpu().double().abs().sum(1, keepdim=True) + 1e-30).all()
        assert (d[2] == 0).all()


def test_rows_at_any_address_streams_and_graphs(group):
    ep = group(256)
    raw = torch.randn(64 * 256 + 1, device="cuda").bfloat16()
    shifted = raw[1:].view(64, 256)    # 2-byte aligned
    whole = shifted.clone()
    a, b = ep.route(shifted, 8), ep.route(whole, 8)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    dw = torch.randn(64, 8, device="cuda")
    assert torch.equal(ep.route_backward(dw, shifted, a[0]), ep.route_backward(dw, whole, a[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = ep.route(whole, 8)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c[0], b[0]) and torch.equal(c[1], b[1])
    idx, w = torch.empty_like(b[0]), torch.empty_like(b[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ep.route(whole, 8, idx=idx, weights=w)
        d = ep.route_backward(dw, whole, idx)
    whole.copy_(torch.randn(64, 256, device="cuda").bfloat16())
    graph.replay()
    want = ep.route(whole, 8)
    assert torch.equal(idx, want[0]) and torch.equal(w, want[1]) and torch.equal(d, ep.route_backward(dw, whole, want[0]))


def test_no_tokens_and_refusals(group):
    from nccl_b200._lib import NcclError
    ep = group(16)
    idx, w = ep.route(torch.empty(0, 16, device="cuda"), 4)
    assert idx.shape == w.shape == (0, 4)
    assert ep.route_backward(w, torch.empty(0, 16, device="cuda"), idx).shape == (0, 16)
    l = torch.randn(5, 16, device="cuda")
    for bad in (l[:, :8], l.double(), l.t().contiguous().t(), l.cpu(), l[0]):
        with pytest.raises(ValueError):
            ep.route(bad, 4)
    for args in (dict(topk=17), dict(topk=0), dict(topk=4, groups=3), dict(topk=4, groups=0), dict(topk=4, groups=4, keep_groups=5), dict(topk=9, groups=4, keep_groups=2),
                 dict(topk=4, scale=0.0), dict(topk=4, scale=math.nan), dict(topk=4, scale=math.inf)):
        with pytest.raises(NcclError):
            ep.route(l, args.pop("topk"), **args)
    for args in (dict(score="tanh"), dict(group_score="mean"), dict(bias=torch.zeros(15, device="cuda")), dict(bias=torch.zeros(16, device="cuda").bfloat16()),
                 dict(bias=torch.zeros(16)), dict(idx=torch.zeros(5, 4, device="cuda", dtype=torch.int32)), dict(weights=torch.zeros(4, 5, device="cuda"))):
        with pytest.raises(ValueError):
            ep.route(l, 4, **args)
    raw = torch.zeros(5 * 16 + 40, device="cuda")
    for kw in (dict(weights=raw[:20].view(5, 4)), dict(idx=raw[10:50].view(torch.int64).view(5, 4))):
        with pytest.raises(NcclError):   # over the logits
            ep.route(raw[:80].view(5, 16), 4, **kw)
    idx, w = ep.route(l, 4)
    place = l.clone()
    assert torch.equal(ep.route_backward(w, place, idx, renormalize=False, out=place), ep.route_backward(w, l, idx, renormalize=False)) and not torch.equal(place, l)
    with pytest.raises(NcclError):
        ep.route_backward(raw[70:90].view(5, 4), l, idx, out=raw[:80].view(5, 16))
    for dw, i in ((w.double(), idx), (w[:, :3], idx), (w, idx[:4])):
        with pytest.raises(ValueError):
            ep.route_backward(dw, l, i)
