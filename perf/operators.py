"""The operators of a mixture-of-experts layer, as measurable cases: what a program that uses this framework calls around
``ExpertParallel.dispatch`` and ``combine``.

    route     ``ExpertParallel.route``: scores, bias, groups, top-k and weights of a batch's router logits;
              with ``train`` also ``route_backward``
    experts   ``ExpertParallel.expert_linear``: one product per expert over the rows that dispatch packed, with bias, activation and
              residual; with ``train`` also ``expert_linear_backward``
    combine   ``ExpertParallel.combine_backward`` and ``dispatch_backward``: the gradients that cross the exchange

``own`` false: the same in elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GATED = ("swiglu", "geglu")


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # decoding one sequence: sigmoid scores, a bias that balances the load, the best four of eight groups
        {"name": "route_token", "kind": "route", "tokens": 1, "experts": 256, "topk": 8, "score": "sigmoid", "dtype": "f32", "bias": True, "groups": 8,
         "keep_groups": 4, "group_score": "top2", "renormalize": True, "scale": 2.5, "masked": False, "train": False},
        # the same router on a prefill batch
        {"name": "route_prefill", "kind": "route", "tokens": 8192, "experts": 256, "topk": 8, "score": "sigmoid", "dtype": "bf16", "bias": True, "groups": 8,
         "keep_groups": 4, "group_score": "top2", "renormalize": True, "scale": 2.5, "masked": False, "train": False},
        # plain softmax weights over an odd number of experts; padding tokens, and experts that are switched off
        {"name": "route_masked", "kind": "route", "tokens": 1999, "experts": 60, "topk": 6, "score": "softmax", "dtype": "f16", "bias": False, "groups": 1,
         "keep_groups": 1, "group_score": "max", "renormalize": False, "scale": 1.0, "masked": True, "train": False},
        # a training step's router, there and back
        {"name": "route_train", "kind": "route", "tokens": 16384, "experts": 128, "topk": 8, "score": "softmax", "dtype": "bf16", "bias": False, "groups": 1,
         "keep_groups": 1, "group_score": "max", "renormalize": True, "scale": 1.0, "masked": False, "train": True},
        # one token on two of eight large experts: their weights are the traffic
        {"name": "experts_token", "kind": "experts", "experts": 8, "tokens": 1, "topk": 2, "k": 4096, "n": 28672, "activation": "swiglu", "bias": False,
         "residual": False, "train": False},
        # a decoding batch on one GPU's share of many experts, a few rows each
        {"name": "experts_decode", "kind": "experts", "experts": 32, "tokens": 64, "topk": 8, "k": 7168, "n": 4096, "activation": "swiglu", "bias": False,
         "residual": False, "train": False},
        # the projection back, with a bias and the layer's input added; sizes that fill no tile
        {"name": "experts_down_ragged", "kind": "experts", "experts": 64, "tokens": 1501, "topk": 6, "k": 1400, "n": 2056, "activation": "none", "bias": True,
         "residual": True, "train": False},
        # a prefill batch: hundreds to thousands of rows for each expert
        {"name": "experts_prefill", "kind": "experts", "experts": 16, "tokens": 4096, "topk": 8, "k": 7168, "n": 4096, "activation": "swiglu", "bias": False,
         "residual": False, "train": False},
        # a training step's gate and up products of large experts, there and back
        {"name": "experts_train", "kind": "experts", "experts": 8, "tokens": 2048, "topk": 2, "k": 4096, "n": 28672, "activation": "swiglu", "bias": False,
         "residual": False, "train": True},
        # the same for small experts with biases, sizes that fill no tile
        {"name": "experts_train_ragged", "kind": "experts", "experts": 5, "tokens": 777, "topk": 2, "k": 1000, "n": 2200, "activation": "gelu", "bias": True,
         "residual": True, "train": True},
        # gradients of a small batch
        {"name": "combine_small", "kind": "combine", "experts": 32, "tokens": 16, "topk": 8, "hidden": 4096, "drop": 0.0},
        # gradients of a training batch, some of its entries dropped
        {"name": "combine_train", "kind": "combine", "experts": 16, "tokens": 4096, "topk": 8, "hidden": 7168, "drop": 0.05},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "route", "experts", "experts", "experts", "combine"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * rng.randint(2, 256 // groups)
        keep = rng.randint(1, groups)
        score = rng.choice(["softmax", "sigmoid"])
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "experts": experts, "topk": rng.randint(1, min(10, experts // groups * keep)), "score": score,
                "dtype": rng.choice(["f32", "bf16", "f16"]), "bias": rng.random() < 0.5, "groups": groups, "keep_groups": keep,
                "group_score": rng.choice(["max", "top2"]), "renormalize": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]),
                "masked": rng.random() < 0.3, "train": rng.random() < 0.4}
    if kind == "combine":
        experts, topk = rng.choice([2, 8, 16, 32]), rng.randint(1, 8)
        return {"kind": kind, "experts": experts, "tokens": _log(rng, 1, 65536 // experts), "topk": min(topk, experts), "hidden": 128 * rng.randint(4, 56),
                "drop": rng.choice([0.0, 0.1])}
    while True:
        train = rng.random() < 0.4
        act = rng.choice(["none", "relu", "gelu", "silu", "swiglu", "swiglu", "geglu"])
        experts = rng.choice([1, 3, 4, 8, 16, 32, 64])
        step = 16 if act in GATED else 8
        c = {"kind": kind, "experts": experts, "tokens": _log(rng, 1, 4096), "topk": rng.randint(1, min(8, experts)), "k": 8 * _log(rng, 16, 896),
             "n": step * _log(rng, 128 // step, 14336 // step), "activation": act, "bias": rng.random() < 0.4, "residual": rng.random() < 0.3, "train": train}
        # neither more products than the largest listed case has, nor more weights
        if c["experts"] * c["tokens"] * c["k"] * c["n"] * (3 if train else 1) < 3e12 and c["experts"] * c["k"] * c["n"] < 9e8:
            return c


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 23)


def _choices(c, g):
    """Logits of a router with popular and unpopular experts."""
    return torch.randn(c["tokens"], c["experts"], device="cuda", generator=g) + 0.5 * torch.randn(1, c["experts"], device="cuda", generator=g)


def _route_inputs(c, seed):
    g = _gen(seed)
    T, E, K = c["tokens"], c["experts"], c["topk"]
    logits = _choices(c, g)
    if c["masked"]:   # padding tokens have no expert at all, some experts are off for everybody
        logits = logits.masked_fill(torch.rand(T, 1, device="cuda", generator=g) < 0.1, -math.inf)
        logits = logits.masked_fill(torch.rand(1, E, device="cuda", generator=g) < 0.1, -math.inf)
    spread = 0.1 if c["score"] == "sigmoid" else 0.5 / E
    bias = spread * torch.randn(E, device="cuda", generator=g) if c["bias"] else None
    grad = torch.randn(T, K, device="cuda", generator=g) if c["train"] else None
    return logits.to(DTYPES[c["dtype"]]), bias, grad


def _experts_inputs(c, seed):
    g = _gen(seed)
    E, cap, K, N = c["experts"], c["tokens"], c["k"], c["n"]
    out = N // 2 if c["activation"] in GATED else N
    counts = torch.bincount(_choices(c, g).topk(c["topk"], dim=1).indices.reshape(-1), minlength=E).int()
    x = torch.randn(E, cap, K, dtype=torch.bfloat16, device="cuda", generator=g)
    w = torch.randn(E, N, K, dtype=torch.bfloat16, device="cuda", generator=g).mul_(1 / math.sqrt(K))
    bias = (0.5 * torch.randn(E, N, device="cuda", generator=g)).bfloat16() if c["bias"] else None
    residual = torch.randn(E, cap, out, dtype=torch.bfloat16, device="cuda", generator=g) if c["residual"] else None
    grad = torch.randn(E, cap, out, dtype=torch.bfloat16, device="cuda", generator=g) if c["train"] else None
    return x, w, counts, bias, residual, grad


def _combine_inputs(c, seed):
    """The gradient of combine's result, the experts' rows and their gradients, and where dispatch put each entry: the rows of an
    expert are packed in any order, -1 stands for an entry without an expert."""
    g = _gen(seed)
    T, E, K, H = c["tokens"], c["experts"], c["topk"], c["hidden"]
    e = _choices(c, g).topk(K, dim=1).indices.reshape(-1)
    if c["drop"]:
        e = e.masked_fill(torch.rand(T * K, device="cuda", generator=g) < c["drop"], E)
    mixed = torch.randperm(T * K, device="cuda", generator=g)
    order = mixed[torch.sort(e[mixed], stable=True).indices]
    start = torch.cumsum(torch.bincount(e, minlength=E + 1), 0) - torch.bincount(e, minlength=E + 1)
    rows = torch.empty(T * K, dtype=torch.int64, device="cuda")
    rows[order] = torch.arange(T * K, device="cuda") - start[e[order]] + e[order] * T
    rows = rows.masked_fill(e == E, -1).int().view(T, K)
    weights = torch.rand(T, K, device="cuda", generator=g)
    dout = torch.randn(T, H, dtype=torch.bfloat16, device="cuda", generator=g)
    y = torch.randn(E, T, H, dtype=torch.bfloat16, device="cuda", generator=g)
    dtoks = torch.randn(E, T, H, dtype=torch.bfloat16, device="cuda", generator=g)
    return dout, y, weights, rows, dtoks


# ------------------------------------------------------------------------------------------------ state
_process = {}


def _ep(experts):
    """The expert-parallel group that such a program keeps."""
    if experts not in _process:
        from nccl_b200 import Communicator, get_unique_id
        from nccl_b200.ops.ep import ExpertParallel
        torch.cuda.set_device(0)
        if "comm" not in _process:
            _process["comm"] = Communicator(1, 0, get_unique_id())
        _process[experts] = ExpertParallel(_process["comm"], experts, 1, 128)
    return _process[experts]


def prepare(case, seed):
    c, s = case, {"case": case, "ep": _ep(case["experts"]) if own else None}
    if c["kind"] == "route":
        s["logits"], s["bias"], s["grad"] = _route_inputs(c, seed)
    elif c["kind"] == "experts":
        s["x"], s["w"], s["counts"], s["bias"], s["residual"], s["grad"] = _experts_inputs(c, seed)
        # rows behind an expert's last are nobody's: they stay as they are
        out = c["n"] // 2 if c["activation"] in GATED else c["n"]
        s["out"] = torch.zeros(c["experts"], c["tokens"], out, dtype=torch.bfloat16, device="cuda")
        if c["train"]:
            s["pre"] = torch.zeros(c["experts"], c["tokens"], c["n"], dtype=torch.float32, device="cuda")
            s["dx"] = torch.zeros_like(s["x"])
    else:
        s["dout"], s["y"], s["weights"], s["rows"], s["dtoks"] = _combine_inputs(c, seed)
        s["dy"] = torch.zeros_like(s["y"])
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _best_first(v):
    """Values and places in descending order, equal ones by place."""
    return torch.sort(v, dim=-1, descending=True, stable=True)


def _plain_route(c, logits, bias):
    """In 64 bits: scores next to each other decide which expert is taken."""
    T, E, K, G = c["tokens"], c["experts"], c["topk"], c["groups"]
    l = logits.double()
    there = l > -math.inf
    top = torch.where(there, l, -1e300).amax(-1, keepdim=True)
    if c["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-l))
    else:
        p = torch.where(there, torch.exp(l - top), 0.0)
        s = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    rank = torch.where(there, s if bias is None else s + bias, -math.inf)
    if G > 1:
        best = _best_first(rank.view(T, G, E // G)).values
        second = best[..., 1] if c["group_score"] == "top2" and E // G > 1 else torch.full_like(best[..., 0], -math.inf)
        of_group = best[..., 0] + torch.where(second > -math.inf, second, 0.0)
        kept = torch.zeros(T, G, dtype=torch.bool, device="cuda").scatter_(1, _best_first(of_group).indices[:, :c["keep_groups"]], True)
        rank = torch.where(kept[..., None].expand(T, G, E // G).reshape(T, E), rank, -math.inf)
    order = _best_first(rank)
    taken, idx = order.values[:, :K] > -math.inf, order.indices[:, :K]
    w = torch.where(taken, s.gather(1, idx), 0.0)
    if c["renormalize"]:
        if c["score"] == "softmax":
            lk = torch.where(taken, l.gather(1, idx), -math.inf)
            w = torch.where(taken, torch.exp(lk - lk.amax(-1, keepdim=True)), 0.0)
            w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
        else:
            w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return torch.where(taken, idx, -1), c["scale"] * w, s


def _plain_route_backward(c, grad, logits, idx, w, s):
    T, E = c["tokens"], c["experts"]
    taken = idx >= 0
    at, g = idx.clamp_min(0), torch.where(taken, c["scale"] * grad.double(), 0.0)
    share = w / c["scale"]
    if c["renormalize"] and c["score"] == "softmax":
        d = share * (g - (g * share).sum(-1, keepdim=True))
        return torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_add_(1, at, d)
    sk = torch.where(taken, s.gather(1, at), 0.0)
    if c["renormalize"]:
        g = torch.where(taken, (g - (g * share).sum(-1, keepdim=True)) / (sk.sum(-1, keepdim=True) + 1e-20), 0.0)
    if c["score"] == "sigmoid":
        return torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_add_(1, at, g * sk * (1 - sk))
    return torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_add_(1, at, g * sk) - s * (g * sk).sum(-1, keepdim=True)


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _normal_cdf(v):
    return 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))


def _activate(act, z):
    """The activation's value and, for its backward, the slopes by z (by gate and by up where it is gated)."""
    if act in GATED:
        half = z.shape[-1] // 2
        gate, up = z[..., :half], z[..., half:]
        value, slope = _activate("silu" if act == "swiglu" else "gelu", gate)
        return value * up, (slope, up, value)
    if act == "relu":
        return z * (z > 0), (z > 0).float()
    if act == "silu":
        s = _sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = _normal_cdf(z)
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _plain_experts(s):
    c = s["case"]
    E, cap, act = c["experts"], c["tokens"], c["activation"]
    used = (torch.arange(cap, device="cuda") < s["counts"][:, None])[..., None]
    x, w = s["x"].float(), s["w"].float()
    z = torch.bmm(x, w.mT)
    if s["bias"] is not None:
        z = z + s["bias"].float()[:, None]
    value, slope = _activate(act, z)
    out = value if s["residual"] is None else value + s["residual"].float()
    out = torch.where(used, out, 0.0).bfloat16()
    if not c["train"]:
        return out
    g = torch.where(used, s["grad"].float(), 0.0)
    dz = torch.cat([g * slope[1] * slope[0], g * slope[2]], -1) if act in GATED else g * slope
    got = {"out": out, "dx": torch.bmm(dz, w).bfloat16(), "dw": torch.bmm(dz.mT, torch.where(used, x, 0.0)).bfloat16()}
    if s["bias"] is not None:
        got["dbias"] = dz.sum(1).bfloat16()
    return got


def _plain_combine(s):
    c = s["case"]
    T, K, H = c["tokens"], c["topk"], c["hidden"]
    there = s["rows"] >= 0
    at = s["rows"].clamp_min(0).long().view(-1)
    w = torch.where(there, s["weights"], 0.0)
    dout = s["dout"].float()
    given = (w[..., None] * dout[:, None]).bfloat16()
    dy = torch.zeros_like(s["y"]).view(-1, H)
    keep = torch.nonzero(there.view(-1)).view(-1)
    dy[at[keep]] = given.view(-1, H)[keep]
    y = s["y"].view(-1, H)[at].view(T, K, H).float()
    dw = torch.where(there, (y * dout[:, None]).sum(-1), 0.0)
    back = s["dtoks"].view(-1, H)[at].view(T, K, H).float()
    dx = torch.where(there[..., None], back, 0.0).sum(1).bfloat16()
    return {"dy": dy.view_as(s["y"]), "dweights": dw, "dx": dx}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if c["kind"] == "route":
        if own:
            rule = dict(score=c["score"], renormalize=c["renormalize"], scale=c["scale"])
            idx, w = s["ep"].route(s["logits"], c["topk"], bias=s["bias"], groups=c["groups"], keep_groups=c["keep_groups"], group_score=c["group_score"], **rule)
            if not c["train"]:
                return {"idx": idx, "weights": w}
            return {"idx": idx, "weights": w, "dlogits": s["ep"].route_backward(s["grad"], s["logits"], idx, **rule)}
        idx, w, score = _plain_route(c, s["logits"], s["bias"])
        if not c["train"]:
            return {"idx": idx, "weights": w.float()}
        return {"idx": idx, "weights": w.float(), "dlogits": _plain_route_backward(c, s["grad"], s["logits"], idx, w, score).to(s["logits"].dtype)}
    if c["kind"] == "experts":
        if not own:
            return _plain_experts(s)
        ep, act = s["ep"], None if c["activation"] == "none" else c["activation"]
        if not c["train"]:
            return ep.expert_linear(s["x"], s["w"], s["counts"], bias=s["bias"], activation=act, residual=s["residual"], out=s["out"])
        out = ep.expert_linear(s["x"], s["w"], s["counts"], bias=s["bias"], activation=act, residual=s["residual"], out=s["out"], pre=s["pre"])
        dx, dw, dbias = ep.expert_linear_backward(s["grad"], s["x"], s["w"], s["counts"], pre=s["pre"], activation=act, need_dbias=c["bias"], dx=s["dx"])
        return {"out": out, "dx": dx, "dw": dw, "dbias": dbias} if c["bias"] else {"out": out, "dx": dx, "dw": dw}
    if not own:
        return _plain_combine(s)
    dy, dw = s["ep"].combine_backward(s["dout"], s["y"], s["weights"], s["rows"], dy=s["dy"])
    return {"dy": dy, "dweights": dw, "dx": s["ep"].dispatch_backward(s["dtoks"], s["rows"])}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    T, E, K = c["tokens"], c["experts"], c["topk"]
    if c["kind"] == "route":
        size = DTYPES[c["dtype"]].itemsize
        there = T * E * size + T * K * 12 + (E * 4 if c["bias"] else 0)
        # back: the weights' gradient in, the logits' out
        return {"bytes": there + (T * K * 4 + T * E * size if c["train"] else 0), "flops": 6 * T * E * (2 if c["train"] else 1)}
    if c["kind"] == "combine":
        H, rows = c["hidden"], T * K * (1 - c["drop"])
        # dout, the experts' rows and their gradients in; the rows' gradients, the weights' and the tokens' out
        return {"bytes": T * H * 2 + 2 * rows * H * 2 + T * K * 12 + rows * H * 2 + T * H * 2, "flops": 4 * rows * H}
    k, n = c["k"], c["n"]
    out = n // 2 if c["activation"] in GATED else n
    rows, active = T * K, E * (1 - (1 - K / E) ** T)   # experts that a token chose, if all are as popular
    there = active * n * k * 2 + rows * (k + out * (2 if c["residual"] else 1)) * 2 + (active * n * 2 if c["bias"] else 0)
    if not c["train"]:
        return {"bytes": there, "flops": 2 * rows * n * k}
    # back: the result's gradient in; the gradients of the rows, of all experts' weights and of their biases out
    return {"bytes": there + rows * (out + k) * 2 + E * n * k * 2 + (E * n * 2 if c["bias"] else 0), "flops": 6 * rows * n * k}


# ------------------------------------------------------------------------------------------------ 64-bit results
def _exact_route(c, logits, bias, grad):
    """Takes one expert after the other; gradients by differentiation."""
    T, E, K, G = c["tokens"], c["experts"], c["topk"], c["groups"]
    l = logits.double()
    off = l.isneginf()
    if c["train"]:
        l.requires_grad_(True)
    safe = torch.where(off, torch.full_like(l, -1e4), l)
    s = torch.special.expit(safe) if c["score"] == "sigmoid" else torch.softmax(safe, -1)
    with torch.no_grad():
        left = (s + bias.double() if bias is not None else s.clone()).masked_fill(off, -math.inf)
        if G > 1:
            view = left.view(T, G, -1)
            two = view.topk(min(2 if c["group_score"] == "top2" else 1, E // G), dim=-1).values
            score = torch.where(view.isneginf().all(-1), -math.inf, two.masked_fill(two.isneginf(), 0).sum(-1))
            for _ in range(G - c["keep_groups"]):   # the worst group goes, of equal ones the last
                worst = G - 1 - score.flip(1).argmin(1)
                view[torch.arange(T, device="cuda"), worst] = -math.inf
                score[torch.arange(T, device="cuda"), worst] = math.inf
        picks = []
        for _ in range(K):
            best = left.argmax(1)
            picks.append(torch.where(left.gather(1, best[:, None])[:, 0].isneginf(), -1, best))
            left[torch.arange(T, device="cuda"), best] = -math.inf
        picks = torch.stack(picks, 1)
    w = s.gather(1, picks.clamp_min(0)) * (picks >= 0)
    if c["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = w / (total + 1e-20 if c["score"] == "sigmoid" else torch.where(total > 0, total, 1.0))
    w = c["scale"] * w
    if not c["train"]:
        return {"idx": None, "weights": w}
    d, = torch.autograd.grad((w * grad.double()).sum(), l)
    return {"idx": None, "weights": w.detach(), "dlogits": d}


def _exact_experts(c, inputs):
    x, w, counts, bias, residual, grad = inputs
    E, cap, n = c["experts"], c["tokens"], c["n"]
    gated = c["activation"] in GATED
    out = torch.zeros(E, cap, n // 2 if gated else n, dtype=torch.float64, device="cuda")
    got = {"out": out}
    if c["train"]:
        # what a gradient is held in is bf16: 64 bits of it all would be several times the case
        got["dx"], got["dw"] = torch.zeros(x.shape, dtype=torch.float32, device="cuda"), torch.zeros(w.shape, dtype=torch.float32, device="cuda")
        if bias is not None:
            got["dbias"] = torch.zeros(E, n, dtype=torch.float64, device="cuda")
    F = torch.nn.functional
    shape = {"none": lambda v: v, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "swiglu": F.silu, "geglu": F.gelu}[c["activation"]]
    for e, rows in enumerate(counts.tolist()):
        if rows == 0:
            continue
        xe, we = x[e, :rows].double().requires_grad_(c["train"]), w[e].double().requires_grad_(c["train"])
        be = (bias[e].double() if bias is not None else torch.zeros(n, dtype=torch.float64, device="cuda")).requires_grad_(c["train"])
        z = F.linear(xe, we, be)
        v = shape(z[:, :n // 2]) * z[:, n // 2:] if gated else shape(z)
        out[e, :rows] = v.detach() if residual is None else v.detach() + residual[e, :rows].double()
        if c["train"]:
            dx, dw, db = torch.autograd.grad(v, (xe, we, be), grad[e, :rows].double())
            got["dx"][e, :rows], got["dw"][e] = dx.float(), dw.float()
            if bias is not None:
                got["dbias"][e] = db
    if not c["train"]:
        return out
    return {k: v.double() for k, v in got.items()}


def _exact_combine(c, inputs):
    """combine is linear in its rows and in its weights: the gradients are those of the sum that defines it."""
    dout, y, weights, rows, dtoks = inputs
    H, none = c["hidden"], rows < 0
    at = rows.long().masked_fill(none, 0)
    g = dout.double()
    dy = torch.zeros(y.shape, dtype=torch.float32, device="cuda").view(-1, H)
    dw = torch.zeros(rows.shape, dtype=torch.float64, device="cuda")
    dx = torch.zeros(dout.shape, dtype=torch.float64, device="cuda")
    for k in range(c["topk"]):
        on = ~none[:, k]
        dy[at[on, k]] = (weights[on, k, None].double() * g[on]).float()
        dw[on, k] = torch.einsum("th,th->t", y.view(-1, H)[at[on, k]].double(), g[on])
        dx[on] += dtoks.view(-1, H)[at[on, k]].double()
    return {"dy": dy.view_as(y).double(), "dweights": dw, "dx": dx}


def exact(case, seed):
    c = case
    if c["kind"] == "route":
        return _exact_route(c, *_route_inputs(c, seed))
    if c["kind"] == "experts":
        return _exact_experts(c, _experts_inputs(c, seed))
    return _exact_combine(c, _combine_inputs(c, seed))
