"""The operators of attention over a sequence that ranks share, as measurable cases: what a program calls on its own rows and on the blocks of keys
and values that come to it.

    rotary    ``ContextParallel.rotary``: rotary positions of queries and keys (with ``inverse``: of their gradients)
    attend    ``ContextParallel.attention``: the result and its log-sum-exp; with ``join`` the last step of a ring, which adds a block to a partial result in fp32
    back      ``ContextParallel.attention_backward``: with ``join`` the last step of a ring, which adds to gradients in fp32

``own`` false: the same in elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def _attention(name, kind, batch, q, kv, heads, kv_heads, dim, dtype="bf16", causal=True, offset=None, lengths=False, join=False, packed=False):
    return {"name": name, "kind": kind, "batch": batch, "q": q, "kv": kv, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal,
            "offset": offset, "lengths": lengths, "join": join, "packed": packed}


def _rotary(name, batch, tokens, heads, kv_heads, dim, turned, dtype="bf16", interleaved=False, scaling=None, given=False, start=0, inverse=False):
    return {"name": name, "kind": "rotary", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "turned": turned, "dtype": dtype,
            "interleaved": interleaved, "scaling": scaling, "given": given, "start": start, "inverse": inverse}


def listed():
    return [
        # decoding one sequence: the new token's queries and keys, far into a long context
        _rotary("rotary_token", 1, 1, 32, 8, 128, 128, scaling="by_parts", given=True),
        # a rank's slice of a long sequence, in the middle of it
        _rotary("rotary_slice", 1, 16384, 32, 8, 128, 128, scaling="by_parts", start=114688),
        # gradients of a padded batch, neighbouring channels turned together, part of each head
        _rotary("rotary_part_back", 3, 1333, 12, 4, 80, 40, "f16", interleaved=True, scaling="linear", given=True, inverse=True),
        # decoding one sequence: the cache is the traffic
        _attention("attend_token", "attend", 1, 1, 4096, 32, 8, 128),
        # decoding a batch of sequences of all lengths
        _attention("attend_cache", "attend", 64, 1, 8192, 32, 8, 128, lengths=True),
        # a padded batch against another sequence, sizes that fill no tile
        _attention("attend_ragged", "attend", 3, 777, 1013, 12, 4, 80, "f16", causal=False, lengths=True),
        # a training or prefill sequence
        _attention("attend_long", "attend", 1, 8192, 8192, 32, 8, 128, packed=True),
        # the last step of a ring: the keys of an earlier rank, all of them visible, join what is there already
        _attention("attend_ring", "attend", 1, 4096, 4096, 32, 8, 128, causal=False, join=True),
        # gradients of a small model's batch
        _attention("back_small", "back", 2, 256, 256, 8, 8, 64, "f16", packed=True),
        # gradients of a padded batch against another sequence, sizes that fill no tile
        _attention("back_ragged", "back", 3, 509, 641, 12, 4, 96, causal=False, lengths=True),
        # gradients of a training sequence
        _attention("back_long", "back", 1, 8192, 8192, 32, 8, 128, packed=True),
        # the ring's last step back: the gradients so far are in fp32
        _attention("back_ring", "back", 1, 4096, 4096, 32, 8, 128, causal=False, join=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "attend", "attend", "attend", "back", "back", "back"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    dim = rng.choice([64, 64, 128, 128, 128, 8 * rng.randint(2, 16)])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "rotary":
        batch, turned = rng.choice([1, 1, 2, 5]), rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)])
        c = _rotary(None, batch, _log(rng, 1, 16384 // batch), heads, kv_heads, dim, turned, rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.5,
                    rng.choice([None, "linear", "ntk", "by_parts"]) if turned > 2 else None, rng.random() < 0.5, rng.choice([0, 4096, 1000000]), rng.random() < 0.4)
    else:
        lengths = rng.random() < 0.4
        batch = _log(rng, 1, 64) if lengths else _log(rng, 1, 8)
        while True:
            # (where every query sees one key only, the gradients of queries and keys are zero: there is nothing to compare)
            least = 1 if kind == "attend" else 2
            kv = _log(rng, least, 16384)
            q = rng.choice([1 if kind == "attend" else kv, kv, _log(rng, least, kv)])
            if batch * heads * q * kv <= 32 * 8192 * 8192 and batch * kv * kv_heads * dim <= 64 * 8192 * 8 * 128:
                break
        causal = rng.random() < 0.6
        # negative: queries in front of the first key see nothing
        offset = rng.choice([None, None, 0, rng.randint(-q if kind == "attend" else 0, kv)]) if causal else None
        c = _attention(None, kind, batch, q, kv, heads, kv_heads, dim, dtype, causal, offset, lengths, rng.random() < 0.3, q == kv and rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6007 + 41)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def _attention_inputs(c, seed):
    """q, k, v, lengths of both sides (or None), what joins, and the gradient of the result."""
    g, t = _gen(seed), DTYPES[c["dtype"]]
    B, Q, K, H, G, D = c["batch"], c["q"], c["kv"], c["heads"], c["kv_heads"], c["dim"]
    if c["packed"]:   # one projection's result
        q, k, v = _randn(g, B, Q, H + 2 * G, D, dtype=t).split((H, G, G), dim=2)
    else:
        q, k, v = _randn(g, B, Q, H, D, dtype=t), _randn(g, B, K, G, D, dtype=t), _randn(g, B, K, G, D, dtype=t)
    q_len = kv_len = None
    if c["lengths"]:   # one sequence of full length, one without a token where there are several
        kv_len = torch.randint(0, K + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        q_len = torch.randint(0, Q + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        kv_len[0], q_len[0] = K, Q
        if B > 2:
            kv_len[1] = 0
        q_len = kv_len if Q == K else None if Q == 1 else q_len
    join, dout = None, None
    if c["kind"] == "attend" and c["join"]:
        join = _randn(g, B, Q, H, D), _randn(g, B, H, Q) + math.log(K)
    if c["kind"] == "back":
        dout = _randn(g, B, Q, H, D, dtype=t)
        if c["join"]:
            join = _randn(g, B, Q, H, D), _randn(g, B, K, G, D), _randn(g, B, K, G, D)
    return q, k, v, q_len, kv_len, join, dout


def _rotary_inputs(c, seed):
    g, t = _gen(seed), DTYPES[c["dtype"]]
    B, T = c["batch"], c["tokens"]
    q, k = _randn(g, B, T, c["heads"], c["dim"], dtype=t), _randn(g, B, T, c["kv_heads"], c["dim"], dtype=t)
    positions = None
    if c["given"]:   # sequences that began at different times
        positions = c["start"] + torch.randint(0, 131072, (B, 1), device="cuda", generator=g) + torch.arange(T, device="cuda")
    return q, k, positions


# the scaled forms: a base of 500000, contexts of 8192 tokens stretched eight times
BASE, ORIGINAL, FACTOR, LOW, HIGH, AMPLITUDE = 500000.0, 8192, 8.0, 1.0, 4.0, 1.2


# ------------------------------------------------------------------------------------------------ state
_process = {}


def _cp():
    """The context-parallel group that such a program keeps."""
    if "cp" not in _process:
        from nccl_b200 import Communicator, get_unique_id
        from nccl_b200.ops.cp import ContextParallel
        torch.cuda.set_device(0)
        _process["cp"] = ContextParallel(Communicator(1, 0, get_unique_id()))
    return _process["cp"]


def prepare(case, seed):
    c, s = case, {"case": case, "cp": _cp() if own else None}
    if c["kind"] == "rotary":
        s["q"], s["k"], s["positions"] = _rotary_inputs(c, seed)
        if own:
            s["freqs"] = s["cp"].rotary_frequencies(c["turned"], base=BASE, scaling=c["scaling"], factor=FACTOR, original_length=ORIGINAL, low=LOW, high=HIGH,
                                                    amplitude=AMPLITUDE if c["scaling"] == "by_parts" else 1.0)
        else:
            s["freqs"] = _plain_frequencies(c)
        return s
    s["q"], s["k"], s["v"], s["q_len"], s["kv_len"], s["join"], s["dout"] = _attention_inputs(c, seed)
    if c["kind"] == "back":   # the forward pass has been
        s["out"], s["lse"] = _plain_attention(s, None)
        s["out"] = s["out"].to(s["q"].dtype)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_frequencies(c):
    """Angles of one step, in 64 bits."""
    i = torch.arange(c["turned"] // 2, dtype=torch.float64, device="cuda")
    base = BASE * FACTOR ** (c["turned"] / (c["turned"] - 2)) if c["scaling"] == "ntk" else BASE
    f = base ** (-2 * i / c["turned"])
    if c["scaling"] == "linear":
        f = f / FACTOR
    if c["scaling"] == "by_parts":   # what turns often keeps its speed, what turns less than once in a context is slowed down
        part = ((ORIGINAL * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = f * (part + (1 - part) / FACTOR)
    return f


def _plain_rotary(s):
    c, r = s["case"], s["case"]["turned"]
    at = s["positions"] if s["positions"] is not None else c["start"] + torch.arange(c["tokens"], device="cuda")[None]
    angle = at.double()[..., None] * s["freqs"]
    amp = AMPLITUDE if c["scaling"] == "by_parts" else 1.0
    cos, sin = (amp * angle.cos()).float()[:, :, None], (amp * angle.sin()).float()[:, :, None]
    if c["inverse"]:
        sin = -sin
    got = []
    for x in (s["q"], s["k"]):
        f = x.float()
        a, b = (f[..., 0:r:2], f[..., 1:r:2]) if c["interleaved"] else (f[..., :r // 2], f[..., r // 2:r])
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1 if c["interleaved"] else -2).flatten(-2)
        got.append(torch.cat([y, f[..., r:]], -1).to(x.dtype))
    return {"q": got[0], "k": got[1]}


def _visible(c, q_len, kv_len):
    """[batch or 1, q, kv]: which keys a query sees; [batch or 1, q]: which queries are there."""
    i, j = torch.arange(c["q"], device="cuda")[None, :, None], torch.arange(c["kv"], device="cuda")[None, None, :]
    nq, nk = (c["q"] if q_len is None else q_len[:, None, None]), (c["kv"] if kv_len is None else kv_len[:, None, None])
    see = (i < nq) & (j < nk)
    if c["causal"]:
        see = see & (j <= i + (nk - nq if c["offset"] is None else c["offset"]))
    return see, (i < nq)[..., 0]


def _grouped(t, G):
    """[B, S, H, D] in 32 bits as [B, G, H / G * S, D]: the rows that share keys and values."""
    B, S, H, D = t.shape
    return t.float().reshape(B, S, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * S, D)


def _ungrouped(t, S):
    B, G, rows, D = t.shape
    return t.view(B, G, rows // S, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, G * rows // S, D)


def _hide(score, see, value):
    """Where a query does not see a key, in place."""
    B, G, rows, K = score.shape
    score.view(B, G, rows // see.shape[1], see.shape[1], K).masked_fill_(~see[:, None, None], value)


def _cleared(t, length):
    """Rows behind the last hold anything."""
    if length is None:
        return t
    return torch.where((torch.arange(t.shape[1], device="cuda") < length[:, None])[..., None, None], t, torch.zeros((), dtype=t.dtype, device="cuda"))


def _plain_attention(s, join):
    """The result in 32 bits, and its log-sum-exp."""
    c = s["case"]
    B, Q, H, D = s["q"].shape
    G = c["kv_heads"]
    see, there = _visible(c, s["q_len"], s["kv_len"])
    q = _grouped(_cleared(s["q"], s["q_len"]), G)
    k, v = (_grouped(_cleared(s[n], s["kv_len"]), G) for n in "kv")
    score = torch.matmul(q, k.mT).mul_(1 / math.sqrt(D))
    _hide(score, see, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse, out = (top + total.log()).view(B, H, Q), _ungrouped(out, Q)
    if join is None:
        return out, lse
    m = torch.maximum(lse, join[1])
    m = torch.where(m > -math.inf, m, 0.0)
    a, b = torch.exp(lse - m), torch.exp(join[1] - m)
    share = lambda w: torch.where(a + b > 0, w / (a + b), 0.0).transpose(1, 2)[..., None]   # noqa: E731
    out, lse = out * share(a) + join[0] * share(b), m + torch.log(a + b)
    return torch.where(there[..., None, None], out, 0.0), torch.where(there[:, None], lse, -math.inf)


def _plain_backward(s):
    c = s["case"]
    B, Q, H, D = s["q"].shape
    K, G, scale = c["kv"], c["kv_heads"], 1 / math.sqrt(D)
    see, _ = _visible(c, s["q_len"], s["kv_len"])
    q, do = (_grouped(_cleared(s[n], s["q_len"]), G) for n in ("q", "dout"))
    out = _grouped(_cleared(s["out"], s["q_len"]), G)
    k, v = (_grouped(_cleared(s[n], s["kv_len"]), G) for n in "kv")
    lse = s["lse"].view(B, G, H // G * Q, 1)
    p = torch.matmul(q, k.mT).mul_(scale)
    p.sub_(torch.where(lse > -math.inf, lse, 0.0)).exp_()
    _hide(p, see, 0.0)
    delta = (do * out).sum(-1, keepdim=True)
    dv = torch.matmul(p.mT, do)
    ds = torch.matmul(do, v.mT).sub_(delta).mul_(p)
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.mT, q) * scale
    got = [_ungrouped(dq, Q), _ungrouped(dk, K), _ungrouped(dv, K)]
    if s["join"] is not None:
        keep = [s["q_len"], s["kv_len"], s["kv_len"]]
        got = [_cleared(a + b, n) for a, b, n in zip(got, s["join"], keep)]
    return [t.to(s["q"].dtype).contiguous() for t in got]


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if c["kind"] == "rotary":
        if not own:
            return _plain_rotary(s)
        q, k = s["cp"].rotary(s["q"], s["k"], s["freqs"], positions=s["positions"], offset=c["start"], interleaved=c["interleaved"], inverse=c["inverse"])
        return {"q": q, "k": k}
    if own:
        rule = dict(causal=c["causal"], offset=c["offset"], q_lengths=s["q_len"], kv_lengths=s["kv_len"])
        if c["kind"] == "attend":
            out, lse = s["cp"].attention(s["q"], s["k"], s["v"], join=s["join"], **rule)
            return {"out": out, "lse": lse}
        dq, dk, dv = s["cp"].attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], add=s["join"], **rule)
        return {"dq": dq, "dk": dk, "dv": dv}
    if c["kind"] == "attend":
        out, lse = _plain_attention(s, s["join"])
        return {"out": out.to(s["q"].dtype), "lse": lse}
    return dict(zip(("dq", "dk", "dv"), _plain_backward(s)))


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(q, kv, causal, offset):
    """Pairs of a query and a key that it sees."""
    if not causal:
        return q * kv
    first = min(max(-offset, 0), q)               # from here on a query sees something,
    full = min(max(kv - 1 - offset, first), q)    # from here on everything
    n = full - first
    return n * (first + offset + 1) + n * (n - 1) // 2 + (q - full) * kv


def work(case):
    c = case
    size = DTYPES[c["dtype"]].itemsize
    if c["kind"] == "rotary":
        n = c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"])
        return {"bytes": 2 * n * c["dim"] * size + (8 * c["batch"] * c["tokens"] if c["given"] else 0), "flops": 3 * n * c["turned"]}
    B, Q, K, H, G, D = c["batch"], c["q"], c["kv"], c["heads"], c["kv_heads"], c["dim"]
    # lengths: the first sequence's are full, the second of several has no key, the others' are uniform; what they leave on average
    left = lambda mean: (1 + mean * (B - 1 if B < 3 else B - 2)) / B if c["lengths"] else 1.0   # noqa: E731
    qs, ks = (1.0 if Q == 1 else left(1 / 2)), left(1 / 2)
    pairs = B * _pairs(Q, K, c["causal"], K - Q if c["offset"] is None else c["offset"]) * left(1 / 2 if Q == 1 else 1 / 3 if Q == K else 1 / 4)
    rows, cols = B * Q * H * qs, B * K * G * ks
    if c["kind"] == "attend":
        joined = rows * (D * 4 + 4) if c["join"] else 0
        return {"bytes": rows * (2 * D * size + 4) + 2 * cols * D * size + joined, "flops": 4 * D * H * pairs}
    joined = (rows + 2 * cols) * D * 4 if c["join"] else 0
    return {"bytes": rows * (4 * D * size + 4) + 4 * cols * D * size + joined, "flops": 10 * D * H * pairs}


# ------------------------------------------------------------------------------------------------ 64-bit results
def _exact_rotary(c, seed):
    """A turn is a product of complex numbers."""
    q, k, positions = _rotary_inputs(c, seed)
    if positions is None:
        positions = (torch.arange(c["tokens"], device="cuda") + c["start"]).expand(c["batch"], -1)
    r, steps = c["turned"], []
    for i in range(r // 2):
        f = math.exp(-2 * i / r * math.log(BASE * FACTOR ** (r / (r - 2)) if c["scaling"] == "ntk" else BASE))
        if c["scaling"] == "linear":
            f /= FACTOR
        elif c["scaling"] == "by_parts":
            turns = ORIGINAL * f / (2 * math.pi)
            part = 0.0 if turns < LOW else 1.0 if turns > HIGH else (turns - LOW) / (HIGH - LOW)
            f = (1 - part) * f / FACTOR + part * f
        steps.append(f)
    angle = positions.double().unsqueeze(-1) * torch.tensor(steps, dtype=torch.float64, device="cuda")
    if c["inverse"]:
        angle = -angle
    turn = torch.polar(torch.full_like(angle, AMPLITUDE if c["scaling"] == "by_parts" else 1.0), angle).unsqueeze(2)

    def one(x):
        y = x.double()
        if c["interleaved"]:
            y[..., :r] = torch.view_as_real(torch.view_as_complex(y[..., :r].reshape(*y.shape[:-1], r // 2, 2).contiguous()) * turn).flatten(-2)
        else:
            z = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * turn
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        return y
    return {"q": one(q), "k": one(k)}


def exact(case, seed):
    """One sequence and one head at a time, over the rows that are there."""
    c = case
    if c["kind"] == "rotary":
        return _exact_rotary(c, seed)
    q, k, v, q_len, kv_len, join, dout = _attention_inputs(c, seed)
    B, Q, H, D = q.shape
    K, G = k.shape[1:3]
    R = H // G
    nq = q_len.tolist() if q_len is not None else [Q] * B
    nk = kv_len.tolist() if kv_len is not None else [K] * B
    if sum(a * b for a, b in zip(nq, nk)) * H * D > 32 * 8192 * 8192 * 128 + 1:
        return None
    f64 = dict(dtype=torch.float64, device="cuda")
    out, lse = torch.zeros(B, Q, H, D, **f64), torch.full((B, H, Q), -math.inf, **f64)
    dq, dk, dv = torch.zeros(B, Q, H, D, **f64), torch.zeros(B, K, G, D, **f64), torch.zeros(B, K, G, D, **f64)
    for b in range(B):
        n, m = nq[b], nk[b]
        if n and m:
            hidden = None
            if c["causal"]:
                shift = m - n if c["offset"] is None else c["offset"]
                hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(shift + 1)
            for h in range(H):
                kh, vh = k[b, :m, h // R].double(), v[b, :m, h // R].double()
                qh = q[b, :n, h].double()
                score = qh @ kh.t() / math.sqrt(D)
                if hidden is not None:
                    score = score.masked_fill(hidden, -math.inf)
                row = torch.logsumexp(score, 1)
                p = torch.exp(score - torch.where(row.isinf(), 0.0, row)[:, None])
                o = p @ vh
                out[b, :n, h], lse[b, h, :n] = o, row
                if c["kind"] == "back":
                    # d(score) = p (g - sum p g) with g = d(out) v^T; that sum is <d(out), out>, of the result as it was handed on
                    do = dout[b, :n, h].double()
                    g = do @ vh.t()
                    dscore = (g - (do * o.to(q.dtype).double()).sum(1, keepdim=True)) * p / math.sqrt(D)
                    dq[b, :n, h] = dscore @ kh
                    dk[b, :m, h // R] += dscore.t() @ qh
                    dv[b, :m, h // R] += p.t() @ do
                del score, p
        if join is not None and c["kind"] == "attend":
            both = torch.logaddexp(lse[b, :, :n], join[1][b, :, :n].double())
            weight = lambda x: torch.exp(x - both).t()[..., None]   # noqa: E731
            out[b, :n] = out[b, :n] * weight(lse[b, :, :n]) + join[0][b, :n].double() * weight(join[1][b, :, :n].double())
            lse[b, :, :n] = both
        if join is not None and c["kind"] == "back":
            dq[b, :n] += join[0][b, :n].double()
            dk[b, :m] += join[1][b, :m].double()
            dv[b, :m] += join[2][b, :m].double()
    if c["kind"] == "attend":
        return {"out": out, "lse": lse}
    return {"dq": dq, "dk": dk, "dv": dv}
