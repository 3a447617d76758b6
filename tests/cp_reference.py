"""Attention and its gradients in 64 bits by their formulas, and how far rounding may take a result from them."""
import math

import torch


def visible(B, Q, K, causal, offset, q_lengths, kv_lengths):
    """[B, Q, K]: whether a query sees a key; [B, Q], [B, K]: whether they are there."""
    i, j = torch.arange(Q)[None, :, None], torch.arange(K)[None, None, :]
    nq = torch.full((B,), Q) if q_lengths is None else q_lengths.cpu().long().clamp(0, Q)
    nk = torch.full((B,), K) if kv_lengths is None else kv_lengths.cpu().long().clamp(0, K)
    see = (i < nq[:, None, None]) & (j < nk[:, None, None])
    if causal:
        off = (nk - nq)[:, None, None] if offset is None else offset
        see = see & (j <= i + off)
    return see, torch.arange(Q)[None] < nq[:, None], torch.arange(K)[None] < nk[:, None]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Reference:
    """out, lse, and with `dout` dq, dk, dv, as fp64 tensors on the CPU, and for each a bound on the error of 16-bit operands with fp32 sums.

    A product's sum of n terms in fp32 is off by at most n * 2^-23 of the sum of their magnitudes (2^-23: the tensor cores may cut off instead of rounding). An
    exponential of a score is off relatively by the score's error, plus 2^-20 for the exponent's rounding and the function. A rounding to 16 bits is off by half a
    step, `u`: one for the probabilities (or ds), one for the result; or by half of the smallest step there is. In fp16 that one matters inside too: probabilities of the forward
    pass are held as multiples of 2^-24 of a largest one of at least 2^-1 (2^7 over the lag of 2^8), those of the backward pass as multiples of 2^-39, and ds as
    multiples of 2^-24 where the largest that could be, 2 |do| |v|, is 2^14 at least."""

    def __init__(self, q, k, v, causal=False, offset=None, scale=None, q_lengths=None, kv_lengths=None, join=None, dout=None, out=None, result=None, add=None, fine=False):
        B, Q, H, D = q.shape
        K, G = k.shape[1:3]
        R = H // G
        scale = 1 / math.sqrt(D) if scale is None else scale
        u = half_step(q.dtype)
        inner = u * u if fine else u   # with "fine" products, what the first rounding of probabilities and ds left is rounded and counted too
        ur = half_step(result or q.dtype)
        tiny = torch.finfo(result or q.dtype).smallest_normal * ur
        f16 = q.dtype == torch.float16
        see, there, key_there = visible(B, Q, K, causal, offset, q_lengths, kv_lengths)
        clear = lambda t, m: torch.where(m[:, :, None, None], t.detach().cpu().double(), torch.zeros((), dtype=torch.float64))   # noqa: E731
        qd, kd, vd = clear(q, there).transpose(1, 2), clear(k, key_there).transpose(1, 2).repeat_interleave(R, 1), clear(v, key_there).transpose(1, 2).repeat_interleave(R, 1)
        s = (qd @ kd.mT * scale).masked_fill(~see[:, None], -math.inf)
        lse = torch.logsumexp(s, -1)
        some = lse > -math.inf
        p = torch.where(see[:, None], torch.exp(s - torch.where(some, lse, 0.0)[..., None]), 0.0)
        # relative error of a probability: of its score, of the log-sum-exp (or maximum and sum) it is divided by
        sabs = (qd.abs() @ kd.abs().mT * scale).masked_fill(~see[:, None], 0.0)
        worst = sabs.amax(-1, keepdim=True) if K else torch.zeros(B, H, Q, 1, dtype=torch.float64)
        rel = 2 * (worst * (D + 4) * 2.0 ** -23 + 2.0 ** -20 + K * 2.0 ** -24)
        o = p @ vd
        oabs = p @ vd.abs()
        vmax = vd.abs().amax(-2, keepdim=True) if K else torch.zeros(B, H, 1, D, dtype=torch.float64)
        e = oabs * (u + rel + K * 2.0 ** -23) + (K * 2.0 ** -24 * vmax if f16 else 0.0)
        self.lse, self.lse_tol = lse, rel[..., 0] + torch.where(some, lse.abs(), 0.0) * 2.0 ** -22
        if join is not None:
            o0, l0 = clear(join[0], there).transpose(1, 2), torch.where(there[:, None], join[1].cpu().double(), -math.inf)
            both = torch.logaddexp(lse, l0)
            w = lambda x: torch.where(both > -math.inf, torch.exp(x - torch.where(both > -math.inf, both, 0.0)), 0.0)[..., None]   # noqa: E731
            moved = rel + 2.0 ** -20 * (1 + torch.where(some, lse.abs(), 0.0) + torch.where(l0 > -math.inf, l0.abs(), 0.0))[..., None]   # relative error of a weight
            e = e * w(lse) + (o.abs() * w(lse) + o0.abs() * w(l0)) * moved
            o = o * w(lse) + o0 * w(l0)
            self.lse, self.lse_tol = both, moved[..., 0] + torch.where(both > -math.inf, both.abs(), 0.0) * 2.0 ** -22
        self.out = o.transpose(1, 2)
        self.out_tol = (e + o.abs() * ur + tiny).transpose(1, 2)
        if dout is None:
            return
        do = clear(dout, there).transpose(1, 2)
        od = clear(out, there).transpose(1, 2) if out is not None else p @ vd
        delta = (do * od).sum(-1, keepdim=True)
        dp = do @ vd.mT
        ds = p * (dp - delta)
        # of ds: its rounding, the probability's relative error, and the errors of dp and delta
        eds = ds.abs() * inner + p * (rel * (dp.abs() + delta.abs()) + D * 2.0 ** -23 * (do.abs() @ vd.abs().mT + (do.abs() * od.abs()).sum(-1, keepdim=True)))
        least = 0.0
        if f16:
            norm = lambda t: t.norm(dim=-1).amax(-1).view(B, G, R).amax(-1).repeat_interleave(R, 1)[..., None, None]   # noqa: E731
            least = 2.0 ** -25
            eds = eds + see[:, None] * 2.0 ** -38 * 2 * norm(do) * norm(vd) if K and Q else eds
        over = lambda t: t.reshape(B, G, R, K, D).sum(2).transpose(1, 2)   # the heads that share keys and values   # noqa: E731
        base = [torch.zeros((), dtype=torch.float64)] * 3 if add is None else [clear(a, m) for a, m in zip(add, (there, key_there, key_there))]

        def bound(t, a, e):   # the result's rounding (and of what it is added to)
            return t + a, e + (t + a).abs() * ur + (t.abs() + a.abs()) * 2.0 ** -23 + tiny
        self.dq, self.dq_tol = bound((scale * ds @ kd).transpose(1, 2), base[0], (scale * (eds + K * 2.0 ** -23 * ds.abs()) @ kd.abs()).transpose(1, 2))
        n = Q * R
        self.dk, self.dk_tol = bound(over(scale * ds.mT @ qd), base[1], over(scale * (eds + n * 2.0 ** -23 * ds.abs()).mT @ qd.abs()))
        self.dv, self.dv_tol = bound(over(p.mT @ do), base[2], over(((inner + rel + n * 2.0 ** -23) * p + least * 2.0 ** -15 * see[:, None]).mT @ do.abs()))


def check(name, got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    same = torch.where(torch.isfinite(want), (got - want).abs() <= tol, got == want)
    if not bool(same.all()):
        at = (~same).nonzero()[0].tolist()
        worst = ((got - want).abs() / tol).nan_to_num(nan=math.inf)[~same].max()
        raise AssertionError("%s: %d of %d values are off, first at %s: %r, not %r +- %.3g; worst %.3g times the bound" % (
            name, int((~same).sum()), same.numel(), at, float(got[tuple(at)]), float(want[tuple(at)]), float(tol.expand_as(want)[tuple(at)]), float(worst)))


def rotary(x, at, turns, amplitude=1.0, interleaved=False, inverse=False):
    """x [B, T, H, D] with its first 2 * len(turns) channels turned, in 64 bits; at [B, T]."""
    y, half = x.detach().cpu().double().clone(), len(turns)
    # a whole number of turns is nothing: what is left is exact to 2^-52 of the product
    part = torch.remainder(at.cpu().double()[..., None] * torch.tensor(turns, dtype=torch.float64), 1.0)
    angle = 2 * math.pi * part * (-1 if inverse else 1)
    c, s = (amplitude * f(angle)[:, :, None] for f in (torch.cos, torch.sin))
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y
