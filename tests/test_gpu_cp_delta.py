"""Gradients of attention where ``delta`` is not what the call's own keys make it: a log-sum-exp that has a gradient of its own, and blocks of keys whose queries' results come from other
blocks as well, with values of other sizes."""
import math
import threading

import pytest

torch = pytest.importorskip("torch")

from cp_reference import check, half_step, visible  # noqa: E402
from test_gpu_cp_calls import Mail, Rank  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def cp():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from nccl_b200 import Communicator, get_unique_id
    from nccl_b200.ops.cp import ContextParallel
    torch.cuda.set_device(0)
    comm = Communicator(1, 0, get_unique_id())
    c = ContextParallel(comm)
    yield c
    torch.cuda.synchronize()
    assert comm.async_error() == 0
    c.destroy()
    comm.destroy()


def randn(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(500 + seed)).to(dtype)


def gradients(dout, q, k, v, lse, delta, causal=False, offset=None, q_lengths=None, kv_lengths=None):
    """{name: (gradient, bound)} in 64 bits, of the numbers as they are given: p = exp(s - lse), ds = p (do.v - delta).

    With 16-bit operands and fp32 sums (2^-23 for each term of a product), a probability is off relatively by `rel`: its score's error, the rounding of the score and of the log-sum-exp
    in units of log 2 (2^-24 of each, and of the constant), 2^-17 for adding the exponent of a scale of up to 2^64, 2^-20 for the exponential. ds is off by what p and
    do.v - delta are, half a step of 16 bits, and in fp16 half of 2^-24 at a scale that brings the most it could be, |do| |v| + |delta|, to 2^14 at least: 2^-39 of that.
    Probabilities are multiples of 2^-39 in fp16."""
    B, Q, H, D = q.shape
    K, G = k.shape[1:3]
    R, scale, u, f16 = H // G, 1 / math.sqrt(D), half_step(q.dtype), q.dtype == F16
    see, there, key_there = visible(B, Q, K, causal, offset, q_lengths, kv_lengths)
    rows = lambda t, m: torch.where(m[:, :, None, None], t.cpu().double(), 0.0).transpose(1, 2)   # noqa: E731
    qd, do = rows(q, there), rows(dout, there)
    kd, vd = (rows(t, key_there).repeat_interleave(R, 1) for t in (k, v))
    lse, delta = lse.cpu().double(), torch.where(there[:, None], delta.cpu().double(), 0.0)
    some = lse > -math.inf
    delta = torch.where(some, delta, 0.0)[..., None]
    lse = torch.where(some, lse, 0.0)[..., None]
    see = see[:, None] & some[..., None]
    p = torch.where(see, torch.exp(qd @ kd.mT * scale - lse), 0.0)
    rel = (qd.abs() @ kd.abs().mT * scale) * (D + 4) * 2.0 ** -23 + lse.abs() * 2.0 ** -22 + 2.0 ** -17 + 2.0 ** -20
    dp, dpabs = do @ vd.mT, do.abs() @ vd.abs().mT
    ds = p * (dp - delta)
    eds = ds.abs() * u + p * (rel * (dp.abs() + delta.abs()) + (D + 2) * 2.0 ** -23 * (dpabs + delta.abs()))
    least = 0.0
    if f16:
        most = lambda t: t.amax(-1).view(B, G, R).amax(-1).repeat_interleave(R, 1)[..., None, None]   # noqa: E731
        eds = eds + see * 2.0 ** -39 * (most(do.norm(dim=-1)) * most(vd.norm(dim=-1)) + most(delta.abs()[..., 0]))
        least = 2.0 ** -40
    over = lambda t: t.reshape(B, G, R, K, D).sum(2).transpose(1, 2)   # the heads that share keys and values   # noqa: E731
    n = Q * R
    return {"dq": ((scale * ds @ kd).transpose(1, 2), (scale * (eds + K * 2.0 ** -23 * ds.abs()) @ kd.abs()).transpose(1, 2)),
            "dk": (over(scale * ds.mT @ qd), over(scale * (eds + n * 2.0 ** -23 * ds.abs()).mT @ qd.abs())),
            "dv": (over(p.mT @ do), over(((u + rel + n * 2.0 ** -23) * p + least * see).mT @ do.abs()))}


def compare(got, want, result):
    """Each value is rounded to fp32 as it leaves the sums, and to `result`."""
    for name, t in zip(("dq", "dk", "dv"), got):
        w, e = want[name]
        assert bool(torch.isfinite(t).all()), name
        check(name, t, w, e + w.abs() * (2.0 ** -23 + half_step(result)) + torch.finfo(result).smallest_normal * half_step(result))


# ------------------------------------------------------------------------------------------------ a gradient of the log-sum-exp
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size", [0.0, 1e-5, 1.0])
@pytest.mark.parametrize("dlse", [2.0 ** -20, 1e-3, 1.0, 100.0, 1e6])
@pytest.mark.parametrize("sizes", [(1, 256, 512, 4, 2, 128), (2, 70, 300, 6, 1, 64), (1, 1, 900, 8, 2, 128)])
def test_a_gradient_of_the_log_sum_exp(cp, dtype, size, dlse, sizes):
    B, Q, K, H, G, D = sizes
    q, k, v = randn(B, Q, H, D, dtype=dtype), randn(B, K, G, D, dtype=dtype, seed=1), randn(B, K, G, D, dtype=dtype, seed=2)
    dout = (randn(B, Q, H, D, seed=3) * size).to(dtype)
    out, lse = cp.attention(q, k, v, causal=True)
    delta = cp.attention_delta(dout, out) - dlse * randn(B, H, Q, seed=4)
    got = cp.attention_backward(dout, q, k, v, None, lse, causal=True, delta=delta, dtype=F32)
    compare(got, gradients(dout, q, k, v, lse, delta, True), F32)


def test_queries_that_see_nothing_have_no_gradient_of_their_log_sum_exp(cp):
    """Whatever is subtracted for a row without keys (a loss of a log-sum-exp of -inf has none) reaches no gradient."""
    B, Q, K, H, G, D = 2, 200, 150, 4, 2, 64
    for dtype in (BF16, F16):
        q, k, v = randn(B, Q, H, D, dtype=dtype), randn(B, K, G, D, dtype=dtype, seed=1), randn(B, K, G, D, dtype=dtype, seed=2)
        dout = randn(B, Q, H, D, dtype=dtype, seed=3)
        out, lse = cp.attention(q, k, v, causal=True, offset=-37)
        assert bool((lse[:, :, :37] == -math.inf).all()) and bool(torch.isfinite(lse[:, :, 37:]).all())
        delta = cp.attention_delta(dout, out)
        want = cp.attention_backward(dout, q, k, v, None, lse, causal=True, offset=-37, delta=delta)
        for junk in (math.nan, math.inf, 1e30):
            bad = delta.clone()
            bad[:, :, :37] = junk
            got = cp.attention_backward(dout, q, k, v, None, lse, causal=True, offset=-37, delta=bad)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ blocks of other sizes
BLOCKS = [(1.0, 1e-3), (1e-3, 1.0), (1.0, 0.0), (0.0, 1.0), (1.0, 1e-3, 0.0)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size", [1e-5, 1.0])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("blocks", BLOCKS)
def test_blocks_with_values_of_other_sizes(cp, dtype, size, D, blocks):
    """What a ring does, a block at a time: results, log-sum-exp and delta are over all keys, the values are one block's. Scores are spread, so that single keys have large shares."""
    B, S, H, G = 1, 256, 4, 2
    n = len(blocks)
    q = (4 * randn(B, S, H, D)).to(dtype)
    k = randn(B, n * S, G, D, dtype=dtype, seed=1)
    v = (randn(B, n * S, G, D, seed=2) * torch.tensor(blocks, device="cuda").repeat_interleave(S)[None, :, None, None]).to(dtype)
    dout = (randn(B, S, H, D, seed=3) * size).to(dtype)
    out, lse = cp.attention(q, k, v)
    delta = cp.attention_delta(dout, out)
    for i in range(n):
        kb, vb = k[:, i * S:(i + 1) * S], v[:, i * S:(i + 1) * S]
        got = cp.attention_backward(dout, q, kb, vb, None, lse, delta=delta, dtype=F32)
        compare(got, gradients(dout, q, kb, vb, lse, delta), F32)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size", [1e-3, 1.0])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("blocks", BLOCKS)
def test_rings_with_values_of_other_sizes(cp, dtype, size, causal, blocks):
    from nccl_b200.parallel.context import ring_attention, ring_attention_backward
    B, S, H, G, D, n = 1, 160, 4, 2, 64, len(blocks)
    q = (4 * randn(B, n * S, H, D)).to(dtype)
    k = randn(B, n * S, G, D, dtype=dtype, seed=1)
    v = (randn(B, n * S, G, D, seed=2) * torch.tensor(blocks, device="cuda").repeat_interleave(S)[None, :, None, None]).to(dtype)
    dout = (randn(B, n * S, H, D, seed=3) * size).to(dtype)
    mail, results, errors = Mail(n), [None] * n, []

    def run(r):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                comm, sl = Rank(mail, r, n, cp.lib), slice(r * S, (r + 1) * S)
                ops = [t[:, sl].transpose(1, 2) for t in (q, k, v)]
                out, lse = ring_attention(comm, *ops, causal=causal, cp=cp, with_lse=True)
                grads = ring_attention_backward(comm, dout[:, sl].transpose(1, 2), *ops, out, lse, causal=causal, cp=cp)
                torch.cuda.current_stream().synchronize()
                results[r] = [t.transpose(1, 2) for t in (out, *grads)] + [lse]
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(r,)) for r in range(n)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    lse = torch.cat([r[4] for r in results], 2)
    out, *got = (torch.cat([r[i] for r in results], 1) for i in range(4))
    # of all blocks at once: no block's scale is smaller than that of the largest values, and the additions in fp32 between blocks are among the 2^-23 for each term
    want = gradients(dout, q, k, v, lse, (dout.cpu().double() * out.cpu().double()).sum(-1).transpose(1, 2), causal, 0 if causal else None)
    compare(got, want, dtype)
