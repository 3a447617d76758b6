"""Calls of ``ContextParallel`` that its documentation allows beyond the plain ones: joined and added results, padding that holds anything, strides, graphs, streams, caches behind 32-bit
offsets, empty tensors, extreme scores and small gradients; and the ring and the Ulysses swap on these kernels."""
import math
import queue
import threading

import pytest

torch = pytest.importorskip("torch")

from cp_reference import Reference, check  # noqa: E402

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


def randn(*shape, dtype=BF16, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(77 + seed)).to(dtype)


def operands(B, Q, K, H, G, D, dtype=BF16, seed=0):
    return randn(B, Q, H, D, dtype=dtype, seed=seed), randn(B, K, G, D, dtype=dtype, seed=seed + 1), randn(B, K, G, D, dtype=dtype, seed=seed + 2)


def lens(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ joined and added
@pytest.mark.parametrize("Q,K", [(1, 3000), (40, 300), (600, 700), (5000, 130)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_join(cp, Q, K, dtype):
    """Every form of the forward pass (few rows, in one part and in several; many rows): results over other keys join, in place too."""
    q, k, v = operands(1, Q, K, 8, 2, 64, dtype)
    join = randn(1, Q, 8, 64, dtype=F32, seed=5), randn(1, 8, Q, dtype=F32, seed=6) + 3
    join[1][:, 0] = -math.inf   # nothing so far
    out, lse = cp.attention(q, k, v, causal=True, join=join)
    ref = Reference(q, k, v, True, join=join)
    check("lse", lse, ref.lse, ref.lse_tol)
    check("out", out, ref.out, ref.out_tol)
    wide = Reference(q, k, v, True, join=join, result=F32)
    mine = join[0].clone(), join[1].clone()
    got = cp.attention(q, k, v, causal=True, join=mine, dtype=F32, out=mine[0], lse=mine[1])
    assert got[0] is mine[0] and torch.equal(mine[1], lse)
    check("out in place", mine[0], wide.out, wide.out_tol)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,Q,K,H,G,D,causal,q_lengths,kv_lengths", [
    (3, 4, 1000, 16, 2, 128, True, (4, 0, 2), (1000, 0, 129)), (2, 32, 300, 1, 1, 64, True, None, (300, 17)), (2, 33, 300, 2, 2, 64, True, None, (300, 17)),
    (2, 6, 260, 15, 3, 40, False, (6, 1), (1, 260)), (40, 1, 2200, 32, 8, 128, True, None, None), (1, 1, 9000, 2, 1, 96, False, None, (8999,)), (4, 1, 5000, 32, 1, 16, True, None, (1, 128, 4097, 4999)),
    (300, 1, 140, 2, 2, 64, True, None, None)])
def test_few_rows(cp, dtype, B, Q, K, H, G, D, causal, q_lengths, kv_lengths):
    q, k, v = operands(B, Q, K, H, G, D, dtype)
    if B == 40:
        kv_lengths = [(i * 977) % (K + 1) for i in range(B)]
    ql, kl = None if q_lengths is None else lens(*q_lengths), None if kv_lengths is None else lens(*kv_lengths)
    rule = dict(causal=causal, q_lengths=ql, kv_lengths=kl)
    got = cp.attention(q, k, v, **rule)
    ref = Reference(q, k, v, causal, None, None, ql, kl)
    check("lse", got[1], ref.lse, ref.lse_tol)
    check("out", got[0], ref.out, ref.out_tol)
    join = randn(B, Q, H, D, dtype=F32, seed=5), randn(B, H, Q, dtype=F32, seed=6)
    for result in (dtype, F32):
        got = cp.attention(q, k, v, join=join, dtype=result, **rule)
        ref = Reference(q, k, v, causal, None, None, ql, kl, join=join, result=result)
        check("lse", got[1], ref.lse, ref.lse_tol)
        check("out", got[0], ref.out, ref.out_tol)


def test_join_of_blocks_is_the_whole(cp):
    """What a ring does: keys in three blocks, the middle one seen in part, the last by no one."""
    q, k, v = operands(2, 300, 900, 6, 3, 96)
    whole = Reference(q, k, v, True, offset=250)
    r = None
    for i in range(3):
        r = cp.attention(q, k[:, 300 * i:300 * i + 300], v[:, 300 * i:300 * i + 300], causal=True, offset=250 - 300 * i, join=r, dtype=F32)
    check("lse", r[1], whole.lse, 4 * whole.lse_tol)
    check("out", r[0], whole.out, whole.out_tol)
    nothing = cp.attention(q, k, v, causal=True, offset=-300)
    assert not nothing[0].any() and bool((nothing[1] == -math.inf).all())


def test_add(cp):
    q, k, v = operands(2, 150, 400, 6, 2, 80)
    dout = randn(2, 150, 6, 80, seed=9)
    out, lse = cp.attention(q, k, v, causal=True, kv_lengths=lens(400, 333), q_lengths=lens(150, 60))
    add = randn(2, 150, 6, 80, dtype=F32, seed=10), randn(2, 400, 2, 80, dtype=F32, seed=11), randn(2, 400, 2, 80, dtype=F32, seed=12)
    rule = dict(causal=True, kv_lengths=lens(400, 333), q_lengths=lens(150, 60))
    for result in (BF16, F32):
        ref = Reference(q, k, v, True, None, None, rule["q_lengths"], rule["kv_lengths"], dout=dout, out=out, result=result, add=add)
        got = cp.attention_backward(dout, q, k, v, out, lse, add=add, dtype=result, **rule)
        for name, t in zip(("dq", "dk", "dv"), got):
            check(name, t, getattr(ref, name), getattr(ref, name + "_tol"))
    mine = [t.clone() for t in add]
    cp.attention_backward(dout, q, k, v, out, lse, add=mine, dtype=F32, dq=mine[0], dk=mine[1], dv=mine[2], **rule)
    assert all(torch.equal(a, b) for a, b in zip(mine, got))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,Q,K,H,G,D", [(1, 1, 1, 1, 1, 8), (1, 3, 500, 8, 2, 128), (2, 200, 70, 4, 4, 64), (1, 1000, 300, 4, 2, 96), (1, 5, 3000, 2, 2, 128)])
def test_small_calls_lose_nothing_inside(cp, dtype, B, Q, K, H, G, D):
    q, k, v = operands(B, Q, K, H, G, D, dtype)
    dout = randn(B, Q, H, D, dtype=dtype, seed=9)
    out, lse = cp.attention(q, k, v, causal=True)
    got = cp.attention_backward(dout, q, k, v, out, lse, causal=True, dtype=F32)
    few = B * G * -(-Q // (128 // (H // G))) * -(-K // 128) <= 64   # products of 128 x 128 (1000 queries on 300 keys are 2 * 16 * 3 = 96: the ordinary bound)
    ref = Reference(q, k, v, True, dout=dout, out=out, result=F32, fine=few)
    for name, t in zip(("dv", "dk", "dq"), got[::-1]):
        check(name, t, getattr(ref, name), getattr(ref, name + "_tol"))


# ------------------------------------------------------------------------------------------------ padding
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("junk", [math.nan, math.inf, "lowest"])
@pytest.mark.parametrize("Q,K,H,G", [(260, 300, 6, 2), (1, 300, 8, 2), (300, 260, 2, 2)])
def test_rows_behind_the_lengths_may_hold_anything(cp, dtype, junk, Q, K, H, G):
    B, D = 4, 72
    junk = torch.finfo(dtype).min if junk == "lowest" else junk
    q, k, v = operands(B, Q, K, H, G, D, dtype)
    dout = randn(B, Q, H, D, dtype=dtype, seed=4)
    ql, kl = lens(Q, max(Q - 131, 1), 0, Q), lens(K - 1, 129, 200, 0)
    rule = dict(causal=True, q_lengths=ql, kv_lengths=kl)

    def filled(with_what):
        ts = [t.clone() for t in (q, k, v, dout)]
        for t, n in zip(ts, (ql, kl, kl, ql)):
            for b in range(B):
                t[b, int(n[b]):] = with_what
        return ts
    got = []
    for what in (0.0, junk):
        a, b, c, d = filled(what)
        out, lse = cp.attention(a, b, c, **rule)
        got.append((out, lse) + cp.attention_backward(d, a, b, c, out, lse, **rule))
    for x, y in zip(*got):
        assert torch.equal(x, y) and not bool(torch.isnan(x).any())
    for b in range(B):
        assert not got[1][0][b, int(ql[b]):].any() and bool((got[1][1][b, :, int(ql[b]):] == -math.inf).all())
        assert not got[1][2][b, int(ql[b]):].any() and not got[1][3][b, int(kl[b]):].any() and not got[1][4][b, int(kl[b]):].any()


def test_lengths_out_of_range_are_taken_as_none_or_all(cp):
    q, k, v = operands(3, 20, 30, 2, 1, 32)
    a = cp.attention(q, k, v, q_lengths=lens(-5, 20, 99), kv_lengths=lens(30, 31, -1))
    b = cp.attention(q, k, v, q_lengths=lens(0, 20, 20), kv_lengths=lens(30, 30, 0))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("sizes", [(0, 5, 5), (2, 0, 5), (2, 5, 0), (2, 0, 0)])
def test_without_rows(cp, sizes):
    B, Q, K = sizes
    q, k, v = operands(B, Q, K, 4, 2, 16)
    out, lse = cp.attention(q, k, v, causal=True)
    assert out.shape == q.shape and not out.any() and bool((lse == -math.inf).all())
    add = torch.ones(q.shape, device="cuda"), torch.ones(k.shape, device="cuda"), torch.ones(k.shape, device="cuda")
    for a in (None, add):
        for g, t in zip(cp.attention_backward(q, q, k, v, out, lse, causal=True, add=a), (q, k, v)):
            assert g.shape == t.shape and bool((g == (0.0 if a is None else 1.0)).all())
    assert cp.attention_delta(q, out).shape == lse.shape


# ------------------------------------------------------------------------------------------------ values
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_that_climb(cp, dtype):
    """Each tile of keys brings larger scores than all before: the running maximum is raised again and again."""
    q, k, v = operands(1, 140, 1500, 2, 1, 128, dtype)
    q = (q.abs() * 0.5).to(dtype)
    k = (k.abs() * torch.linspace(0.1, 4, 1500, device="cuda")[None, :, None, None]).to(dtype)
    out, lse = cp.attention(q, k, v)
    ref = Reference(q, k, v)
    check("lse", lse, ref.lse, ref.lse_tol)
    check("out", out, ref.out, ref.out_tol)
    flipped = cp.attention(q, k.flip(1), v.flip(1))
    check("falling", flipped[0], ref.out, ref.out_tol)


def test_not_a_number_stays_in_its_row(cp):
    q, k, v = operands(1, 300, 500, 4, 2, 64)
    want = cp.attention(q, k, v)
    q[0, 17, 1] = math.nan
    out, lse = cp.attention(q, k, v)
    assert bool(torch.isnan(out[0, 17, 1]).all()) and bool(torch.isnan(lse[0, 1, 17]))
    out[0, 17, 1], lse[0, 1, 17] = want[0][0, 17, 1], want[1][0, 1, 17]
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("size", [2.0 ** -24, 2.0 ** -12, 2.0 ** 8])
def test_fp16_gradients_of_any_size(cp, size):
    """Products inside are scaled by what the largest could be: small gradients do not vanish, large ones do not overflow."""
    q, k, v = operands(1, 400, 700, 4, 2, 64, F16)
    dout = (randn(1, 400, 4, 64, dtype=F32, seed=8) * size).half()
    out, lse = cp.attention(q, k, v)
    got = cp.attention_backward(dout, q, k, v, out, lse, dtype=F32)
    ref = Reference(q, k, v, dout=dout, out=out, result=F32)
    for name, t in zip(("dq", "dk", "dv"), got):
        check(name, t, getattr(ref, name), getattr(ref, name + "_tol"))


def test_gradients_against_differences(cp):
    """Along a random direction of each operand: the change of <dout, attention> in 64 bits, to the second order of the step and the bounds of the gradients."""
    q, k, v = operands(1, 70, 90, 4, 2, 32)
    dout = randn(1, 70, 4, 32, seed=8)
    out, lse = cp.attention(q, k, v, causal=True)
    got = cp.attention_backward(dout, q, k, v, out, lse, causal=True, dtype=F32)
    ref = Reference(q, k, v, True, dout=dout, out=out, result=F32)
    eps = 2.0 ** -12

    class Wide:   # an operand in 64 bits that says it is bf16, for the bounds that are not looked at here
        def __init__(self, t):
            self.t, self.shape, self.dtype = t, t.shape, BF16

        def detach(self):
            return self.t

    def loss(ops):
        return float((Reference(*[Wide(t) for t in ops], True).out * dout.cpu().double()).sum())
    base = [t.cpu().double() for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        step = torch.randn(base[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        value = lambda e: loss([t + e * step if j == i else t for j, t in enumerate(base)])   # noqa: E731
        first, second = (value(eps) - value(-eps)) / (2 * eps), (value(2 * eps) - value(-2 * eps)) / (4 * eps)
        bound = float((getattr(ref, name + "_tol") * step.abs()).sum()) + 2 * abs(second - first)
        # (the result that the gradient was given is rounded to bf16, the differences' is not: through <dout, out>, by half a step of each value)
        if name != "dv":
            inner = (dout.cpu().double().abs() * out.cpu().double().abs()).sum(-1).transpose(1, 2)[..., None] * 2.0 ** -8
            s = torch.exp((base[0].transpose(1, 2) @ base[1].transpose(1, 2).repeat_interleave(2, 1).mT) / math.sqrt(32) - ref.lse[..., None]).clamp_max(1.0)
            other = base[1].transpose(1, 2).repeat_interleave(2, 1) if name == "dq" else base[0].transpose(1, 2)
            push = (s * inner) @ other.abs() if name == "dq" else ((s * inner).mT @ other.abs()).view(1, 2, 2, 90, 32).sum(2)
            bound += float((push.transpose(1, 2) * step.abs()).sum()) / math.sqrt(32)
        assert abs(float((got[i].cpu().double() * step).sum()) - first) <= bound, name


# ------------------------------------------------------------------------------------------------ layouts
def test_strides(cp):
    """Heads in front of tokens, slices of one projection, a batch with gaps: the same bits as contiguous tensors give."""
    B, S, H, G, D = 2, 333, 6, 2, 64
    x = randn(B + 1, S + 3, H + 2 * G, D)[1:, 2:-1]
    q, k, v = x.split((H, G, G), dim=2)
    c = [t.contiguous() for t in (q, k, v)]
    dout = randn(B, S, H, D, seed=3)
    want = cp.attention(*c, causal=True)
    wants = cp.attention_backward(dout, *c, *want, causal=True)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, dout, want[0])]
    for ops, d, o in (((q, k, v), dout, want[0]), (heads_first[:3], heads_first[3], heads_first[4])):
        got = cp.attention(*ops, causal=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(torch.equal(a, b) for a, b in zip(cp.attention_backward(d, *ops, o, want[1], causal=True), wants))
    one = cp.attention(q[:1, :1], k[:1], v[:1])   # (sizes of one: strides say nothing)
    assert torch.equal(one[0], cp.attention(c[0][:1, :1], c[1][:1], c[2][:1])[0])


def test_a_cache_behind_32_bits(cp):
    """Keys and values of the second sequence lie more than 2^32 bytes, and 2^31 elements, behind the first one's."""
    far = (1 << 31) + 4096
    pool = torch.empty(far + 2 * 700 * 2 * 64, dtype=BF16, device="cuda")
    k = pool.as_strided((2, 700, 2, 64), (far, 128, 64, 1))
    v = pool.as_strided((2, 700, 2, 64), (far, 128, 64, 1), 700 * 128)
    q, kc, vc = operands(2, 3, 700, 8, 2, 64)
    k.copy_(kc)
    v.copy_(vc)
    dout = randn(2, 3, 8, 64, seed=3)
    out, lse = cp.attention(q, k, v, causal=True)
    want = cp.attention(q, kc, vc, causal=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert all(torch.equal(a, b) for a, b in zip(cp.attention_backward(dout, q, k, v, out, lse, causal=True), cp.attention_backward(dout, q, kc, vc, out, lse, causal=True)))


def test_outputs_that_share_memory_are_refused(cp):
    from nccl_b200._lib import NcclError
    q, k, v = operands(1, 64, 64, 4, 4, 64)
    out, lse = cp.attention(q, k, v)
    flat = torch.zeros(64 * 4 * 64 + 8, device="cuda")
    join = flat[:-8].view(1, 64, 4, 64), lse.clone()
    for kw in (dict(out=q), dict(out=k), dict(out=v), dict(join=join, out=flat[:64 * 4 * 32].view(BF16).view(1, 64, 4, 64)), dict(join=join, dtype=F32, out=flat[8:].view(1, 64, 4, 64))):
        with pytest.raises(NcclError):
            cp.attention(q, k, v, **kw)
    for kw in (dict(dq=q), dict(dk=v), dict(dq=out), dict(dk=torch.empty_like(k), dv=None, dq=k)):
        with pytest.raises(NcclError):
            cp.attention_backward(out.clone(), q, k, v, out, lse, **kw)
    g = torch.empty_like(k)
    with pytest.raises(NcclError):
        cp.attention_backward(out.clone(), q, k, v, out, lse, dk=g, dv=g)
    freqs = cp.rotary_frequencies(64)
    big = randn(1, 65, 4, 64)
    with pytest.raises(NcclError):
        cp.rotary(big[:, :64], None, freqs, out=(big[:, 1:], None))
    with pytest.raises(NcclError):
        cp.rotary(q, k, freqs, out=(k, q))
    torch.cuda.synchronize()


def test_turned_in_place(cp):
    from nccl_b200._lib import NcclError
    freqs = cp.rotary_frequencies(64)

    def layouts():   # a storage, and two tensors in it whose rows lie between one another
        x = randn(2, 9, 6, 64)
        yield x, x[:, :, :4], x[:, :, 4:]
        yield x, x[:, :, ::2], x[:, :, 1::2]
        x = randn(2, 6, 9, 64).transpose(1, 2)
        yield x, x[:, :, 2:], x[:, :, :2]
        x = randn(9, 2, 6, 64).transpose(0, 1)
        yield x, x[:, :, :3], x[:, :, 3:]
    for x, q, k in layouts():
        wq, wk = cp.rotary(q.clone(), k.clone(), freqs, offset=5)
        before = x.clone()
        aside = torch.empty(k.shape, device="cuda", dtype=k.dtype)
        cp.rotary(q, k, freqs, offset=5, out=(q, aside))   # the other only read
        assert torch.equal(q, wq) and torch.equal(aside, wk)
        x.copy_(before)
        cp.rotary(q, k, freqs, offset=5, out=(q, k))
        assert torch.equal(q, wq) and torch.equal(k, wk)
    x, y = randn(1, 9, 6, 64), randn(1, 9, 6, 64)
    for q, k, out in ((x, x, (x, x)), (x, x, (x, y)), (x, x, (y, x)), (x[:, :, :4], x[:, :, 3:], (x[:, :, :4], x[:, :, 3:])), (x[:, :5], x[:, 4:], (x[:, :5], x[:, 4:])),
                      (x, y, (x, x.as_strided(x.shape, (0, 128, 64, 1))))):
        with pytest.raises(NcclError):
            cp.rotary(q, k, freqs, out=out)


def test_numbers_in_tensors_are_read_by_every_call(cp):
    q, k, v = operands(1, 40, 90, 2, 2, 64)
    scale, offset = torch.tensor(0.5), torch.tensor(3)
    for s, o in ((0.5, 3), (0.25, 40)):
        scale.fill_(s)
        offset.fill_(o)
        got, want = cp.attention(q, k, v, causal=True, offset=offset, scale=scale), cp.attention(q, k, v, causal=True, offset=o, scale=s)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(TypeError):
        cp.attention(q, k, v, causal=True, offset=2.5)


# ------------------------------------------------------------------------------------------------ graphs, streams, threads
def test_graphs_and_streams(cp):
    """Two captured calls with workspaces of their own, replayed in turn with new inputs, beside eager ones on another stream."""
    shapes = [(1, 1, 3000, 8, 2, 64), (2, 200, 333, 4, 2, 96)]
    graphs = []
    for i, s in enumerate(shapes):
        q, k, v = operands(*s, F16, seed=20 + i)
        d = randn(*q.shape, dtype=F16, seed=30 + i)
        cp.attention_backward(d, q, k, v, *cp.attention(q, k, v, causal=True), causal=True)   # (warm)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, lse = cp.attention(q, k, v, causal=True)
            grads = cp.attention_backward(d, q, k, v, out, lse, causal=True)
        graphs.append((g, (q, k, v, d), (out, lse) + grads))
    for turn in range(3):
        side = torch.cuda.Stream()
        for i, (g, ins, outs) in enumerate(graphs):
            for t in ins:
                t.copy_(randn(*t.shape, dtype=F16, seed=100 * turn + i))
        for g, _, _ in graphs:
            g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = []
            for _, (q, k, v, d), _ in graphs:
                out, lse = cp.attention(q, k, v, causal=True)
                again.append((out, lse) + cp.attention_backward(d, q, k, v, out, lse, causal=True))
        torch.cuda.synchronize()
        for (_, _, outs), want in zip(graphs, again):
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_threads(cp):
    """Calls of several host threads on streams of their own."""
    ins = [operands(1, 300 + 8 * i, 500, 4, 2, 64, seed=40 + i) for i in range(4)]
    want = [cp.attention(*t, causal=True) for t in ins]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = cp.attention(*ins[i], causal=True)
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------------ the recipes
class Mail:
    """Stands for the network between ranks that are threads of this process: copies in stream order. No kernel waits for another rank."""

    def __init__(self, n):
        self.box = {(a, b): queue.Queue() for a in range(n) for b in range(n)}


class Rank:
    def __init__(self, mail, rank, nranks, lib):
        self.mail, self.rank, self.nranks, self.lib = mail, rank, nranks, lib

    def _on(self, stream):
        return stream if stream is not None else torch.cuda.current_stream()

    def send(self, t, peer, stream=None):
        with torch.cuda.stream(self._on(stream)):
            e = torch.cuda.Event()
            c = t.clone()
            e.record()
        self.mail.box[self.rank, peer].put((c, e))

    def recv(self, t, peer, stream=None):
        c, e = self.mail.box[peer, self.rank].get(timeout=60)
        with torch.cuda.stream(self._on(stream)):
            torch.cuda.current_stream().wait_event(e)
            t.copy_(c)
        c.record_stream(self._on(stream))

    def all_to_all(self, send, recv, stream=None):
        for p in range(self.nranks):
            self.send(send.view(self.nranks, -1)[p], p, stream)
        for p in range(self.nranks):
            self.recv(recv.view(self.nranks, -1)[p], p, stream)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n", [1, 2, 3])
def test_ring_and_ulysses(cp, n, causal):
    """Rotary positions, attention and gradients of a sequence that n ranks share, against 64 bits over the whole of it."""
    from nccl_b200.parallel.context import ring_attention, ring_attention_backward, ulysses_attention, ulysses_attention_backward
    B, S, H, G, D = 2, 160, 6, 3, 64
    q, k, v = operands(B, S * n, S * n, H, G, D, seed=60)
    dout = randn(B, S * n, H, D, seed=66)
    freqs = cp.rotary_frequencies(D)
    tq, tk = cp.rotary(q, k, freqs)
    mail, results, errors = Mail(n), [None] * n, []

    def run(r):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                comm, sl = Rank(mail, r, n, cp.lib), slice(r * S, (r + 1) * S)
                mine = cp.rotary(q[:, sl], k[:, sl], freqs, offset=r * S)
                assert torch.equal(mine[0], tq[:, sl]) and torch.equal(mine[1], tk[:, sl])
                ops = [t.transpose(1, 2) for t in (*mine, v[:, sl])]
                d = dout[:, sl].transpose(1, 2)
                out, lse = ring_attention(comm, *ops, causal=causal, cp=cp, with_lse=True)
                ring = ring_attention_backward(comm, d, *ops, out, lse, causal=causal, cp=cp)
                res = [[t.transpose(1, 2) for t in (out, *ring)], lse]
                if H % n == 0 and G % n == 0:
                    o, state = ulysses_attention(comm, *[t.contiguous() for t in (*mine, v[:, sl])], causal=causal, cp=cp, with_state=True)
                    res.append([o, *ulysses_attention_backward(comm, dout[:, sl].contiguous(), state, causal=causal, cp=cp)])
                torch.cuda.current_stream().synchronize()
                results[r] = res
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(r,)) for r in range(n)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    out = torch.cat([r[0][0] for r in results], 1)
    ref = Reference(tq, tk, v, causal, 0 if causal else None, dout=dout, out=out)
    check("lse", torch.cat([r[1] for r in results], 2), ref.lse, 2 * n * ref.lse_tol)
    for which in (0, 2):
        if len(results[0]) <= which:
            continue
        for i, name in enumerate(("out", "dq", "dk", "dv")):
            # fp32 partial results are added up to n times, each time rounded (2^-24 of the sums, which the bounds' own 2^-23 of magnitudes covers)
            check(name, torch.cat([r[which][i] for r in results], 1), getattr(ref, name), getattr(ref, name + "_tol"))
