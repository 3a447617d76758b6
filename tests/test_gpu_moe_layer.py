"""Gradients across the exchange, and a whole mixture-of-experts layer there and back, against 64-bit references."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

HALF, U32 = 2.0 ** -8, 2.0 ** -24   # half a unit in the last place of bf16 and fp32, relative


@pytest.fixture(scope="module")
def comm():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from nccl_b200 import Communicator, get_unique_id
    torch.cuda.set_device(0)
    c = Communicator(1, 0, get_unique_id())
    yield c
    torch.cuda.synchronize()
    assert c.async_error() == 0
    c.destroy()


def routing(T, E, K, drop, g):
    idx = torch.rand(T, E, device="cuda", generator=g).topk(K, dim=1).indices
    if drop:
        idx = torch.where(torch.rand(T, K, device="cuda", generator=g) < drop, torch.full_like(idx, -1), idx)
    return idx.contiguous()


@pytest.mark.parametrize("T,cap,E,K,H,drop", [(1, 1, 1, 1, 128, 0.0), (5, 9, 256, 8, 640, 0.2), (64, 64, 32, 16, 1024, 0.0), (131, 140, 8, 3, 384, 0.1), (700, 800, 16, 9, 256, 1.0),
                                              (3000, 3000, 4, 2, 128, 0.3)])
def test_gradients_of_dispatch_and_combine(comm, T, cap, E, K, H, drop):
    from nccl_b200.ops.ep import ExpertParallel
    ep = ExpertParallel(comm, E, cap, H)
    g = torch.Generator(device="cuda").manual_seed(T + K)
    for turn in range(2):   # the second dispatch finds the records of the first
        x, idx, w = torch.randn(T, H, device="cuda", generator=g).bfloat16(), routing(T, E, K, drop, g), torch.rand(T, K, device="cuda", generator=g)
        toks, _, counts = ep.dispatch(x, idx, w, fp8=False, send_only=turn == 1)
        if turn == 1:
            with pytest.raises(Exception):
                ep.dispatch_rows()   # the rows are still on their way
            ep.complete()
        rows = ep.dispatch_rows()
        assert torch.equal(rows >= 0, idx >= 0)
        on = rows >= 0
        assert torch.equal(toks.view(-1, H)[rows[on].long()], x[:, None].expand(T, K, H)[on])
        assert torch.equal(rows[on].long() // cap, idx[on]) and rows[on].unique().numel() == int(on.sum())

        y = torch.randn(E, cap, H, device="cuda", generator=g).bfloat16()
        y.view(-1, H)[torch.ones(E * cap, dtype=torch.bool, device="cuda").index_fill_(0, rows[on].long(), False)] = math.nan   # rows of nobody
        dout = torch.randn(T, H, device="cuda", generator=g).bfloat16()
        dy = torch.full_like(y, 77.0)
        got, dw = ep.combine_backward(dout, y, w, rows, dy=dy)
        assert got is dy
        want = (w[..., None].double() * dout[:, None].double())[on]
        named = rows[on].long()
        # one product in fp32 (half a unit) and a rounding to bf16
        assert ((dy.view(-1, H)[named].double() - want).abs() <= (HALF + 2 * U32) * want.abs() + 1e-39).all()
        rest = torch.ones(E * cap, dtype=torch.bool, device="cuda").index_fill_(0, named, False)
        assert (dy.view(-1, H)[rest] == 77.0).all()
        terms = torch.zeros(T, K, H, dtype=torch.float64, device="cuda")
        terms[on] = y.view(-1, H)[named].double() * dout[:, None].expand(T, K, H)[on].double()
        # H products and additions in fp32: H units at most of the sum of what is added
        assert ((dw.double() - terms.sum(2)).abs() <= (H + 2) * U32 * terms.abs().sum(2)).all()
        again = ep.combine_backward(dout, y, w, rows)
        assert torch.equal(again[1], dw) and torch.equal(again[0].view(-1, H)[named], dy.view(-1, H)[named])
        place = y.clone()
        assert ep.combine_backward(dout, place, w, rows, dy=place)[0] is place   # the gradients in the rows' place
        assert torch.equal(place.view(-1, H)[named], dy.view(-1, H)[named])

        dtoks = torch.randn(E, cap, H, device="cuda", generator=g).bfloat16()
        dx = ep.dispatch_backward(dtoks, rows)
        back = torch.zeros(T, K, H, dtype=torch.float64, device="cuda")
        back[on] = dtoks.view(-1, H)[named].double()
        ref = back.sum(1)
        assert ((dx.double() - ref).abs() <= HALF * ref.abs() + 2 * K * U32 * back.abs().sum(1)).all()
    ep.destroy()


def test_rows_of_entries_that_dispatch_left_out(comm):
    """A token that names an expert twice takes two rows; what goes beyond the capacity has none."""
    from nccl_b200.ops.ep import ExpertParallel
    ep = ExpertParallel(comm, 4, 16, 256)
    x, w = torch.randn(16, 256, device="cuda").bfloat16(), torch.rand(16, 2, device="cuda")
    idx = torch.zeros(16, 2, dtype=torch.int64, device="cuda")   # 32 entries for the 16 rows of expert 0
    ep.dispatch(x, idx, w, fp8=False)
    rows = ep.dispatch_rows()
    on = rows >= 0
    assert int(on.sum()) == 16 and rows[on].unique().numel() == 16 and int(rows.max()) == 15
    idx = torch.full((16, 2), -1, dtype=torch.int64, device="cuda")
    ep.dispatch(x, idx, w, fp8=False)
    assert (ep.dispatch_rows() == -1).all()
    ep.destroy()


def test_rows_that_name_nothing(comm):
    """Row numbers outside the tensor are as good as none."""
    from nccl_b200.ops.ep import ExpertParallel
    ep = ExpertParallel(comm, 4, 16, 128)
    dout, y, w = torch.randn(2, 128, device="cuda").bfloat16(), torch.randn(6, 128, device="cuda").bfloat16(), torch.rand(2, 3, device="cuda")
    rows = torch.tensor([[-1, 6, 2], [1 << 30, -(1 << 31), 5]], dtype=torch.int32, device="cuda")
    dy = torch.zeros_like(y)
    _, dw = ep.combine_backward(dout, y, w, rows, dy=dy)
    assert (dw[:, :2] == 0).all() and (dy[[0, 1, 3, 4]] == 0).all() and (dw[:, 2] != 0).all()
    assert torch.equal(ep.dispatch_backward(y, rows), y[[2, 5]])
    assert (ep.dispatch_backward(y[:0], rows) == 0).all()
    ep.destroy()


def _layer(comm, T, cap, H, F, E, K, score, seed):
    from nccl_b200.ops.ep import ExpertParallel
    ep = ExpertParallel(comm, E, cap, H)
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    gate = (torch.randn(E, H, device="cuda", generator=g) / math.sqrt(H)).float()
    w1 = (torch.randn(E, 2 * F, H, device="cuda", generator=g) / math.sqrt(H)).bfloat16()
    w2 = (torch.randn(E, H, F, device="cuda", generator=g) / math.sqrt(F)).bfloat16()
    bias = 0.1 * torch.randn(E, device="cuda", generator=g)
    dout = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    rule = dict(score=score, scale=2.0)
    b16 = dict(dtype=torch.bfloat16, device="cuda")
    buf = {"toks": torch.zeros(E, cap, H, **b16), "pre": torch.zeros(E, cap, 2 * F, **b16), "act": torch.zeros(E, cap, F, **b16), "y": torch.zeros(E, cap, H, **b16)}

    def step():
        logits = x.float() @ gate.T
        idx, w = ep.route(logits, K, bias=bias, groups=2, keep_groups=1, group_score="top2", **rule)
        toks, _, counts = ep.dispatch(x, idx, w, fp8=False, toks=buf["toks"])
        act = ep.expert_linear(toks, w1, counts, activation="swiglu", out=buf["act"], pre=buf["pre"])
        y = ep.expert_linear(act, w2, counts, out=buf["y"])
        out = ep.combine(y)
        rows = ep.dispatch_rows()
        dy, dw = ep.combine_backward(dout, y, w, rows)
        dact, dw2, _ = ep.expert_linear_backward(dy, act, w2, counts)
        dtoks, dw1, _ = ep.expert_linear_backward(dact, toks, w1, counts, pre=buf["pre"], activation="swiglu")
        dx = ep.dispatch_backward(dtoks, rows)
        return {"out": out, "dx": dx, "dw1": dw1, "dw2": dw2, "dlogits": ep.route_backward(dw, logits, idx, **rule), "idx": idx, "logits": logits}

    def reference(idx):
        xd, w1d, w2d = (t.double().requires_grad_(True) for t in (x, w1, w2))
        l = (x.float() @ gate.T).double().requires_grad_(True)
        s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
        wk = s.gather(1, idx)
        wk = 2.0 * wk / wk.sum(1, keepdim=True)
        out = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        for e in range(E):
            t, k = torch.nonzero(idx == e, as_tuple=True)
            z = xd[t] @ w1d[e].T
            y = (torch.nn.functional.silu(z[:, :F]) * z[:, F:]) @ w2d[e].T
            out = out.index_add(0, t, wk[t, k, None] * y)
        grads = torch.autograd.grad((out * dout.double()).sum(), (xd, w1d, w2d, l))
        return dict(zip(("out", "dx", "dw1", "dw2", "dlogits"), (out.detach(),) + grads))

    return ep, step, reference


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,cap,H,F,E,K", [(1, 1, 128, 64, 4, 2), (300, 320, 256, 176, 8, 3), (1000, 1000, 640, 384, 6, 2)])
def test_layer_there_and_back(comm, T, cap, H, F, E, K, score):
    ep, step, reference = _layer(comm, T, cap, H, F, E, K, score, T)
    got = step()
    want = reference(got["idx"])
    for name in ("out", "dx", "dw1", "dw2", "dlogits"):
        # every tensor on the way (six to bf16 at most) is rounded by up to 2^-8 of itself: independent errors of a third of that in
        # the mean square, over norms that the products carry on. The whole must stay below the sum of their largest.
        far = (got[name].double() - want[name]).norm() / want[name].norm()
        assert far <= 6 * HALF, (name, float(far))
    ep.destroy()


def test_captured_layer(comm):
    """The whole step in a graph, beside an eager step of another layer: the same sums up to the order of dispatch's rows."""
    ep, step, reference = _layer(comm, 200, 200, 256, 128, 4, 2, "softmax", 1)
    other, step2, _ = _layer(comm, 100, 128, 128, 64, 8, 2, "sigmoid", 2)
    eager = step()
    before = step2()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        graph.replay()
        beside = step2()
    torch.cuda.synchronize()
    # rows of one expert in another order change nothing but the order of dw's sums
    for name in ("out", "dx", "dlogits", "idx"):
        assert torch.equal(held[name], eager[name]), name
    want = reference(eager["idx"])
    for name in ("dw1", "dw2"):
        assert (held[name].double() - want[name]).norm() <= 6 * HALF * want[name].norm()
    for name in ("out", "dx", "dlogits", "idx"):
        assert torch.equal(beside[name], before[name]), name
    del graph
    ep.destroy()
    other.destroy()


def test_as_many_tokens_as_31_bits_count(comm):
    """The last token and its neighbours, where steps of 32-bit counters pass their end."""
    from nccl_b200.ops.ep import ExpertParallel
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB")
    ep, T = ExpertParallel(comm, 1, 4, 128), (1 << 31) - 1
    ends = [0, 1, T // 2, T - 5000, T - 2, T - 1]
    y = torch.arange(1, 33, device="cuda", dtype=torch.float32).bfloat16().view(4, 8)
    rows = torch.full((T, 1), -1, device="cuda", dtype=torch.int32)
    for i, t in enumerate(ends):
        rows[t] = i % 4
    dx = torch.ones(T, 8, device="cuda", dtype=torch.bfloat16)
    ep.dispatch_backward(y, rows, out=dx)
    for i, t in enumerate(ends):
        assert torch.equal(dx[t], y[i % 4]), t
        if 0 < t < T - 1:
            assert not dx[t + 2 - (t == T - 2) * 4].any()
    rows.fill_(-1)
    rows[T - 1] = 2
    weights, dweights, dy = torch.full((T, 1), 0.5, device="cuda"), torch.ones(T, 1, device="cuda"), torch.zeros_like(y)
    ep.combine_backward(dx, y, weights, rows, dy=dy, dweights=dweights)
    assert torch.equal(dy[2], dx[T - 1] / 2) and not dy[[0, 1, 3]].any()
    assert dweights[T - 1].item() == (dx[T - 1].float() * y[2].float()).sum().item() and not dweights[[0, 1, T - 5000, T - 2]].any()
    del dx, rows, weights, dweights
    logits = torch.zeros(T, 1, device="cuda", dtype=torch.bfloat16)
    logits[T - 2] = -math.inf
    idx, w = ep.route(logits, 1)
    assert idx[[0, T - 3, T - 2, T - 1], 0].tolist() == [0, 0, -1, 0] and w[[0, T - 3, T - 2, T - 1], 0].tolist() == [1, 1, 0, 1]
    grad = ep.route_backward(w, logits, idx, score="sigmoid", renormalize=False, out=logits)
    assert grad[[0, T - 3, T - 2, T - 1], 0].tolist() == [0.25, 0.25, 0.0, 0.25]


def test_refusals(comm):
    from nccl_b200._lib import NcclError
    from nccl_b200.ops.ep import ExpertParallel
    ep = ExpertParallel(comm, 4, 16, 128)
    with pytest.raises(ValueError):
        ep.dispatch_rows()
    flat = ExpertParallel(comm, 4, 16, 128, layout="rank_major")
    x, idx, w = torch.randn(3, 128, device="cuda").bfloat16(), torch.zeros(3, 2, dtype=torch.int64, device="cuda"), torch.rand(3, 2, device="cuda")
    flat.dispatch(x, idx, w, fp8=False)
    with pytest.raises(NcclError):
        flat.dispatch_rows()
    y, rows = torch.randn(4, 16, 128, device="cuda").bfloat16(), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for args in ((x.float(), y, w, rows), (x, y.float(), w, rows), (x, y[..., :64], w, rows), (x, y, w.double(), rows), (x, y, w, rows.long()), (x, y, w, rows[:2]),
                 (x, y, w[:, :1], rows), (x[:, :100].contiguous(), y[..., :100].contiguous(), w, rows), (x, y.transpose(0, 1), w, rows), (x.cpu(), y, w, rows)):
        with pytest.raises(ValueError):
            ep.combine_backward(*args)
    for kw in (dict(dy=x), dict(dweights=w[:1])):
        with pytest.raises(ValueError):
            ep.combine_backward(x, y, w, rows, **kw)
    with pytest.raises(NcclError):   # over the weights that it reads
        ep.combine_backward(x, y, w, rows, dweights=w)
    for args in ((y.float(), rows), (y, rows.long()), (y, rows[0]), (y.transpose(0, 1), rows), (y[0, 0], rows)):
        with pytest.raises(ValueError):
            ep.dispatch_backward(*args)
    with pytest.raises(NcclError):
        ep.dispatch_backward(y, rows, out=y.view(-1, 128)[:3])
    none = rows[:0]
    assert ep.dispatch_backward(y, none).shape == (0, 128)
    assert ep.combine_backward(x[:0], y, w[:0], none)[1].shape == (0, 2)
    ep.destroy()
    flat.destroy()
