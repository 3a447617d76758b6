"""The experts' products, forward and backward, against 64-bit references with bounds that follow from the roundings on the way."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8      # rounding to bf16, relative
U32 = 2.0 ** -23      # an fp32 addition in the tensor cores, which need not round to nearest


@pytest.fixture(scope="module")
def ep():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from nccl_b200 import Communicator, get_unique_id
    from nccl_b200.ops.ep import ExpertParallel
    torch.cuda.set_device(0)
    c = Communicator(1, 0, get_unique_id())
    e = ExpertParallel(c, 4, 1, 128)
    yield e
    torch.cuda.synchronize()
    assert c.async_error() == 0
    e.destroy()
    c.destroy()


def base_of(act):
    return {"swiglu": "silu", "geglu": "gelu"}.get(act, act)


def value_slope(act, z):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def forward(act, x, w, b, r):
    """(out, its bound, pre, its bound) of one expert in 64 bits."""
    z = x @ w.T + (0 if b is None else b)
    dz = x.shape[1] * U32 * (x.abs() @ w.abs().T) + U32 * z.abs()   # one addition per step of the sum, and the bias
    n = w.shape[0]
    gate, up, dg, du = (z[:, : n // 2], z[:, n // 2:], dz[:, : n // 2], dz[:, n // 2:]) if act in ("swiglu", "geglu") else (z, None, dz, None)
    v, _ = value_slope(base_of(act), gate)
    # slopes are 1.13 at most; the activation's own arithmetic is off by some units of fp32 of its argument
    e = 1.13 * dg + 32 * U32 * gate.abs()
    if up is not None:
        v, e = v * up, e * up.abs() + (v.abs() + e) * du
    if r is not None:
        v = v + r
    return v, e + HALF * (v.abs() + e) + U32 * v.abs(), z, dz + HALF * (z.abs() + dz)


def backward(act, dout, x, w, pre):
    """(dx, bound, dw, bound, dbias, bound) of one expert from the pre-activations as the forward call rounded them."""
    n = w.shape[0]
    if act is None:
        dz, e = dout, torch.zeros_like(dout)
    else:
        gate = pre[:, : n // 2] if act in ("swiglu", "geglu") else pre
        v, s = value_slope(base_of(act), gate)
        v_err, s_err = 32 * U32 * (gate.abs() + 1), 32 * U32 * (gate.abs() + 1) ** 2
        if act in ("swiglu", "geglu"):
            up = pre[:, n // 2:]
            dz = torch.cat([dout * up * s, dout * v], 1)
            e = torch.cat([dout.abs() * up.abs() * s_err, dout.abs() * v_err], 1)
        else:
            dz, e = dout * s, dout.abs() * s_err
    er = e + HALF * (dz.abs() + e) if act is not None else e   # rounded before the products
    rows = dout.shape[0]
    dx, ex = dz @ w, er @ w.abs() + n * U32 * (dz.abs() @ w.abs())
    dw, ew = dz.T @ x, er.T @ x.abs() + rows * U32 * (dz.abs().T @ x.abs())
    db, eb = dz.sum(0), e.sum(0) + rows * U32 * dz.abs().sum(0)
    return dx, ex + HALF * (dx.abs() + ex), dw, ew + HALF * (dw.abs() + ew), db, eb + HALF * (db.abs() + eb)


def make(E, cap, n, k, act, seed, bias, residual, counts):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cols = n // 2 if act in ("swiglu", "geglu") else n
    x = torch.randn(E, cap, k, device="cuda", generator=g).bfloat16()
    w = (torch.randn(E, n, k, device="cuda", generator=g) / math.sqrt(k)).bfloat16()
    b = torch.randn(E, n, device="cuda", generator=g).bfloat16() if bias else None
    r = torch.randn(E, cap, cols, device="cuda", generator=g).bfloat16() if residual else None
    dout = torch.randn(E, cap, cols, device="cuda", generator=g).bfloat16()
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    return x, w, b, r, dout, c


def within(got, ref, bound):
    return bool(((got.double() - ref).abs() <= bound).all())


def check(ep, E, cap, n, k, act, counts, bias=False, residual=False, seed=5):
    """Forward and backward; rows that are not in use hold NaN before and must hold the same bits behind."""
    x, w, b, r, dout, c = make(E, cap, n, k, act, seed, bias, residual, counts)
    used = [min(max(v, 0), cap) for v in counts] if counts is not None else [cap] * E
    mark = 12345.0
    cols = dout.shape[2]
    out = torch.full((E, cap, cols), mark, dtype=torch.bfloat16, device="cuda")
    pre = torch.full((E, cap, n), mark, dtype=torch.bfloat16, device="cuda")
    dx = torch.full((E, cap, k), mark, dtype=torch.bfloat16, device="cuda")
    for e in range(E):
        for t in (x, dout) + (() if r is None else (r,)):
            t[e, used[e]:] = math.nan
    got = ep.expert_linear(x, w, c, bias=b, activation=act, residual=r, out=out, pre=pre)
    assert got is out
    dxs, dw, db = ep.expert_linear_backward(dout, x, w, c, pre=pre, activation=act, need_dbias=True, dx=dx)
    again = ep.expert_linear_backward(dout, x, w, c, pre=pre, activation=act, need_dbias=True)
    if act is None:
        lone = ep.expert_linear_backward(dout, x, w, c)
        assert torch.equal(lone[1], dw) and lone[2] is None
    assert torch.equal(again[1], dw) and torch.equal(again[2], db)   # the same bits every time
    for e in range(E):
        m = used[e]
        for t in (out, pre, dx):
            assert (t[e, m:] == mark).all(), "rows behind the last were written"
        xd, wd = x[e, :m].double(), w[e].double()
        v, ve, z, ze = forward(act, xd, wd, None if b is None else b[e].double(), None if r is None else r[e, :m].double())
        assert within(out[e, :m], v, ve)
        assert within(pre[e, :m], z, ze)
        assert torch.equal(again[0][e, :m], dx[e, :m])
        a, ae, ww, we, bb, be = backward(act, dout[e, :m].double(), xd, wd, pre[e, :m].double())
        assert within(dx[e, :m], a, ae)
        assert within(dw[e], ww, we)
        assert within(db[e], bb, be)
        if m == 0:
            assert (dw[e] == 0).all() and (db[e] == 0).all()


# rows of one expert: none, one, the ends of boxes and tiles, more than a tile and than two
@pytest.mark.parametrize("counts", [[0], [1], [15], [16], [17], [31], [32], [33], [63], [64], [65], [127], [128], [129], [255], [257]])
def test_rows_of_one_expert(ep, counts):
    check(ep, 1, 300, 136, 200, "silu", counts, bias=True, residual=True)


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu", "swiglu", "geglu"])
@pytest.mark.parametrize("E,cap,n,k,counts", [
    (3, 40, 16, 8, [0, 40, 7]),                          # the smallest sizes
    (2, 200, 16, 8, [200, 3]),                           # and on pairs
    (5, 70, 272, 72, [70, 0, 0, 33, 1]),                 # tiles that hang over on every side
    (4, 300, 528, 392, [299, 128, 0, 200]),
    (2, 1, 512, 256, [1, 0]),                            # a single token
    (2, 130, 1040, 136, None),                           # every row in use
    (3, 64, 32, 1032, [1000, -5, 64]),                   # counts beyond the rows there are, and below none
])
def test_activations_and_sizes(ep, act, E, cap, n, k, counts):
    check(ep, E, cap, n, k, act, counts, bias=True, residual=act in (None, "swiglu"))


def test_smallest_ungated(ep):
    check(ep, 2, 5, 8, 8, None, [5, 1], bias=True, residual=True)
    check(ep, 2, 150, 8, 8, "gelu", [150, 1], bias=True)


def test_captured_as_a_process_first_calls():
    """Kernels that have not been loaded yet, in a graph."""
    import os
    import subprocess
    import sys
    code = """
import torch
from nccl_b200 import Communicator, get_unique_id
from nccl_b200.ops.ep import ExpertParallel
torch.cuda.set_device(0)
c = Communicator(1, 0, get_unique_id())
ep = ExpertParallel(c, 4, 1, 128)
x, w, d = (torch.randn(4, *s, device="cuda").bfloat16() for s in ((200, 64), (96, 64), (200, 96)))
n, l = torch.tensor([3, 200, 0, 50], dtype=torch.int32, device="cuda"), torch.randn(9, 4, device="cuda")
def step():
    idx, g = ep.route(l, 2, score="sigmoid")
    return ep.expert_linear(x, w, n), ep.expert_linear_backward(d, x, w, n)[1], ep.route_backward(g, l, idx, score="sigmoid")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
want = step()
torch.cuda.synchronize()
assert torch.equal(got[0][1], want[0][1]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


def test_many_experts_few_of_them_used(ep):
    counts = [0] * 256
    for e, m in ((0, 3), (7, 1), (130, 40), (255, 17)):
        counts[e] = m
    check(ep, 256, 48, 48, 64, "swiglu", counts)


@pytest.mark.parametrize("E,cap,n,k,act,counts", [
    (2, 2100, 768, 512, None, [2049, 1111]),              # several panels of row tiles
    (8, 700, 4096, 512, "swiglu", [700, 650, 3, 0, 129, 256, 511, 512]),
    (64, 300, 2008, 64, "gelu", [(37 * e) % 301 for e in range(64)]),      # many tiles of rows that are no whole packs of 32 bytes
    (64, 300, 4016, 64, "geglu", [(53 * e) % 301 for e in range(64)]),
])
def test_large(ep, E, cap, n, k, act, counts):
    check(ep, E, cap, n, k, act, counts, bias=act is None or E == 64, residual=E == 64)


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu", "swiglu", "geglu"])
@pytest.mark.parametrize("n,residual", [(272, False), (272, True), (528, True), (560, False), (2064, True)])
def test_results_do_not_depend_on_what_else_is_kept(ep, act, n, residual):
    """With and without the pre-activations kept, results take different ways to memory."""
    counts = [200, 0, 131, 77, 256]
    x, w, b, r, _, c = make(5, 256, n, 136, act, n, True, residual, counts)
    pre = torch.empty(5, 256, n, dtype=torch.bfloat16, device="cuda")
    lone, kept = ep.expert_linear(x, w, c, bias=b, activation=act, residual=r), ep.expert_linear(x, w, c, bias=b, activation=act, residual=r, pre=pre)
    place = None
    if residual:
        place = r.clone()
        ep.expert_linear(x, w, c, bias=b, activation=act, residual=place, out=place)
    for e, m in enumerate(counts):
        v, bound, _, _ = forward(act, x[e, :m].double(), w[e].double(), b[e].double(), None if r is None else r[e, :m].double())
        assert within(lone[e, :m], v, bound) and torch.equal(lone[e, :m], kept[e, :m])
        if residual:
            assert torch.equal(place[e, :m], lone[e, :m]) and torch.equal(place[e, m:], r[e, m:])


# The second CTA of a pair has neither a row nor a column of such tiles, and many steps in which to fall behind
@pytest.mark.parametrize("n,k", [(48, 8192), (8192, 48), (64, 64)])
def test_tiles_that_one_cta_of_a_pair_has_no_part_in(ep, n, k):
    check(ep, 64, 160, n, k, "relu", [(7 * e) % 120 for e in range(64)])
    x, w = torch.randn(64, 160, k, device="cuda").bfloat16(), torch.randn(64, n, k, device="cuda").bfloat16()
    c = torch.tensor([(11 * e) % 120 + 1 for e in range(64)], dtype=torch.int32, device="cuda")
    d = torch.randn(64, 160, n, device="cuda").bfloat16()
    for _ in range(50):
        ep.expert_linear(x, w, c)
        ep.expert_linear_backward(d, x, w, c)
    torch.cuda.synchronize()
    assert ep.comm.async_error() == 0


def test_residual_in_place_and_none_kept(ep):
    x, w, b, r, _, c = make(3, 50, 64, 128, "gelu", 9, True, True, [50, 0, 20])
    want = ep.expert_linear(x, w, c, bias=b, activation="gelu", residual=r, out=torch.zeros(3, 50, 64, dtype=torch.bfloat16, device="cuda"))
    before = r.clone()
    assert ep.expert_linear(x, w, c, bias=b, activation="gelu", residual=r, out=r) is r
    for e, m in enumerate([50, 0, 20]):
        assert torch.equal(r[e, :m], want[e, :m]) and torch.equal(r[e, m:], before[e, m:])


def test_wanted_gradients_alone(ep):
    x, w, b, _, dout, c = make(3, 50, 64, 128, "silu", 9, True, False, [50, 0, 20])
    pre = torch.empty(3, 50, 64, dtype=torch.bfloat16, device="cuda")
    ep.expert_linear(x, w, c, bias=b, activation="silu", pre=pre)
    dx, dw, db = ep.expert_linear_backward(dout, x, w, c, pre=pre, activation="silu", need_dbias=True)
    got = ep.expert_linear_backward(dout, x, w, c, pre=pre, activation="silu", need_dx=False)
    assert got[0] is None and got[2] is None and torch.equal(got[1], dw)
    got = ep.expert_linear_backward(dout, x, w, c, pre=pre, activation="silu", need_dw=False)
    assert got[1] is None and torch.equal(got[0][0], dx[0]) and torch.equal(got[0][2, :20], dx[2, :20])
    got = ep.expert_linear_backward(dout, x, w, c, pre=pre, activation="silu", need_dx=False, need_dw=False, need_dbias=True)
    assert torch.equal(got[2], db)


@pytest.mark.parametrize("E,cap,n,k,act,counts", [(3, 50, 72, 128, "silu", [50, 0, 20]), (3, 300, 2200, 8, "gelu", [300, 0, 129]), (2, 129, 16, 64, "swiglu", [1, 129]),
                                                  (256, 20, 8, 8, None, [20, 0] * 128)])
def test_bias_gradient_is_the_same_whatever_else_is_wanted(ep, E, cap, n, k, act, counts):
    """A kernel of its own adds the slices up, or a warp of a product that follows: the same sums in the same order."""
    x, w, b, _, dout, c = make(E, cap, n, k, act, 3, True, False, counts)
    pre = torch.empty(E, cap, n, dtype=torch.bfloat16, device="cuda")
    ep.expert_linear(x, w, c, bias=b, activation=act, pre=pre)
    alone = ep.expert_linear_backward(dout, x, w, c, pre=pre, activation=act, need_dx=False, need_dw=False, need_dbias=True)[2]
    for dx, dw in ((True, False), (False, True), (True, True)):
        got = ep.expert_linear_backward(dout, x, w, c, pre=pre, activation=act, need_dx=dx, need_dw=dw, need_dbias=True, dbias=torch.full_like(alone, math.nan))
        assert torch.equal(got[2], alone), (dx, dw)
    bound, mass = 2.0 ** -8, 2.0 ** -24 * cap   # one rounding of the result; an addition a row, in fp32
    if act is None:
        for e, m in enumerate(counts):
            rows = dout[e, :m].double()
            assert within(alone[e], rows.sum(0), bound * rows.sum(0).abs() + mass * rows.abs().sum(0) * (1 + bound))


def test_values_that_are_not_finite_stay_with_their_row(ep):
    x, w, _, _, _, c = make(2, 40, 64, 64, None, 1, False, False, [40, 40])
    want = ep.expert_linear(x, w, c)
    x[0, 3, 5], x[1, 20, 0] = math.nan, math.inf
    got = ep.expert_linear(x, w, c)
    touched = torch.zeros(2, 40, dtype=torch.bool, device="cuda")
    touched[0, 3] = touched[1, 20] = True
    assert torch.equal(got[~touched], want[~touched]) and torch.isnan(got[0, 3]).all() and not torch.isfinite(got[1, 20]).any()


def test_streams_graphs_and_changing_counts(ep):
    """A captured forward and backward is replayed with other counts; an eager call on another stream runs beside it."""
    E, cap, n, k = 4, 150, 512, 256
    x, w, _, _, dout, c = make(E, cap, n, k, "swiglu", 3, False, False, [150, 20, 0, 77])
    out, pre = torch.zeros(E, cap, n // 2, dtype=torch.bfloat16, device="cuda"), torch.zeros(E, cap, n, dtype=torch.bfloat16, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)

    def step():
        ep.expert_linear(x, w, c, activation="swiglu", out=out, pre=pre)
        ep.expert_linear_backward(dout, x, w, c, pre=pre, activation="swiglu", dx=dx, dw=dw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for counts in ([1, 2, 3, 4], [0, 0, 0, 0], [150, 150, 150, 150]):
        c.copy_(torch.tensor(counts, dtype=torch.int32))
        for t in (out, pre, dx, dw):
            t.zero_()
        graph.replay()
        got = [t.clone() for t in (out, pre, dx, dw)]
        for t in (out, pre, dx, dw):
            t.zero_()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, (out, pre, dx, dw)))


def test_no_rows_and_refusals(ep):
    from nccl_b200._lib import NcclError
    bf = dict(dtype=torch.bfloat16, device="cuda")
    x, w, c = torch.randn(2, 16, 32, device="cuda").bfloat16(), torch.randn(2, 48, 32, device="cuda").bfloat16(), torch.tensor([16, 3], dtype=torch.int32, device="cuda")
    none = torch.empty(2, 0, 32, **bf)
    assert ep.expert_linear(none, w, c).shape == (2, 0, 48)
    dx, dw, db = ep.expert_linear_backward(torch.empty(2, 0, 48, **bf), none, w, c, need_dbias=True)
    assert dx.shape == none.shape and (dw == 0).all() and (db == 0).all()
    d = torch.randn(2, 16, 48, device="cuda").bfloat16()
    for args, kw in (((x.float(), w, c), {}), ((x, w.float(), c), {}), ((x, w[:, :, :16], c), {}), ((x, w, c.long()), {}), ((x, w, c[:1]), {}), ((x[0], w, c), {}),
                     ((x, w[:1], c), {}), ((x.transpose(0, 1), w, c), {}), ((x, w, c.cpu()), {}), ((x.cpu(), w, c), {}), ((x, w, c), dict(activation="tanh")),
                     ((x, w[:, :40].contiguous(), c), dict(activation="swiglu")), ((x[:, :, :12].contiguous(), w[:, :, :12].contiguous(), c), {}),
                     ((x, w, c), dict(bias=torch.zeros(2, 47, **bf))), ((x, w, c), dict(residual=d.float())), ((x, w, c), dict(out=d[:, :8])), ((x, w, c), dict(pre=x))):
        with pytest.raises(ValueError):
            ep.expert_linear(*args, **kw)
    with pytest.raises(ValueError):
        ep.expert_linear(torch.empty(2, 16, 0, **bf), torch.empty(2, 48, 0, **bf), c)
    for args, kw in (((d[:, :, :40].contiguous(), x, w, c), {}), ((d, x, w, c), dict(activation="gelu")), ((d, x, w, c), dict(activation="gelu", pre=x)),
                     ((d, x, w, c), dict(dx=d)), ((d, x, w, c), dict(need_dbias=True, dbias=d))):
        with pytest.raises(ValueError):
            ep.expert_linear_backward(*args, **kw)
    # outputs that share memory with inputs or one another
    square = torch.randn(2, 32, 32, device="cuda").bfloat16()
    s = torch.randn(2, 32, 32, device="cuda").bfloat16()
    for kw in (dict(out=s), dict(out=square), dict(pre=s)):
        with pytest.raises(NcclError):
            ep.expert_linear(s, square, c, **kw)
    o = torch.empty_like(s)
    with pytest.raises(NcclError):
        ep.expert_linear(s, square, c, out=o, pre=o)
    for kw in (dict(dx=s), dict(dx=square), dict(dx=o, dw=o), dict(dw=s)):
        with pytest.raises(NcclError):
            ep.expert_linear_backward(o if "dw" in kw and "dx" not in kw else torch.empty_like(s), s, square, c, **kw)
    raw = torch.zeros(2 * 16 * 32 + 4, **bf)
    with pytest.raises(NcclError):   # 8-byte aligned
        ep.expert_linear(raw[4:].view(2, 16, 32), w, c)
