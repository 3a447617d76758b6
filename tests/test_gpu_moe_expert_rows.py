"""The experts' products where the rows of a group's experts differ widely, and in buffers that hold far more rows than are in use, against
64-bit references."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

HALF, U32 = 2.0 ** -8, 2.0 ** -23   # a rounding to bf16; an fp32 addition in the tensor cores, which need not round to nearest


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


# whole sixteens of rows in all experts but a few: many tiles of d(W) in a row need no zeros, and then one does, at any stage of the ring
@pytest.mark.parametrize("counts", [[640] * 12 + [633], [16, 32, 48, 64, 80, 96, 112] * 4 + [1], [64] * 9 + [0] * 5 + [7] + [128] * 9 + [129], [0] * 30 + [5], [256, 3] * 12])
def test_weight_gradients_of_experts_of_which_few_end_inside_a_step(ep, counts):
    E, cap, n, k = len(counts), max(counts), 1304, 520   # more tiles of an expert than pairs that share them
    g = torch.Generator(device="cuda").manual_seed(sum(counts))
    x = torch.randn(E, cap, k, device="cuda", generator=g).bfloat16()
    dout = torch.randn(E, cap, n, device="cuda", generator=g).bfloat16()
    w = torch.empty(E, n, k, device="cuda", dtype=torch.bfloat16)
    for e, m in enumerate(counts):
        x[e, m:] = dout[e, m:] = math.nan
    c = torch.tensor(counts, dtype=torch.int32, device="cuda")
    _, dw, _ = ep.expert_linear_backward(dout, x, w, c, need_dx=False)
    for e, m in enumerate(counts):
        d, xe = dout[e, :m].double(), x[e, :m].double()
        ref, far = d.T @ xe, m * U32 * (d.abs().T @ xe.abs())
        assert ((dw[e].double() - ref).abs() <= far + HALF * (ref.abs() + far)).all(), e


# columns that end at every eight of a lane's steps and of the tiles, on single CTAs and on pairs (with `pre` and few tiles results go straight from registers)
@pytest.mark.parametrize("n", [8, 16, 24, 40, 64, 72, 88, 104, 136, 248, 264, 296])
@pytest.mark.parametrize("cap,counts", [(70, [70, 3, 33]), (300, [300, 129, 1])])
def test_residual_in_the_results_place(ep, n, cap, counts):
    E, k = len(counts), 72
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(E, cap, k, device="cuda", generator=g).bfloat16()
    w = (torch.randn(E, n, k, device="cuda", generator=g) / math.sqrt(k)).bfloat16()
    r = torch.randn(E, cap, n, device="cuda", generator=g).bfloat16()
    c = torch.tensor(counts, dtype=torch.int32, device="cuda")
    for e, m in enumerate(counts):
        r[e, m:] = 77.0
    out, pre = r.clone(), torch.empty_like(r)
    assert ep.expert_linear(x, w, c, residual=out, out=out, pre=pre) is out
    for e, m in enumerate(counts):
        z, far = x[e, :m].double() @ w[e].double().T, k * U32 * (x[e, :m].double().abs() @ w[e].double().abs().T)
        v = z + r[e, :m].double()
        assert ((out[e, :m].double() - v).abs() <= far + U32 * v.abs() + HALF * (v.abs() + far)).all() and (out[e, m:] == 77.0).all()


def _product(ep, E, cap, n, k, counts, act, bias):
    g = torch.Generator(device="cuda").manual_seed(E + cap)
    x = torch.full((E, cap, k), math.nan, device="cuda", dtype=torch.bfloat16)
    for e, m in enumerate(counts):
        x[e, :m] = torch.randn(m, k, device="cuda", generator=g).bfloat16()
    w = (torch.randn(E, n, k, device="cuda", generator=g) / math.sqrt(k)).bfloat16()
    b = torch.randn(E, n, device="cuda", generator=g).bfloat16() if bias else None
    cols = n // 2 if act == "swiglu" else n
    out = torch.full((E, cap, cols), 77.0, device="cuda", dtype=torch.bfloat16)
    ep.expert_linear(x, w, torch.tensor(counts, dtype=torch.int32, device="cuda"), bias=b, activation=act, out=out)
    for e, m in enumerate(counts):
        xd, wd = x[e, :m].double(), w[e].double()
        z = xd @ wd.T + (b[e].double() if bias else 0)
        far = k * U32 * (xd.abs() @ wd.abs().T) + U32 * z.abs()
        if act == "swiglu":
            # silu's slope is 1.1 at most; its own arithmetic is off by some units of its argument
            gate, up, dg, du = z[:, :cols], z[:, cols:], far[:, :cols], far[:, cols:]
            v, ev = gate * torch.sigmoid(gate), 1.1 * dg + 32 * U32 * gate.abs()
            z, far = v * up, ev * up.abs() + (v.abs() + ev) * du
        assert ((out[e, :m].double() - z).abs() <= far + HALF * (z.abs() + far) + U32 * z.abs()).all(), e
        assert (out[e, m:] == 77.0).all()


# what a group sized for prefill does when it decodes: few rows, or none, in buffers for thousands
@pytest.mark.parametrize("act,bias", [(None, False), (None, True), ("swiglu", False)])
@pytest.mark.parametrize("E,cap,counts", [(8, 4096, [1, 0, 0, 0, 0, 1, 0, 0]), (8, 4096, [0] * 7 + [1]), (4, 3001, [3, 128, 129, 0]), (256, 512, [e % 5 for e in range(256)]),
                                          (256, 8, [8 - e % 9 for e in range(256)])])
def test_few_rows_in_large_buffers(ep, E, cap, counts, act, bias):
    _product(ep, E, cap, 144, 200, counts, act, bias)


def test_gradients_of_few_rows_in_large_buffers(ep):
    E, cap, n, k, counts = 6, 4096, 208, 136, [1, 0, 17, 0, 64, 2]
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dout = (torch.randn(E, cap, c, device="cuda", generator=g).bfloat16() for c in (k, n))
    w = (torch.randn(E, n, k, device="cuda", generator=g) / math.sqrt(k)).bfloat16()
    for e, m in enumerate(counts):
        x[e, m:] = dout[e, m:] = math.nan
    dx = torch.full_like(x, 77.0)
    dx, dw, db = ep.expert_linear_backward(dout, x, w, torch.tensor(counts, dtype=torch.int32, device="cuda"), need_dbias=True, dx=dx)
    for e, m in enumerate(counts):
        d, xe, we = dout[e, :m].double(), x[e, :m].double(), w[e].double()
        for got, ref, size, terms in ((dx[e, :m], d @ we, d.abs() @ we.abs(), n), (dw[e], d.T @ xe, d.abs().T @ xe.abs(), m), (db[e], d.sum(0), d.abs().sum(0), m)):
            far = terms * U32 * size
            assert ((got.double() - ref).abs() <= far + HALF * (ref.abs() + far)).all(), e
        assert (dx[e, m:] == 77.0).all()
