"""Pre-activations that are kept in fp32: what the forward call keeps, and gradients from them, against 64-bit references."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_moe_experts import U32, backward, ep, forward, make, value_slope, within  # noqa: E402,F401

pytestmark = pytest.mark.gpu


# single CTAs, pairs that store straight from registers, and (enough tiles, a residual or rows that are no whole packs) pairs that go through shared memory
@pytest.mark.parametrize("E,cap,n,k,counts,residual", [(3, 70, 144, 72, [70, 0, 9], True), (4, 64, 88, 40, [64, 1, 33, 17], False), (3, 300, 272, 136, [300, 129, 0], True), (2, 513, 520, 64, None, False),
                                                       (64, 300, 1208, 72, [e * 5 % 301 for e in range(64)], False), (64, 260, 1216, 64, [260 - e for e in range(64)], True)])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu", "swiglu", "geglu"])
def test_kept_in_fp32(ep, E, cap, n, k, counts, residual, act):  # noqa: F811
    if act in ("swiglu", "geglu"):
        n *= 2
    x, w, b, r, dout, c = make(E, cap, n, k, act, 7, True, residual, counts)
    used = counts or [cap] * E
    pre = torch.full((E, cap, n), 12345.0, device="cuda")
    half = torch.zeros(E, cap, n, dtype=torch.bfloat16, device="cuda")
    out = ep.expert_linear(x, w, c, bias=b, activation=act, residual=r, pre=pre)
    same = ep.expert_linear(x, w, c, bias=b, activation=act, residual=r, pre=half)
    dx, dw, db = ep.expert_linear_backward(dout, x, w, c, pre=pre if act else None, activation=act, need_dbias=True)
    for e, m in enumerate(used):
        assert (pre[e, m:] == 12345.0).all(), "rows behind the last were written"
        assert torch.equal(out[e, :m], same[e, :m]) and torch.equal(pre[e, :m].bfloat16(), half[e, :m])
        xd, wd = x[e, :m].double(), w[e].double()
        z = xd @ wd.T + b[e].double()
        # one addition per step of the sum, and the bias; no rounding behind them
        assert within(pre[e, :m], z, k * U32 * (xd.abs() @ wd.abs().T) + U32 * z.abs())
        a, ae, ww, we, bb, be = backward(act, dout[e, :m].double(), xd, wd, pre[e, :m].double())
        assert within(dx[e, :m], a, ae) and within(dw[e], ww, we) and within(db[e], bb, be)


def test_gradients_are_off_by_two_roundings(ep):  # noqa: F811
    """That of the activation's gradient, which is an operand, and that of the result. They are independent: their squares add up. Products with
    random matrices keep the relative size of an error to some per cent."""
    rows, n, k = 512, 2048, 512
    x, w, _, _, dout, _ = make(1, rows, n, k, "swiglu", 3, False, False, None)
    pre = torch.empty(1, rows, n, device="cuda")
    ep.expert_linear(x, w, None, activation="swiglu", pre=pre)
    dx, dw, _ = ep.expert_linear_backward(dout, x, w, None, pre=pre, activation="swiglu")
    z = x[0].double() @ w[0].double().T
    gate, up, g = z[:, : n // 2], z[:, n // 2:], dout[0].double()
    v, s = value_slope("silu", gate)
    dz = torch.cat([g * up * s, g * v], 1)

    def rounding(t):
        return float((t.bfloat16().double() - t).norm() / t.norm())

    for got, ref in ((dx[0], dz @ w[0].double()), (dw[0], dz.T @ x[0].double())):
        far = float((got.double() - ref).norm() / ref.norm())
        assert far <= 1.1 * (rounding(dz) ** 2 + rounding(ref) ** 2) ** 0.5


def test_refusals(ep):  # noqa: F811
    from nccl_b200._lib import NcclError
    x, w, _, _, dout, _ = make(2, 16, 32, 24, "silu", 1, False, False, None)
    pre = torch.empty(2, 16, 32, device="cuda")
    for bad in (pre.half(), pre.double(), pre[:, :8], pre.transpose(0, 1), pre.cpu()):
        with pytest.raises(ValueError):
            ep.expert_linear(x, w, None, activation="silu", pre=bad)
        with pytest.raises(ValueError):
            ep.expert_linear_backward(dout, x, w, None, pre=bad, activation="silu")
    # the second half of what fp32 takes counts too
    raw = torch.zeros(2 * 16 * 32 * 2, device="cuda")
    over = raw[2 * 16 * 32 - 16 * 16:].view(torch.bfloat16)[: 2 * 16 * 32].view(2, 16, 32)
    with pytest.raises(NcclError):
        ep.expert_linear(x, w, None, activation="silu", pre=raw[: 2 * 16 * 32].view(2, 16, 32), out=over)
    with pytest.raises(NcclError):
        ep.expert_linear_backward(dout, x, w, None, pre=raw[: 2 * 16 * 32].view(2, 16, 32), activation="silu", dx=over.view(-1)[: 2 * 16 * 24].view(2, 16, 24))
