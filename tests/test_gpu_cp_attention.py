"""Attention of ``ContextParallel``: results, log-sum-exp and gradients against 64 bits, with bounds that count each rounding."""
import math

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


def inputs(B, Q, K, H, G, D, dtype, seed=0, packed=False):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)   # noqa: E731
    if packed:
        assert Q == K
        return r(B, Q, H + 2 * G, D).split((H, G, G), dim=2)
    return r(B, Q, H, D), r(B, K, G, D), r(B, K, G, D)


def lens(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


FORWARD = [
    # B, Q, K, H, G, D, dtype, causal, offset, q_lengths, kv_lengths
    (1, 128, 128, 1, 1, 128, BF16, False, None, None, None),
    (1, 1, 1, 1, 1, 8, BF16, False, None, None, None),
    (2, 1, 257, 8, 2, 128, BF16, True, None, None, None),
    (1, 1, 4096, 32, 8, 128, BF16, True, None, None, None),
    (3, 1, 700, 8, 8, 64, F16, True, None, None, [700, 0, 129]),
    (2, 3, 300, 6, 2, 96, F16, True, None, None, [300, 2]),
    (1, 130, 130, 2, 2, 64, F16, True, None, None, None),
    (2, 257, 515, 6, 2, 80, BF16, True, 0, None, None),
    (2, 257, 515, 7, 1, 40, F16, True, -13, None, None),
    (2, 200, 333, 5, 5, 128, BF16, False, None, [200, 77], [333, 128]),
    (3, 200, 333, 3, 1, 128, F16, True, None, [0, 77, 200], [333, 128, 0]),
    (1, 2500, 1100, 8, 1, 128, BF16, True, -700, None, None),
    (4, 300, 640, 40, 8, 128, BF16, True, None, None, [640, 513, 512, 1]),
    (2, 1024, 1024, 16, 16, 64, F16, True, None, None, None),
    (1, 77, 20000, 4, 2, 128, F16, False, None, None, None),
    (1, 2, 9, 130, 2, 16, BF16, True, None, None, None),
    (1, 5, 200, 128, 1, 128, BF16, False, None, None, None),
]


@pytest.mark.parametrize("case", FORWARD, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_attention(cp, case):
    B, Q, K, H, G, D, dtype, causal, offset, ql, kl = case
    q, k, v = inputs(B, Q, K, H, G, D, dtype)
    ql, kl = lens(ql), lens(kl)
    out, lse = cp.attention(q, k, v, causal=causal, offset=offset, q_lengths=ql, kv_lengths=kl)
    ref = Reference(q, k, v, causal, offset, None, ql, kl)
    check("lse", lse, ref.lse, ref.lse_tol)
    check("out", out, ref.out, ref.out_tol)


BACKWARD = [
    (1, 128, 128, 1, 1, 128, BF16, False, None, None, None),
    (1, 1, 2, 1, 1, 8, BF16, False, None, None, None),
    (2, 1, 257, 8, 2, 128, BF16, True, None, None, None),
    (2, 256, 256, 8, 8, 64, F16, True, None, None, None),
    (2, 257, 515, 6, 2, 80, BF16, True, 0, None, None),
    (2, 300, 515, 7, 1, 40, F16, True, -13, None, None),
    (3, 200, 333, 3, 1, 128, F16, True, None, [0, 77, 200], [333, 128, 0]),
    (2, 509, 641, 12, 4, 96, BF16, False, None, [509, 130], [641, 128]),
    (1, 1300, 700, 4, 1, 128, BF16, True, -300, None, None),
    (1, 1024, 1024, 4, 2, 128, BF16, True, None, None, None),
    (1, 3, 40, 128, 1, 64, F16, False, None, None, None),
]


@pytest.mark.parametrize("case", BACKWARD, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_attention_backward(cp, case):
    B, Q, K, H, G, D, dtype, causal, offset, ql, kl = case
    q, k, v = inputs(B, Q, K, H, G, D, dtype, 1)
    dout = torch.randn(B, Q, H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)).to(dtype)
    ql, kl = lens(ql), lens(kl)
    rule = dict(causal=causal, offset=offset, q_lengths=ql, kv_lengths=kl)
    out, lse = cp.attention(q, k, v, **rule)
    got = cp.attention_backward(dout, q, k, v, out, lse, **rule)
    ref = Reference(q, k, v, causal, offset, None, ql, kl, dout=dout, out=out)
    for name, t in zip(("dv", "dk", "dq"), got[::-1]):
        check(name, t, getattr(ref, name), getattr(ref, name + "_tol"))
    again = cp.attention_backward(dout, q, k, v, None, lse, delta=cp.attention_delta(dout, out, ql), **rule)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
