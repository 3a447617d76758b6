"""Backward passes with few tiles: several CTAs share one's partners, and their sums are added up afterwards."""
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


CASES = [
    # B, Q, K, H, G, D, dtype, causal, offset, q_lengths, kv_lengths
    (1, 1500, 260, 8, 1, 128, BF16, True, 100, None, None),          # dk, dv of few keys
    (1, 20, 4000, 4, 2, 64, F16, True, None, None, None),            # dq of few queries
    (2, 700, 900, 4, 1, 96, F16, False, None, [700, 333], [900, 0]),
    (2, 700, 900, 4, 1, 96, BF16, True, None, [129, 700], [900, 385]),
    (1, 3000, 3000, 2, 2, 40, BF16, True, None, None, None),
    (1, 64, 64, 1, 1, 16, BF16, True, None, None, None),
]


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_parts(cp, case, add):
    B, Q, K, H, G, D, dtype, causal, offset, ql, kl = case
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s, t=dtype: torch.randn(*s, device="cuda", generator=g).to(t)   # noqa: E731
    q, k, v, dout = r(B, Q, H, D), r(B, K, G, D), r(B, K, G, D), r(B, Q, H, D)
    sums = (r(B, Q, H, D, t=F32), r(B, K, G, D, t=F32), r(B, K, G, D, t=F32)) if add else None
    ql, kl = (None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ql, kl))
    rule = dict(causal=causal, offset=offset, q_lengths=ql, kv_lengths=kl)
    out, lse = cp.attention(q, k, v, **rule)
    for result in (dtype, F32):
        ref = Reference(q, k, v, causal, offset, None, ql, kl, dout=dout, out=out, result=result, add=sums)
        got = cp.attention_backward(dout, q, k, v, out, lse, add=sums, dtype=result, **rule)
        for name, t in zip(("dv", "dk", "dq"), got[::-1]):
            check(name, t, getattr(ref, name), getattr(ref, name + "_tol"))
    again = cp.attention_backward(dout, q, k, v, out, lse, add=sums, dtype=F32, **rule)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    if add:
        cp.attention_backward(dout, q, k, v, out, lse, add=sums, dtype=F32, dq=sums[0], dk=sums[1], dv=sums[2], **rule)
        assert all(torch.equal(a, b) for a, b in zip(sums, got))
