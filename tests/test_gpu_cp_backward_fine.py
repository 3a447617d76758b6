"""Backward calls that do not fill the GPU lose nothing by rounding probabilities and ds to 16 bits; where they fill it, at most half a step of each. On both sides of the edge."""
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


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("over", [0, 1])
@pytest.mark.parametrize("layout", ["heads", "batch", "keys"])
def test_calls_at_the_edge(cp, dtype, D, over, layout):
    """One tile of queries for each owner; as many products of tiles as half of the SMs, and one more."""
    products = torch.cuda.get_device_properties(0).multi_processor_count // 2 + over
    B, Q, K, H = {"heads": (1, 100, 120, products), "batch": (products, 70, 128, 1), "keys": (1, 60, 128 * products - 5, 1)}[layout]
    r = lambda i, *s: torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(900 + i)).to(dtype)   # noqa: E731
    q, k, v, dout = r(0, B, Q, H, D), r(1, B, K, H, D), r(2, B, K, H, D), r(3, B, Q, H, D)
    out, lse = cp.attention(q, k, v, causal=True)
    got = cp.attention_backward(dout, q, k, v, out, lse, causal=True, dtype=F32)
    ref = Reference(q, k, v, True, dout=dout, out=out, result=F32, fine=not over)
    for name, t in zip(("dv", "dk", "dq"), got[::-1]):
        check(name, t, getattr(ref, name), getattr(ref, name + "_tol"))
    again = cp.attention_backward(dout, q, k, v, out, lse, causal=True, dtype=F32)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
