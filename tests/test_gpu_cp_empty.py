"""Tensors without an element may have any strides and any place: nothing of them is read."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


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


def empties(B, heads, D):
    """[B, 0, heads, D] with strides that an operand with rows may not have, and one that it may."""
    t = dict(dtype=torch.bfloat16, device="cuda")
    return [torch.empty(1, 0, heads, D, **t).expand(B, 0, heads, D), torch.empty(B, 0, 1, D, **t).expand(B, 0, heads, D), torch.empty(B, 0, heads, D + 3, **t)[..., 3:],
            torch.empty(B, heads, D, 0, **t).permute(0, 3, 1, 2), torch.empty(B, 9, heads, D, **t)[:, 4:4]]


@pytest.mark.parametrize("Q", [1, 40, 300])
def test_no_keys(cp, Q):
    B, H, G, D = 3, 4, 2, 16
    q = torch.randn(B, Q, H, D, device="cuda").bfloat16()
    for none in empties(B, G, D):
        out, lse = cp.attention(q, none, none, causal=True)
        assert not out.any() and bool((lse == -math.inf).all())
        join = torch.randn(B, Q, H, D, device="cuda"), torch.randn(B, H, Q, device="cuda")
        got = cp.attention(q, none, none, join=join, dtype=torch.float32)
        assert torch.equal(got[0], join[0]) and torch.equal(got[1], join[1])
        dq, dk, dv = cp.attention_backward(q, q, none, none, out, lse, causal=True)
        assert not dq.any() and dk.shape == dv.shape == none.shape


@pytest.mark.parametrize("K", [1, 300])
def test_no_queries(cp, K):
    B, H, G, D = 3, 4, 2, 16
    k = torch.randn(B, K, G, D, device="cuda").bfloat16()
    for none in empties(B, H, D):
        out, lse = cp.attention(none, k, k, causal=True)
        assert out.shape == none.shape and lse.shape == (B, H, 0)
        dq, dk, dv = cp.attention_backward(none, none, k, k, none, lse, causal=True)
        assert dq.shape == none.shape and not dk.any() and not dv.any()
        assert cp.attention_delta(none, none).shape == lse.shape
