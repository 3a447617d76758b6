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
