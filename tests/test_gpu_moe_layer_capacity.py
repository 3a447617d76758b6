"""A whole mixture-of-experts layer of a group that is sized for many more tokens than a step has, there and back."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_moe_layer import HALF, _layer, comm  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,cap,H,F,E,K", [(1, 4096, 256, 128, 8, 2), (37, 4096, 384, 176, 16, 4), (3, 129, 128, 64, 256, 8)])
def test_layer_of_few_tokens(comm, T, cap, H, F, E, K, score):  # noqa: F811
    ep, step, reference = _layer(comm, T, cap, H, F, E, K, score, T)
    got = step()
    want = reference(got["idx"])
    for name in ("out", "dx", "dw1", "dw2", "dlogits"):
        # the tensors on the way (six to bf16 at most) are rounded by up to 2^-8 of themselves, as independent errors
        far = (got[name].double() - want[name]).norm() / want[name].norm()
        assert far <= 6 * HALF, (name, float(far))
    ep.destroy()
