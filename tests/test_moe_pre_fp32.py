"""What the calls hand to the library for pre-activations of either type: tensors in host memory, with the library's calls recorded."""
import pytest

torch = pytest.importorskip("torch")

from test_moe_arguments import ep  # noqa: E402,F401


@pytest.mark.parametrize("activation,code", [(None, 0), ("gelu", 2), ("swiglu", 4)])
def test_the_type_of_pre_goes_with_the_activation(ep, activation, code):  # noqa: F811
    x, w = torch.zeros(2, 5, 16, dtype=torch.bfloat16), torch.zeros(2, 32, 16, dtype=torch.bfloat16)
    dout = torch.zeros(2, 5, 16 if activation == "swiglu" else 32, dtype=torch.bfloat16)
    for dtype, more in ((torch.bfloat16, 0), (torch.float32, 256)):
        pre = torch.zeros(2, 5, 32, dtype=dtype)
        ep.expert_linear(x, w, None, activation=activation, pre=pre)
        ep.expert_linear_backward(dout, x, w, None, activation=activation, pre=pre)
        there, back = ep.calls[-2:]
        assert there[0] == "ncclEpExpertLinear" and there[8] == pre.data_ptr() and there[-2] == code + more
        # without an activation it is not looked at
        assert back[0] == "ncclEpExpertLinearBackward" and back[6] == (pre.data_ptr() if code else None) and back[-2] == (code + more if code else 0)
    for bad in (torch.zeros(2, 5, 32).half(), torch.zeros(2, 5, 16), torch.zeros(2, 32, 5).transpose(1, 2)):
        with pytest.raises(ValueError):
            ep.expert_linear(x, w, None, activation=activation, pre=bad)
        if code:
            with pytest.raises(ValueError):
                ep.expert_linear_backward(dout, x, w, None, activation=activation, pre=bad)
