"""What ``dispatch_rows`` refuses before anything reaches a GPU."""
import pytest

torch = pytest.importorskip("torch")


def test_a_group_whose_only_dispatch_was_refused_has_no_rows():
    from nccl_b200.ops.ep import ExpertParallel
    e = ExpertParallel.__new__(ExpertParallel)
    e.torch, e._device, e._place, e._raw_stream = torch, -1, torch.device("cpu"), lambda device: 0
    e.handle, e._keep = 5, None   # the refused call has made the handle and kept nothing
    calls = []
    e._moe = {"ncclEpDispatchRows": lambda *args: calls.append(args) or 0}
    with pytest.raises(ValueError):
        e.dispatch_rows()
    assert not calls
