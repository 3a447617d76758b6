"""``dispatch_rows`` after calls of ``dispatch`` and ``combine`` that were refused or are still on their way."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ep():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from nccl_b200 import Communicator, get_unique_id
    from nccl_b200.ops.ep import ExpertParallel
    torch.cuda.set_device(0)
    c = Communicator(1, 0, get_unique_id())
    e = ExpertParallel(c, 4, 16, 128)
    yield e
    torch.cuda.synchronize()
    assert c.async_error() == 0
    e.destroy()
    c.destroy()


def inputs(T, K=2):
    return torch.randn(T, 128, device="cuda").bfloat16(), torch.rand(T, 4, device="cuda").topk(K, dim=1).indices, torch.rand(T, K, device="cuda")


def good(rows, toks, x, idx):
    T, K = idx.shape
    return torch.equal(rows.long() // 16, idx) and torch.equal(toks.view(-1, 128)[rows.view(-1).long()].view(T, K, 128), x[:, None].expand(T, K, 128))


def test_rows_after_a_dispatch_that_was_refused(ep):
    """The rows are those of the dispatch before, as many as it had."""
    from nccl_b200._lib import NcclError
    x, idx, w = inputs(3)
    more, more_idx, more_w = inputs(16)
    toks, _, _ = ep.dispatch(x, idx, w, fp8=False)
    for given in (more[:5], more.float()[:, :64]):   # another number of tokens; another hidden size
        with pytest.raises(NcclError):
            ep.dispatch(given.contiguous(), more_idx, more_w, fp8=False)
    held = torch.full((64,), 77, dtype=torch.int32, device="cuda")
    rows = ep.dispatch_rows(rows=held[:6].view(3, 2))
    assert good(rows, toks, x, idx) and (held[6:] == 77).all()


def test_no_rows_after_nothing_but_a_refusal(ep):
    from nccl_b200._lib import NcclError
    x, idx, w = inputs(4)
    with pytest.raises(NcclError):
        ep.dispatch(x[:3], idx, w, fp8=False)
    with pytest.raises(ValueError):
        ep.dispatch_rows()
    rows = torch.full((4, 2), 77, dtype=torch.int32, device="cuda")
    assert ep._moe["ncclEpDispatchRows"](ep.handle, rows.data_ptr(), ep._stream())   # the library's own answer
    torch.cuda.synchronize()
    assert (rows == 77).all()
    toks, _, _ = ep.dispatch(x, idx, w, fp8=False)
    assert good(ep.dispatch_rows(), toks, x, idx)


def test_rows_while_a_combine_is_on_its_way(ep):
    x, idx, w = inputs(5)
    toks, _, _ = ep.dispatch(x, idx, w, fp8=False)
    before = ep.dispatch_rows()
    out = ep.combine(toks.clone(), send_only=True)
    rows = ep.dispatch_rows()
    ep.complete()
    assert torch.equal(rows, before) and good(rows, toks, x, idx)
    # the token itself times the sum of its weights: three roundings of fp32 and one to bf16
    want = x.double() * w.double().sum(1, keepdim=True)
    assert ((out.double() - want).abs() <= (2.0 ** -8 + 4 * 2.0 ** -24) * want.abs()).all()
