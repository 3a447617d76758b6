"""Gradients of ring attention and of the Ulysses swap on CPU ranks (host-only communicators over sockets), against differentiation of attention over the whole sequence."""
import pytest

torch = pytest.importorskip("torch")

from mp_util import run_ranks  # noqa: E402

ENV = {"NCCL_B200_HOST_ONLY": "1", "NCCL_SOCKET_IFNAME": "lo"}
B, H, S, D = 2, 6, 9, 16


def _inputs(n):
    g = torch.Generator().manual_seed(12)
    return [torch.randn(B, H, S * n, D, generator=g) for _ in range(4)]


def _rank(rank, nranks, uid, causal):
    import torch
    torch.set_num_threads(2)
    from nccl_b200 import Communicator
    from nccl_b200.parallel.context import ring_attention, ring_attention_backward, ulysses_attention, ulysses_attention_backward
    comm = Communicator(nranks, rank, uid)
    q, k, v, dout = [t[:, :, rank * S:(rank + 1) * S].contiguous() for t in _inputs(nranks)]
    plain = ring_attention(comm, q, k, v, causal=causal)
    out, lse = ring_attention(comm, q, k, v, causal=causal, with_lse=True)
    assert torch.equal(plain, out)
    ring = ring_attention_backward(comm, dout, q, k, v, out, lse, causal=causal)
    qs, ks, vs, ds = [t.transpose(1, 2).contiguous() for t in (q, k, v, dout)]
    o, state = ulysses_attention(comm, qs, ks, vs, causal=causal, with_state=True)
    assert torch.equal(o, ulysses_attention(comm, qs, ks, vs, causal=causal))
    uly = [t.transpose(1, 2) for t in ulysses_attention_backward(comm, ds, state, causal=causal)]
    comm.destroy()
    return [t.numpy() for t in ring], [t.numpy() for t in uly], lse.numpy()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n", [1, 2, 3])
def test_gradients_of_a_shared_sequence(n, causal):
    res = run_ranks(_rank, n, args=(causal,), env=ENV, timeout=200)
    q, k, v, dout = _inputs(n)
    ins = [t.double().requires_grad_(True) for t in (q, k, v)]
    s = ins[0] @ ins[1].mT / D ** 0.5
    if causal:
        s = s.masked_fill(~torch.ones(S * n, S * n, dtype=torch.bool).tril(), float("-inf"))
    lse = torch.logsumexp(s, -1)
    want = torch.autograd.grad(torch.softmax(s, -1) @ ins[2], ins, dout.double())
    # fp32: a sum of at most S * n * H terms of a few products each, relative to the largest values
    for r in range(n):
        sl = slice(r * S, (r + 1) * S)
        assert (torch.from_numpy(res[r][2]).double() - lse[:, :, sl]).abs().max() <= 2e-5
        for which in (0, 1):
            for got, w in zip(res[r][which], want):
                assert (torch.from_numpy(got.copy()).double() - w[:, :, sl]).abs().max() <= 2e-5 * w.abs().max()
