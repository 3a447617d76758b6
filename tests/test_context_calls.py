"""What the ring and the Ulysses swap hand on, without a GPU: streams and events recorded, the kernels' calls recorded."""
import contextlib
import types

import pytest

torch = pytest.importorskip("torch")

from test_cp_arguments import cp, shape_at  # noqa: E402, F401


class FakeStream:
    def __init__(self, name, log):
        self.name, self.log = name, log

    def wait_event(self, event):
        self.log.append((self.name, "waits for", event.on))


class FakeComm:
    nranks, rank, lib = 2, 0, None

    def __init__(self, log):
        self.log = log

    def send(self, t, peer, stream=None):
        self.log.append(("send", stream.name))

    def recv(self, t, peer, stream=None):
        self.log.append(("recv", stream.name))


def test_the_ring_is_ordered_with_the_streams_of_its_own_gpu(monkeypatch):
    """The exchange waits for what the tensors' GPU has been given, and that GPU's stream for the exchange, whichever GPU is the current one."""
    from nccl_b200.parallel import context
    log, entered = [], []
    place = torch.device("cuda", 3)

    class FakeEvent:
        on = None

        def record(self, stream=None):
            self.on = (stream or torch.cuda.current_stream()).name

    @contextlib.contextmanager
    def enter(stream):
        entered.append(stream)
        yield
        entered.pop()

    def current_stream(device=None):
        return entered[-1] if entered else FakeStream("main of %s" % ("the current GPU" if device is None else torch.device(device)), log)

    monkeypatch.setattr(torch.cuda, "Event", FakeEvent)
    monkeypatch.setattr(torch.cuda, "stream", enter)
    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    monkeypatch.setattr(context, "group", lambda lib: contextlib.nullcontext())
    ring = context._Ring(FakeComm(log), True, place, FakeStream("side", log))
    done = ring.pass_on(torch.zeros(1), torch.zeros(1))
    ring.wait(done)
    assert log == [("side", "waits for", "main of cuda:3"), ("send", "side"), ("recv", "side"), ("main of cuda:3", "waits for", "side")]
    ring.wait(None)
    assert len(log) == 4


def test_ulysses_of_one_rank_takes_any_strides(cp):   # noqa: F811
    """As with more ranks, where the swap lays the tensors out anew."""
    from nccl_b200.parallel.context import ulysses_attention, ulysses_attention_backward
    comm = types.SimpleNamespace(nranks=1, rank=0)
    wide = [torch.randn(2, 5, heads, 20).bfloat16() for heads in (4, 2, 2)]
    q, k, v = (t[..., :16] for t in wide)
    out, state = ulysses_attention(comm, q, k, v, causal=True, cp=cp, with_state=True)
    assert out.shape == q.shape
    d = shape_at(cp.calls[0][2])
    assert list(d.q_stride) == [320, 64, 16] and list(d.k_stride) == list(d.v_stride) == [160, 32, 16]
    assert all(torch.equal(a, b) for a, b in zip(state[:3], (q, k, v)))
    grads = ulysses_attention_backward(comm, wide[0][..., 4:], state, causal=True, cp=cp)
    assert [g.shape for g in grads] == [t.shape for t in (q, k, v)] and cp.calls[1][0] == "ncclCpAttentionBackward"
    fits = [t.contiguous() for t in (q, k, v)]
    ulysses_attention(comm, *fits, cp=cp)
    assert cp.calls[2][3:6] == tuple(t.data_ptr() for t in fits)   # what fits is read where it is


@pytest.mark.parametrize("recipe", ["ring", "ulysses"])
def test_rows_off_the_16_byte_grid_are_copied(cp, recipe):   # noqa: F811
    """Contiguous tensors, too, that begin where the kernels' copies cannot."""
    from nccl_b200.parallel.context import ring_attention, ring_attention_backward, ulysses_attention, ulysses_attention_backward
    comm = types.SimpleNamespace(nranks=1, rank=0, lib=None)

    def off(*shape):   # [batch, sequence, heads, dim]
        n = torch.Size(shape).numel()
        flat = torch.randn(n + 8).bfloat16()
        begin = next(i for i in range(1, 8) if (flat.data_ptr() + 2 * i) % 16)
        return flat[begin:begin + n].view(shape)
    q, k, v, dout = off(2, 5, 4, 16), off(2, 5, 2, 16), off(2, 5, 2, 16), off(2, 5, 4, 16)
    if recipe == "ring":
        q, k, v, dout = (t.transpose(1, 2) for t in (q, k, v, dout))
        out, lse = ring_attention(comm, q, k, v, cp=cp, with_lse=True)
        grads = ring_attention_backward(comm, dout, q, k, v, out, lse, cp=cp)
    else:
        out, state = ulysses_attention(comm, q, k, v, cp=cp, with_state=True)
        grads = ulysses_attention_backward(comm, dout, state, cp=cp)
    assert [g.shape for g in grads] == [t.shape for t in (q, k, v)]
    assert all(p % 16 == 0 for call in cp.calls for p in call[3:5])
