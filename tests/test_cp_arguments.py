"""What the context-parallel operators refuse before anything reaches a GPU, and what they hand to the library: tensors in host memory, with the library's calls
recorded."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture()
def cp():
    from nccl_b200.core import BF16, FP16, FP32
    from nccl_b200.ops.cp import ContextParallel
    c = ContextParallel.__new__(ContextParallel)
    c.torch, c._device, c._place, c.handle, c._shapes = torch, -1, torch.device("cpu"), 111, {}
    c._raw_stream, c._codes = (lambda device: 222), {torch.float16: FP16, torch.bfloat16: BF16, torch.float32: FP32}
    c.calls = []

    class Lib:
        @staticmethod
        def ncclCpAttentionWork(handle, at):
            return 0

        @staticmethod
        def ncclCpAttentionBackwardWork(handle, at):
            return 64

    c.lib = Lib()

    def record(name):
        def call(*args):
            c.calls.append((name,) + args)
            return 0
        return call

    c._calls = {n: record(n) for n in ("ncclCpAttention", "ncclCpAttentionBackward", "ncclCpAttentionDelta", "ncclCpRotary")}
    return c


def qkv(B=2, Q=5, K=7, H=4, G=2, D=16, dtype=torch.bfloat16):
    return torch.randn(B, Q, H, D).to(dtype), torch.randn(B, K, G, D).to(dtype), torch.randn(B, K, G, D).to(dtype)


def shape_at(at):
    from nccl_b200.ops.cp import _Attention
    return ctypes.cast(at, ctypes.POINTER(_Attention)).contents


def test_attention_hands_over_its_shape(cp):
    from nccl_b200.ops.cp import MAGIC, _Attention
    q, k, v = qkv()
    lengths = torch.tensor([7, 3], dtype=torch.int32)
    out, lse = cp.attention(q, k, v, causal=True, kv_lengths=lengths)
    name, handle, at, pq, pk, pv, nq, nk, jo, jl, po, pl, work, stream = cp.calls[0]
    assert (name, handle, pq, pk, pv, nq, nk, jo, jl, po, pl, work, stream) == ("ncclCpAttention", 111, q.data_ptr(), k.data_ptr(), v.data_ptr(), None, lengths.data_ptr(), None, None,
                                                                                out.data_ptr(), lse.data_ptr(), None, 222)
    d = shape_at(at)
    assert (d.size, d.magic, d.type, d.result_type) == (ctypes.sizeof(_Attention), MAGIC, 9, 9)
    assert (d.batch, d.q_tokens, d.kv_tokens, d.heads, d.kv_heads, d.head_dim, d.mask, d.offset) == (2, 5, 7, 4, 2, 16, 2, 0) and math.isclose(d.scale, 0.25)
    assert list(d.q_stride) == [5 * 64, 64, 16] and list(d.k_stride) == list(d.v_stride) == [7 * 32, 32, 16]
    assert out.dtype == torch.bfloat16 and out.shape == q.shape and lse.dtype == torch.float32 and lse.shape == (2, 4, 5)
    join = torch.zeros(2, 5, 4, 16), torch.zeros(2, 4, 5)
    got = cp.attention(q.half(), k.half(), v.half(), causal=True, offset=-3, scale=2, join=join, dtype=torch.float32, out=join[0], lse=join[1])
    d = shape_at(cp.calls[1][2])
    assert got[0] is join[0] and got[1] is join[1] and cp.calls[1][8:10] == (join[0].data_ptr(), join[1].data_ptr())
    assert (d.type, d.result_type, d.mask, d.offset, d.scale) == (6, 7, 1, -3, 2.0)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    cp.attention(heads_first, k, v)
    d = shape_at(cp.calls[2][2])
    assert list(d.q_stride) == [5 * 64, 16, 80] and d.mask == 0
    for i in range(600):   # descriptions do not pile up
        cp.attention(q, k, v, scale=1.0 + i)
    assert len(cp._shapes) <= 256


def test_a_shape_in_use_outlives_the_store(cp):
    import weakref
    q, k, v = qkv()
    result, kept, alive = cp._result, [], []

    def clearing(*args):
        kept.extend(weakref.ref(s[-1][0]) for s in cp._shapes.values())
        cp._shapes.clear()
        return result(*args)

    cp._result = clearing
    cp._calls["ncclCpAttention"] = cp._calls["ncclCpAttentionBackward"] = lambda *args: alive.append(kept[-1]() is not None) or 0
    out, lse = cp.attention(q, k, v)
    cp.attention_backward(out, q, k, v, out, lse)
    assert alive == [True, True]


def bad_operands(t):
    other = torch.randn(*t.shape[:3], 2 * t.shape[3]).to(t.dtype)
    return [t.float(), t[0], t[..., :12], other[..., ::2], t[:1].expand_as(t), torch.randn(*t.shape[:3], 20).to(t.dtype)[..., :16]]


def test_attention_refuses(cp):
    q, k, v = qkv()
    for i in range(3):
        for bad in bad_operands((q, k, v)[i]):
            args = [q, k, v]
            args[i] = bad
            with pytest.raises(ValueError):
                cp.attention(*args)
    flat = torch.randn(2 * 5 * 64 + 8).bfloat16()
    base = next(i for i in range(1, 8) if (flat.data_ptr() + 2 * i) % 16)
    with pytest.raises(ValueError):   # rows off the 16-byte grid
        cp.attention(flat[base:base + 640].view(2, 5, 4, 16), k, v)
    five = torch.randn(2, 7, 5, 16).bfloat16()
    wide = torch.randn(2, 5, 4, 136).bfloat16()
    many = torch.randn(1, 1, 258, 8).bfloat16()
    for args in ((q, five, five), (q, k, v[:, :6]), (q, k[:1], v[:1]), (wide, wide, wide), (q, k[:, :, :0], v[:, :, :0]), (many, many[:, :, :2], many[:, :, :2])):
        with pytest.raises(ValueError):
            cp.attention(*args)
    lse, o32 = torch.zeros(2, 4, 5), torch.zeros(2, 5, 4, 16)
    i32 = torch.tensor([1, 2], dtype=torch.int32)
    for kw in (dict(offset=1), dict(scale=0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(scale=1e-60), dict(dtype=torch.float16), dict(q_lengths=i32.long()),
               dict(kv_lengths=i32[:1]), dict(join=(o32.bfloat16(), lse)), dict(join=(o32, lse[:1])), dict(join=(o32[:, :, :, :8], lse)), dict(out=o32), dict(lse=lse.double()),
               dict(causal=True, offset=1 << 62), dict(dtype=torch.float32, out=o32.bfloat16())):
        with pytest.raises(ValueError):
            cp.attention(q, k, v, **kw)
    assert not cp.calls
    cp.handle = None
    with pytest.raises(ValueError):
        cp.attention(q, k, v)


def test_backward_hands_over_and_refuses(cp):
    q, k, v = qkv()
    out, lse = cp.attention(q, k, v, causal=True, offset=2)
    dout = torch.randn_like(q)
    dq, dk, dv = cp.attention_backward(dout, q, k, v, out, lse, causal=True, offset=2)
    name, handle, at, pd, pq, pk, pv, po, pl, delta, nq, nk, a0, a1, a2, gq, gk, gv, work, stream = cp.calls[-1]
    assert (name, pd, pq, pk, pv, po, pl, delta, nq, nk, a0, a1, a2) == ("ncclCpAttentionBackward", dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                                                                         None, None, None, None, None, None)
    assert (gq, gk, gv, stream) == (dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), 222) and work
    assert dq.shape == q.shape and dk.shape == dv.shape == k.shape and dq.dtype == torch.bfloat16
    delta = cp.attention_delta(dout, out)
    assert delta.shape == lse.shape and cp.calls[-1][0] == "ncclCpAttentionDelta"
    sums = torch.zeros(q.shape), torch.zeros(k.shape), torch.zeros(k.shape)
    got = cp.attention_backward(dout, q, k, v, None, lse, delta=delta, add=sums, dtype=torch.float32, dq=sums[0], dk=sums[1], dv=sums[2])
    assert all(a is b for a, b in zip(got, sums)) and cp.calls[-1][12:18] == tuple(t.data_ptr() for t in sums + sums) and cp.calls[-1][7] is None
    n = len(cp.calls)
    for bad in bad_operands(dout):
        with pytest.raises(ValueError):
            cp.attention_backward(bad, q, k, v, out, lse)
        with pytest.raises(ValueError):
            cp.attention_backward(dout, q, k, v, bad, lse)
        with pytest.raises(ValueError):
            cp.attention_delta(bad, out)
    for args, kw in (((dout, q, k, v, None, lse), {}), ((dout, q, k, v, out, lse.half()), {}), ((dout, q, k, v, out, lse[:, :2]), {}), ((dout, q, k, v, out, lse), dict(delta=delta[..., :2])),
                     ((dout, q, k, v, out, lse), dict(add=(sums[0], sums[1], sums[2].half()))), ((dout, q, k, v, out, lse), dict(dq=sums[0])),
                     ((dout, q, k, v, out, lse), dict(dtype=torch.float32, dk=dk)), ((dout, q, k, v, out, lse), dict(offset=1)), ((dout, q, k, v, out, lse), dict(scale=0))):
        with pytest.raises(ValueError):
            cp.attention_backward(*args, **kw)
    with pytest.raises(ValueError):
        cp.attention_delta(dout, out.float())
    assert len(cp.calls) == n


def test_rotary_hands_over_and_refuses(cp):
    from nccl_b200.ops.cp import MAGIC, _Rotary
    freqs = cp.rotary_frequencies(12, base=100.0, amplitude=0.5)
    q, k = torch.randn(2, 5, 4, 16), torch.randn(2, 5, 1, 16)
    at = torch.arange(10).view(2, 5)
    a, b = cp.rotary(q, k, freqs, positions=at, interleaved=True, inverse=True)
    name, handle, d, x0, x1, y0, y1, pos, turns, stream = cp.calls[0]
    assert (name, x0, x1, y0, y1, pos, turns) == ("ncclCpRotary", q.data_ptr(), k.data_ptr(), a.data_ptr(), b.data_ptr(), at.data_ptr(), freqs.turns.data_ptr())
    d = ctypes.cast(d, ctypes.POINTER(_Rotary)).contents
    assert (d.size, d.magic, d.type, d.batch, d.tokens, d.head_dim, d.half, list(d.heads)) == (ctypes.sizeof(_Rotary), MAGIC, 7, 2, 5, 16, 6, [4, 1])
    assert (d.interleaved, d.inverse, d.positions64, d.amplitude, list(d.position_stride)) == (1, 1, 1, 0.5, [5, 1])
    assert list(d.x_stride[0]) == list(d.y_stride[0]) == [320, 64, 16] and list(d.x_stride[1]) == [80, 16, 16]
    assert torch.allclose(freqs.turns, torch.tensor([100.0 ** (-2 * i / 12) / (2 * math.pi) for i in range(6)], dtype=torch.float64), rtol=1e-15)
    t = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert cp.rotary(t, None, freqs, offset=3, out=(t, None)) == (t, None)
    d = ctypes.cast(cp.calls[1][2], ctypes.POINTER(_Rotary)).contents
    assert list(d.y_stride[0]) == [320, 16, 80] and d.offset == 3 and list(d.heads) == [4, 0] and cp.calls[1][3] == cp.calls[1][5] and cp.calls[1][4] is None and cp.calls[1][7] is None
    n = len(cp.calls)
    for args, kw in (((q.double(), None, freqs), {}), ((q[0], None, freqs), {}), ((q, k.half(), freqs), {}), ((q, k[:, :4], freqs), {}), ((q, k[..., :8], freqs), {}),
                     ((q[..., ::2], None, freqs), {}), ((q[..., :8], None, freqs), {}), ((q, None, freqs.turns), {}), ((q, k, freqs), dict(positions=at.float())),
                     ((q, k, freqs), dict(positions=at[:1])), ((q, k, freqs), dict(out=(q, k.half()))), ((q, k, freqs), dict(out=(q[:, :4], k))), ((q, k, freqs), dict(offset=1 << 62)),
                     ((q[:, :, :0], None, freqs), {})):
        with pytest.raises(ValueError):
            cp.rotary(*args, **kw)
    for args, kw in (((3,), {}), ((0,), {}), ((2048,), {}), ((8,), dict(base=0)), ((8,), dict(scaling="half")), ((2,), dict(scaling="ntk", factor=2)), ((8,), dict(scaling="by_parts", factor=2)),
                     ((8,), dict(scaling="by_parts", factor=2, original_length=10, low=4, high=4)), ((8,), dict(amplitude=math.inf)), ((8,), dict(factor=0, scaling="linear"))):
        with pytest.raises(ValueError):
            cp.rotary_frequencies(*args, **kw)
    assert len(cp.calls) == n


def test_scaled_frequencies():
    from nccl_b200.ops.cp import rotary_turns
    plain = rotary_turns(16, 10000.0)
    assert rotary_turns(16, 10000.0, "linear", 4.0) == [t / 4 for t in plain]
    ntk = rotary_turns(16, 10000.0, "ntk", 4.0)
    assert math.isclose(ntk[0], plain[0]) and math.isclose(ntk[-1], plain[-1] / 4)   # the fastest pair keeps its speed, the slowest is four times slower
    parts = rotary_turns(16, 10000.0, "by_parts", 4.0, original_length=1000, low=1.0, high=4.0)
    for p, t in zip(parts, plain):
        turns = 1000 * t
        keep = 1.0 if turns >= 4 else 0.0 if turns <= 1 else (turns - 1) / 3
        assert math.isclose(p, t * keep + t / 4 * (1 - keep), rel_tol=1e-14)
    assert any(p == t for p, t in zip(parts, plain)) and any(math.isclose(p, t / 4) for p, t in zip(parts, plain))


def test_entry_points_without_a_context(lib):
    """Null contexts, and communicators without a GPU, are refused."""
    import os
    from nccl_b200 import Communicator, get_unique_id
    vp = ctypes.c_void_p
    for name, words in (("ncclCpAttention", 13), ("ncclCpAttentionBackward", 19), ("ncclCpAttentionDelta", 7), ("ncclCpRotary", 9)):
        fn = getattr(lib, name)
        fn.argtypes = [vp] * words
        assert fn(*[None] * words) == 4
    for name in ("ncclCpAttentionWork", "ncclCpAttentionBackwardWork"):
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = [vp, vp], ctypes.c_size_t
        assert fn(None, None) == 0
    assert lib.ncclCpDestroy(None) == 0
    before = os.environ.get("NCCL_B200_HOST_ONLY")
    os.environ["NCCL_B200_HOST_ONLY"] = "1"
    try:
        comm = Communicator(1, 0, get_unique_id())
        h = vp()
        lib.ncclCpCreate.argtypes = [vp, ctypes.POINTER(vp)]
        assert lib.ncclCpCreate(comm.handle, ctypes.byref(h)) == 4 and not h.value
        comm.destroy()
    finally:
        if before is None:
            del os.environ["NCCL_B200_HOST_ONLY"]
        else:
            os.environ["NCCL_B200_HOST_ONLY"] = before
