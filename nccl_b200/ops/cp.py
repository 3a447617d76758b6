"""Attention over a sequence that is cut across ranks: what a rank computes on its own rows and on the blocks of keys and values that come to it.

    cp    = ContextParallel(comm)
    freqs = cp.rotary_frequencies(head_dim, base=500000.0)
    q, k  = cp.rotary(q, k, freqs, offset=rank * S)                    # q [B, S, heads, D], k [B, S, kv_heads, D]: this rank's rows of the sequence
    out, lse = cp.attention(q, k, v, causal=True)                      # lse [B, heads, S]: log-sum-exp of each query's scores
    dq, dk, dv = cp.attention_backward(dout, q, k, v, out, lse, causal=True)
    dq, dk = cp.rotary(dq, dk, freqs, offset=rank * S, inverse=True)   # gradients go back through the inverse

A block of keys that another rank sent joins what is there already, in fp32, and its gradients are added to those under way
(``parallel.context.ring_attention`` and ``ring_attention_backward`` do this around a ring):

    out, lse = cp.attention(q, k, v, causal=True, dtype=torch.float32)
    out, lse = cp.attention(q, k_other, v_other, join=(out, lse))      # rounded to q's type; with dtype=torch.float32 the next block can join
    delta = cp.attention_delta(dout, out)
    dq, dk, dv = cp.attention_backward(dout, q, k_other, v_other, None, lse, delta=delta, add=(dq, dk, dv), dtype=torch.float32)

A cache is read by the same call, one query or more for each sequence: ``cp.attention(q, k_cache, v_cache, causal=True, kv_lengths=lengths)``.

Every call is local to the communicator's GPU, runs on its current stream and keeps nothing: results and workspaces come from the framework's allocator, so that calls may be
captured, replayed, and made on several streams at once; no call keeps a history for autograd (gradients come from the backward calls). Reference parity: the reference has no compute kernels; programs like these use its send / receive and all-to-all
(src/collectives.cc) around their own.
"""
import ctypes
import functools
import math
import operator

from .. import _lib
from ..core import BF16, FP16, FP32, current_stream

MAGIC = 0xC9A77E17

_Strides = ctypes.c_longlong * 3


class _Attention(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("type", ctypes.c_int), ("result_type", ctypes.c_int)] + [(n, ctypes.c_int) for n in (
        "batch", "q_tokens", "kv_tokens", "heads", "kv_heads", "head_dim", "mask")] + [("scale", ctypes.c_float), ("offset", ctypes.c_longlong)] + [
            (n, _Strides) for n in ("q_stride", "k_stride", "v_stride", "dout_stride", "out_stride")]


class _Rotary(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("type", ctypes.c_int), ("batch", ctypes.c_int), ("tokens", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("half", ctypes.c_int), ("heads", ctypes.c_int * 2), ("interleaved", ctypes.c_int), ("inverse", ctypes.c_int), ("positions64", ctypes.c_int),
                ("amplitude", ctypes.c_float), ("offset", ctypes.c_longlong), ("position_stride", ctypes.c_longlong * 2), ("x_stride", _Strides * 2), ("y_stride", _Strides * 2)]


class RotaryFrequencies:
    """Turns per position of each pair of channels (fp64, on a GPU) and what the pairs are multiplied by."""

    def __init__(self, turns, amplitude):
        self.turns, self.amplitude = turns, amplitude
        self.half = turns.numel()


def rotary_turns(dim, base=10000.0, scaling=None, factor=1.0, original_length=None, low=1.0, high=4.0):
    """The turns per position of ``dim // 2`` pairs as a list of Python floats; see ``ContextParallel.rotary_frequencies``."""
    if dim <= 0 or dim % 2 or dim > 1024:
        raise ValueError("%r channels to turn: an even number, at most 1024" % (dim,))
    if not (base > 0 and factor > 0):
        raise ValueError("base = %r and factor = %r must be positive" % (base, factor))
    if scaling not in (None, "linear", "ntk", "by_parts"):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'by_parts', not %r" % (scaling,))
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("'ntk' scales the base so that the slowest pair is slowed down and the fastest is not: it needs two pairs")
        base = base * factor ** (dim / (dim - 2))
    turns = []
    for i in range(dim // 2):
        t = base ** (-2 * i / dim) / (2 * math.pi)
        if scaling == "linear":
            t /= factor
        if scaling == "by_parts":
            if not original_length or not high > low:
                raise ValueError("'by_parts' needs original_length, and high > low")
            keep = min(max((original_length * t - low) / (high - low), 0.0), 1.0)
            t *= keep + (1 - keep) / factor
        turns.append(t)
    return turns


class ContextParallel:
    def __init__(self, comm):
        import torch
        self.torch = torch
        self.comm, self.lib = comm, comm.lib
        L, P = self.lib, ctypes.c_void_p
        L.ncclCpCreate.argtypes = [P, ctypes.POINTER(P)]
        L.ncclCpDestroy.argtypes = [P]
        for name in ("ncclCpAttentionWork", "ncclCpAttentionBackwardWork"):
            getattr(L, name).argtypes = [P, P]
            getattr(L, name).restype = ctypes.c_size_t
        h = ctypes.c_void_p()
        _lib.check(L.ncclCpCreate(comm.handle, ctypes.byref(h)), "ncclCpCreate", L)
        self.handle = h
        fast = _lib.fastcall()
        self._calls = {}
        for name, words in (("ncclCpAttention", 13), ("ncclCpAttentionBackward", 19), ("ncclCpAttentionDelta", 7), ("ncclCpRotary", 9)):
            getattr(L, name).argtypes = [P] * words
            entry = _lib.address(L, name) if fast else None
            self._calls[name] = functools.partial(fast.invoke, entry) if entry else getattr(L, name)
        dev = ctypes.c_int()
        _lib.check(L.ncclCommCuDevice(comm.handle, ctypes.byref(dev)), "ncclCommCuDevice", L)
        self._device, self._place = dev.value, torch.device("cuda", dev.value)
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or current_stream
        self._codes = {torch.float16: FP16, torch.bfloat16: BF16, torch.float32: FP32}
        self._shapes = {}   # by sizes and strides: (the library's description, bytes of workspace)

    def destroy(self):
        if self.handle:
            _lib.check(self.lib.ncclCpDestroy(self.handle), "ncclCpDestroy", self.lib)
            self.handle = None

    # ------------------------------------------------------------------ calls and checks
    def _call(self, name, *args):
        if not self.handle:
            raise ValueError("this context has been destroyed")
        rc = self._calls[name](self.handle, *args, self._raw_stream(self._device))
        if rc:
            _lib.check(rc, name, self.lib)

    def _remember(self, key, make):
        """What `make`, which checks what the key says, gives for it, from the last call with that key; whoever uses it holds it, so that another thread may clear the store."""
        got = self._shapes.get(key)
        if got is None:
            got = make()
            if len(self._shapes) >= 256:
                self._shapes.clear()
            self._shapes[key] = got
        return got

    def _need(self, name, t, dtype, shape):
        """Checks a tensor: type, shape, contiguous, on the communicator's GPU."""
        if t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == self._device:
            return
        raise ValueError("%s must be a contiguous %s tensor %s on cuda:%d, not %s %s%s on %s" % (
            name, str(dtype).replace("torch.", ""), list(shape), self._device, str(t.dtype).replace("torch.", ""), list(t.shape),
            "" if t.is_contiguous() else " (strided)", t.device))

    def _result(self, name, t, dtype, shape):
        if t is None:
            return self.torch.empty(*shape, dtype=dtype, device=self._place)   # (sizes one by one: 0.7 us less than as a tuple)
        self._need(name, t, dtype, shape)
        return t

    def _operand(self, name, t, dtype, shape):
        """Checks what a tensor's sizes and strides say: type, shape, and that its rows are where the kernels' copies can begin. (Where it is, each call checks.)"""
        if t.dtype is not dtype or t.shape != shape:
            raise ValueError("%s must be a %s tensor %s, not %s %s" % (name, str(dtype).replace("torch.", ""), list(shape), str(t.dtype).replace("torch.", ""), list(t.shape)))
        st = t.stride()
        if t.numel() and ((st[3] != 1 and shape[3] > 1) or any(n > 1 and (s <= 0 or s % 8) for n, s in zip(shape[:3], st))):
            raise ValueError("%s needs its channels next to each other, rows that begin at multiples of 16 bytes, and no repeated rows, not strides %s: give a contiguous copy" % (name, list(st)))
        return st

    def _at(self, name, t):
        """Address of an operand whose sizes are checked."""
        p = t.data_ptr()
        if t.get_device() != self._device or p % 16:
            raise ValueError("%s must be on cuda:%d, at a multiple of 16 bytes, not on %s at %#x" % (name, self._device, t.device, p))
        return p

    @staticmethod
    def _tuple(name, given, n):
        given = tuple(given)
        if len(given) != n:
            raise ValueError("%s must be %d tensors, not %d" % (name, n, len(given)))
        return given

    def _lengths(self, name, t, batch):
        if t is None:
            return None
        self._need(name, t, self.torch.int32, (batch,))
        return t.data_ptr()

    def _sizes(self, q, k, v):
        if q.dim() != 4 or k.dim() != 4 or q.dtype not in (self.torch.float16, self.torch.bfloat16):
            raise ValueError("q must be an fp16 or bf16 tensor [batch, tokens, heads, channels] and k, v alike, not %s %s and %s" % (
                str(q.dtype).replace("torch.", ""), list(q.shape), list(k.shape)))
        B, Q, H, D = q.shape
        K, G = k.shape[1], k.shape[2]
        if k.shape[0] != B or k.shape[3] != D or not G or not H or H % G or H // G > 128 or not D or D % 8 or D > 128:
            raise ValueError("q %s and k %s: the same batch and channels (a multiple of 8, at most 128), heads of k that divide those of q (at most 128 to one)" % (list(q.shape), list(k.shape)))
        if max(Q, K) > 1 << 29 or B * (Q * H + K * G) >> 31:
            raise ValueError("q %s and k %s are too many rows" % (list(q.shape), list(k.shape)))
        return B, Q, K, H, G, D

    @staticmethod
    def _numbers(causal, offset, scale):
        """What a call is remembered by: numbers, where a caller has given a tensor that may hold another one next time."""
        return bool(causal), None if offset is None else operator.index(offset), None if scale is None else float(scale)

    @staticmethod
    def _mask(causal, offset, scale, D):
        """(mask, offset, scale) as the library takes them."""
        if offset is not None and not causal:
            raise ValueError("offset says where a causal mask lies: without one there is nothing to offset")
        scale = 1 / math.sqrt(D) if scale is None else scale
        if not 0 < scale < math.inf or not 0 < ctypes.c_float(scale).value < math.inf:
            raise ValueError("scale = %r must be positive and finite" % (scale,))
        if offset is not None and abs(offset) >> 62:
            raise ValueError("offset = %r" % (offset,))
        return (0 if not causal else 2 if offset is None else 1), (0 if offset is None else offset), scale

    def _describe(self, sizes, dtype, result, mask, strides, work):
        """The library's description of a call, its address, and the bytes of workspace that it takes."""
        B, Q, K, H, G, D = sizes
        d = _Attention(ctypes.sizeof(_Attention), MAGIC, self._codes[dtype], self._codes[result], B, Q, K, H, G, D, mask[0], mask[2], mask[1])
        for name, st in zip(("q_stride", "k_stride", "v_stride", "dout_stride", "out_stride"), strides):
            if st is not None:
                getattr(d, name)[:] = st[:3]
        at = ctypes.addressof(d)
        return d, at, work(self.handle, at) if work else 0

    def _work(self, size):
        return self.torch.empty(size, dtype=self.torch.uint8, device=self._place)

    def _result_type(self, dtype, q):
        dtype = q.dtype if dtype is None else dtype
        if dtype is not q.dtype and dtype is not self.torch.float32:
            raise ValueError("dtype must be %s like q, or float32, not %s" % (str(q.dtype).replace("torch.", ""), dtype))
        return dtype

    # ------------------------------------------------------------------ attention
    def attention(self, q, k, v, causal=False, offset=None, scale=None, q_lengths=None, kv_lengths=None, join=None, dtype=None, out=None, lse=None):
        """(softmax(scale q k^T) v, its log-sum-exp): [batch, queries, heads, channels] in q's type (``dtype``: or float32) and fp32 [batch, heads, queries].

        q [batch, queries, heads, channels], k and v [batch, keys, kv_heads, channels], fp16 or bf16; head h reads key head h // (heads // kv_heads). Tensors may be strided
        (slices of one projection's result, heads in front of tokens), rows at multiples of 16 bytes; channels are a multiple of 8, at most 128. ``scale``: 1 / sqrt(channels) if None.

        ``causal``: query i sees keys j <= i + ``offset``; None: the last query sees every key (offset = keys - queries of its sequence). ``q_lengths``, ``kv_lengths`` (int32
        [batch]): rows of each sequence that are there; what lies behind them may be anything, and gets zeros. A query that sees no key gets zeros and
        a log-sum-exp of -inf. ``join``: (out, lse) over other keys, fp32 (``dtype=torch.float32`` gives that): the result is over both; they may be ``out`` and ``lse``.

        Sums and statistics are fp32; probabilities are rounded to q's type (by at most half a step each) before they meet v."""
        torch = self.torch
        causal, offset, scale = self._numbers(causal, offset, scale)

        def make():
            sizes = B, Q, K, H, G, D = self._sizes(q, k, v)
            strides = self._operand("q", q, q.dtype, (B, Q, H, D)), self._operand("k", k, q.dtype, (B, K, G, D)), self._operand("v", v, q.dtype, (B, K, G, D))
            result = self._result_type(dtype, q)
            like = result is q.dtype and q.is_contiguous()   # (the result is: 0.3 us less to ask for)
            return sizes, result, like, self._describe(sizes, q.dtype, result, self._mask(causal, offset, scale, D), strides, self.lib.ncclCpAttentionWork)
        (B, Q, K, H, G, D), result, like, (d, at, size) = self._remember(
            (q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, causal, offset, scale, dtype), make)
        pq, pk, pv = self._at("q", q), self._at("k", k), self._at("v", v)
        nq, nk = self._lengths("q_lengths", q_lengths, B), self._lengths("kv_lengths", kv_lengths, B)
        join_out = join_lse = None
        if join is not None:
            join = self._tuple("join", join, 2)
            self._need("join[0]", join[0], torch.float32, (B, Q, H, D))
            self._need("join[1]", join[1], torch.float32, (B, H, Q))
            join_out, join_lse = join[0].data_ptr(), join[1].data_ptr()
        out = torch.empty_like(q) if like and out is None else self._result("out", out, result, (B, Q, H, D))
        lse = self._result("lse", lse, torch.float32, (B, H, Q))
        work = self._work(size) if size else None   # (held until the call is made)
        self._call("ncclCpAttention", at, pq, pk, pv, nq, nk, join_out, join_lse, out.data_ptr(), lse.data_ptr(), work.data_ptr() if size else None)
        return out, lse

    def attention_delta(self, dout, out, q_lengths=None, delta=None):
        """fp32 [batch, heads, queries]: <dout, out> of each row, which every backward call of these queries needs. Where the log-sum-exp has a gradient of its own, subtract it:
        of any size, also in fp16. (Of queries that see no key what is here is not used.)"""
        if out.dim() != 4 or out.dtype not in (self.torch.float16, self.torch.bfloat16):
            raise ValueError("out must be an fp16 or bf16 tensor [batch, tokens, heads, channels], not %s %s" % (str(out.dtype).replace("torch.", ""), list(out.shape)))
        B, Q, H, D = out.shape

        def make():
            sizes = self._sizes(out, out, out)
            strides = None, None, None, self._operand("dout", dout, out.dtype, (B, Q, H, D)), self._operand("out", out, out.dtype, (B, Q, H, D))
            return self._describe(sizes, out.dtype, out.dtype, (0, 0, 1.0), strides, None)
        d, at, _ = self._remember((out.shape, out.stride(), out.dtype, dout.shape, dout.stride(), dout.dtype), make)
        nq = self._lengths("q_lengths", q_lengths, B)
        delta = self._result("delta", delta, self.torch.float32, (B, H, Q))
        self._call("ncclCpAttentionDelta", at, self._at("dout", dout), self._at("out", out), nq, delta.data_ptr())
        return delta

    def attention_backward(self, dout, q, k, v, out, lse, causal=False, offset=None, scale=None, q_lengths=None, kv_lengths=None, delta=None, add=None, dtype=None, dq=None, dk=None,
                           dv=None):
        """(dq, dk, dv) of ``attention`` from the gradient of its result, laid out like q, k and v, in q's type (``dtype``: or float32); the probabilities are computed again
        from ``lse``. Mask, scale and lengths as the forward call had them; rows behind the lengths get zeros.

        ``out`` and ``lse`` are the result over all keys of the queries: where blocks were joined, the last one's. ``delta``: what ``attention_delta`` gives (out may then be
        None). A ``delta`` of any size, and one that the keys of other calls have a part in, are taken in fp16 too. ``add``: fp32 (dq, dk, dv) so far, to which these are added; they may be the results' tensors. The same call gives the same bits."""
        torch = self.torch
        causal, offset, scale = self._numbers(causal, offset, scale)

        def make():
            sizes = B, Q, K, H, G, D = self._sizes(q, k, v)
            strides = (self._operand("q", q, q.dtype, (B, Q, H, D)), self._operand("k", k, q.dtype, (B, K, G, D)), self._operand("v", v, q.dtype, (B, K, G, D)),
                       self._operand("dout", dout, q.dtype, (B, Q, H, D)), None if out is None else self._operand("out", out, q.dtype, (B, Q, H, D)))
            result = self._result_type(dtype, q)
            return sizes, result, self._describe(sizes, q.dtype, result, self._mask(causal, offset, scale, D), strides, self.lib.ncclCpAttentionBackwardWork)
        (B, Q, K, H, G, D), result, (d, at, size) = self._remember(
            (q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, causal, offset, scale, dtype, dout.shape, dout.stride(), dout.dtype,
             None if out is None else (out.shape, out.stride(), out.dtype)), make)
        if out is None and delta is None:
            raise ValueError("out or delta must be given")
        pd, pq, pk, pv, po = self._at("dout", dout), self._at("q", q), self._at("k", k), self._at("v", v), None if out is None else self._at("out", out)
        self._need("lse", lse, torch.float32, (B, H, Q))
        if delta is not None:
            self._need("delta", delta, torch.float32, (B, H, Q))
        nq, nk = self._lengths("q_lengths", q_lengths, B), self._lengths("kv_lengths", kv_lengths, B)
        sq, sk = (B, Q, H, D), (B, K, G, D)
        given = (None, None, None)
        if add is not None:
            add = self._tuple("add", add, 3)
            for name, t, shape in zip(("add[0]", "add[1]", "add[2]"), add, (sq, sk, sk)):
                self._need(name, t, torch.float32, shape)
            given = [t.data_ptr() for t in add]
        dq, dk, dv = self._result("dq", dq, result, sq), self._result("dk", dk, result, sk), self._result("dv", dv, result, sk)
        work = self._work(size) if size else None   # (held until the call is made)
        self._call("ncclCpAttentionBackward", at, pd, pq, pk, pv, po, lse.data_ptr(), None if delta is None else delta.data_ptr(), nq, nk, *given, dq.data_ptr(), dk.data_ptr(),
                   dv.data_ptr(), work.data_ptr() if size else None)
        return dq, dk, dv

    # ------------------------------------------------------------------ rotary positions
    def rotary_frequencies(self, dim, base=10000.0, scaling=None, factor=1.0, original_length=None, low=1.0, high=4.0, amplitude=1.0):
        """What ``rotary`` takes: pair i of ``dim // 2`` turns by base ** (-2 i / dim) per position. For contexts ``factor`` times as long as a model was trained on,
        ``scaling``: "linear" slows every pair down by the factor; "ntk" raises the base so that the slowest pair is slowed down by it and the fastest is not;
        "by_parts" slows down pairs that make fewer than ``low`` turns in ``original_length`` positions, leaves those with more than ``high`` as they are, and blends between.
        ``amplitude`` multiplies the turned channels."""
        if not math.isfinite(amplitude):
            raise ValueError("amplitude = %r must be finite" % (amplitude,))
        return RotaryFrequencies(self.torch.tensor(rotary_turns(dim, base, scaling, factor, original_length, low, high), dtype=self.torch.float64, device=self._place), float(amplitude))

    def rotary(self, q, k, freqs, positions=None, offset=0, interleaved=False, inverse=False, out=None):
        """(q, k) with their first 2 * freqs.half channels turned by position, the others as they are; k may be None (and is then None).

        q, k [batch, tokens, heads, channels], fp16, bf16 or fp32, any strides with channels next to each other. The position of a token is ``positions`` (int32 or int64 [batch, tokens]),
        or ``offset`` + its index: a rank that holds rows from `begin` on gives ``offset=begin``. Pairs are channels (i, i + half), with ``interleaved`` (2 i, 2 i + 1).
        ``inverse`` turns back: the gradient's way. ``out``: (q, k) tensors for the results, which may be q and k themselves. Angles are reduced to a turn in 64 bits."""
        torch = self.torch
        if not isinstance(freqs, RotaryFrequencies):
            raise ValueError("freqs must come from rotary_frequencies")
        yq, yk = (None, None) if out is None else out
        offset, interleaved, inverse = operator.index(offset), bool(interleaved), bool(inverse)

        def make():
            if q.dim() != 4 or q.dtype not in self._codes or (k is not None and (k.dim() != 4 or k.dtype is not q.dtype or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
                raise ValueError("q and k must be fp16, bf16 or fp32 tensors [batch, tokens, heads, channels] that differ in heads only, not %s %s and %s" % (
                    str(q.dtype).replace("torch.", ""), list(q.shape), None if k is None else [str(k.dtype).replace("torch.", ""), list(k.shape)]))
            B, T, _, D = q.shape
            if 2 * freqs.half > D:
                raise ValueError("frequencies of %d channels, and heads of %d" % (2 * freqs.half, D))
            if B * T >> 31 or abs(offset) >> 62:
                raise ValueError("%d sequences of %d tokens, offset %r" % (B, T, offset))
            d = _Rotary(ctypes.sizeof(_Rotary), MAGIC, self._codes[q.dtype], B, T, D, freqs.half)
            d.interleaved, d.inverse, d.amplitude, d.offset = interleaved, inverse, freqs.amplitude, offset
            if positions is not None:
                if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (B, T) or min(positions.stride()) < 0:
                    raise ValueError("positions must be an int32 or int64 tensor [%d, %d], not %s %s" % (B, T, str(positions.dtype).replace("torch.", ""), list(positions.shape)))
                d.positions64, d.position_stride[:] = positions.dtype is torch.int64, positions.stride()
            for i, (x, y) in enumerate(((q, yq), (k, yk))):
                if x is None:
                    continue
                if not x.shape[2] or (x.stride(3) != 1 and D > 1):
                    raise ValueError("q and k must have heads, and channels next to each other: %s, strides %s" % (list(x.shape), list(x.stride())))
                if y is not None and (y.dtype is not x.dtype or y.shape != x.shape or (y.stride(3) != 1 and D > 1)):
                    raise ValueError("results must be like q and k, with channels next to each other")
                d.heads[i] = x.shape[2]
                d.x_stride[i][:] = x.stride()[:3]
                d.y_stride[i][:] = (x.shape[1] * x.shape[2] * D, x.shape[2] * D, D) if y is None else y.stride()[:3]
            return d, ctypes.addressof(d), q.is_contiguous(), k is not None and k.is_contiguous()
        d, at, q_like, k_like = self._remember((q.shape, q.stride(), q.dtype, None if k is None else (k.shape, k.stride(), k.dtype), freqs.half, freqs.amplitude, interleaved, inverse, offset,
                                None if positions is None else (positions.shape, positions.stride(), positions.dtype),
                                None if yq is None else (yq.shape, yq.stride(), yq.dtype), None if yk is None else (yk.shape, yk.stride(), yk.dtype)), make)
        dev = self._device
        if yq is None:
            yq = torch.empty_like(q) if q_like else torch.empty(*q.shape, dtype=q.dtype, device=self._place)
        if k is None:
            yk, pk, to = None, None, None
        else:
            if yk is None:
                yk = torch.empty_like(k) if k_like else torch.empty(*k.shape, dtype=k.dtype, device=self._place)
            if k.get_device() != dev or yk.get_device() != dev:
                raise ValueError("k and its result must be on cuda:%d, not on %s and %s" % (dev, k.device, yk.device))
            pk, to = k.data_ptr(), yk.data_ptr()
        if q.get_device() != dev or yq.get_device() != dev:
            raise ValueError("q and its result must be on cuda:%d, not on %s and %s" % (dev, q.device, yq.device))
        if freqs.turns.get_device() != self._device or (positions is not None and positions.get_device() != self._device):
            raise ValueError("frequencies and positions must be on cuda:%d" % self._device)
        self._call("ncclCpRotary", at, q.data_ptr(), pk, yq.data_ptr(), to, None if positions is None else positions.data_ptr(), freqs.turns.data_ptr())
        return yq, yk
