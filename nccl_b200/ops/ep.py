"""Expert-parallel MoE dispatch / combine on torch tensors (wraps the ncclEp* C API).

    ep = ExpertParallel(comm, num_experts=256, max_tokens=4096, hidden=7168)
    toks, scales, counts = ep.dispatch(x, topk_idx, topk_weights, fp8=True)
        # toks [E_local, n*max_tokens, hidden] (e4m3 bytes), scales [E_local, n*max_tokens, hidden/128], counts [E_local]
    y = experts(toks, scales, counts)           # bf16 [E_local, n*max_tokens, hidden]
    out = ep.combine(y)                         # bf16 [tokens, hidden]: sum_k w[t,k] * y(expert k of t)

Layouts with one copy of a token per destination rank instead of one per expert (fewer bytes when a token selects
several experts of one rank): ``layout="rank_major"`` gives toks [n, max_tokens, hidden] (row = source rank, token
index) and ``layout="flat"`` gives the received tokens packed as [n*max_tokens, hidden]; both also return the routing
rows ``ep.recv_topk_idx`` (expert ids that are local to this rank, else -1) and ``ep.recv_topk_weights``. The caller
applies its local experts and the weights and gives one pre-reduced row per received token to ``combine``.

The rest of a mixture-of-experts layer, forward and backward, on the rows of the default layout (``fp8=False``):

    idx, weights = ep.route(logits, topk, score="sigmoid", bias=balance, groups=8, keep_groups=4, group_score="top2", scale=2.5)
    toks, _, counts = ep.dispatch(x, idx, weights, fp8=False)
    pre = torch.empty(ep.El, ep.cap, 2 * ffn, dtype=torch.float32, device="cuda")       # (or bf16: half the memory, less exact gradients)
    act = ep.expert_linear(toks, w_gate_up, counts, activation="swiglu", pre=pre)       # w_gate_up [El, 2 * ffn, hidden]
    y = ep.expert_linear(act, w_down, counts)                                           # w_down [El, hidden, ffn]
    out = ep.combine(y)

    rows = ep.dispatch_rows()                                                           # (before the next dispatch)
    dy, dweights = ep.combine_backward(dout, y, weights, rows)
    dact, dw_down, _ = ep.expert_linear_backward(dy, act, w_down, counts)
    dtoks, dw_gate_up, _ = ep.expert_linear_backward(dact, toks, w_gate_up, counts, pre=pre, activation="swiglu")
    dx = ep.dispatch_backward(dtoks, rows)
    dlogits = ep.route_backward(dweights, logits, idx, score="sigmoid", scale=2.5)
"""
import ctypes
import functools

from .. import _lib
from ..core import BF16, FP16, FP32, INT64, current_stream

EP_MAGIC = 0xC00FFFEE
TENSOR_MAGIC = 0xCAFECAFE


class EpTensor(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("ndim", ctypes.c_uint), ("datatype", ctypes.c_int),
                ("data", ctypes.c_void_p), ("win_hdl", ctypes.c_void_p), ("win_offset", ctypes.c_uint64),
                ("sizes", ctypes.POINTER(ctypes.c_size_t))]


class AllocCfg(ctypes.Structure):
    _fields_ = [("alloc_fn", ctypes.c_void_p), ("free_fn", ctypes.c_void_p), ("context", ctypes.c_void_p)]


class GroupCfg(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("version", ctypes.c_uint), ("algorithm", ctypes.c_int),
                ("num_experts", ctypes.c_uint), ("max_dispatch_tokens_per_rank", ctypes.c_uint), ("max_recv_tokens_per_rank", ctypes.c_uint),
                ("max_token_bytes", ctypes.c_uint), ("rdma_buffer_size", ctypes.c_ulong), ("num_qp_per_rank", ctypes.c_uint),
                ("num_channels", ctypes.c_uint), ("max_num_sms", ctypes.c_uint), ("alloc", AllocCfg), ("enable_mask", ctypes.c_uint),
                ("timeout_ns", ctypes.c_uint64)]


class LayoutInfo(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("expert_counters", ctypes.POINTER(EpTensor)),
                ("src_rank_counters", ctypes.POINTER(EpTensor)), ("expert_offsets", ctypes.POINTER(EpTensor)),
                ("recv_total_counter", ctypes.POINTER(EpTensor))]


class DispIn(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("tokens", ctypes.POINTER(EpTensor)),
                ("topk_weights", ctypes.POINTER(EpTensor)), ("scales", ctypes.POINTER(EpTensor))]


class DispOut(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("tokens", ctypes.POINTER(EpTensor)),
                ("topk_weights", ctypes.POINTER(EpTensor)), ("scales", ctypes.POINTER(EpTensor)), ("topk_idx", ctypes.POINTER(EpTensor))]


class DispCfg(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("send_only", ctypes.c_uint), ("round_scales", ctypes.c_uint), ("pass_direction", ctypes.c_int)]


class CombCfg(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("send_only", ctypes.c_uint), ("pass_direction", ctypes.c_int)]


class CombIO(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("tokens", ctypes.POINTER(EpTensor)), ("topk_weights", ctypes.POINTER(EpTensor))]


class RouteCfg(ctypes.Structure):
    _fields_ = [("size", ctypes.c_uint), ("magic", ctypes.c_uint), ("score", ctypes.c_int), ("groups", ctypes.c_int), ("keep_groups", ctypes.c_int),
                ("group_score", ctypes.c_int), ("renormalize", ctypes.c_int), ("scale", ctypes.c_float)]


def _tensor(t, code):
    sizes = (ctypes.c_size_t * t.dim())(*t.shape)
    et = EpTensor(ctypes.sizeof(EpTensor), TENSOR_MAGIC, t.dim(), code, t.data_ptr(), None, 0, sizes)
    et._keep = (sizes, t)
    return et


def _hdr(s):
    s.size = ctypes.sizeof(s)
    s.magic = EP_MAGIC
    return s


class ExpertParallel:
    LAYOUTS = {"expert_major": 1, "rank_major": 2, "flat": 3}
    SCORES = {"softmax": 0, "sigmoid": 1}
    GROUP_SCORES = {"max": 0, "top2": 1}
    PRE_FP32 = 256   # beside the activation's code
    ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3, "swiglu": 4, "geglu": 5}

    def __init__(self, comm, num_experts, max_tokens, hidden, max_sms=0, timeout_ms=0, enable_mask=False, layout="expert_major"):
        import torch
        self.torch = torch
        self.layout = layout
        self.layout_code = self.LAYOUTS[layout]
        self.comm, self.lib = comm, comm.lib
        self.E, self.n, self.H, self.max_tokens = num_experts, comm.nranks, hidden, max_tokens
        self.El = num_experts // comm.nranks
        self.cap = comm.nranks * max_tokens
        L = self.lib
        vp, pvp = ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)
        L.ncclEpCreateGroup.argtypes = [pvp, vp, ctypes.POINTER(GroupCfg)]
        L.ncclEpGroupDestroy.argtypes = [vp]
        L.ncclEpCreateHandle.argtypes = [pvp, vp, ctypes.c_int, ctypes.POINTER(EpTensor), vp, vp, vp]
        L.ncclEpUpdateHandle.argtypes = [vp, ctypes.POINTER(EpTensor), vp, vp]
        L.ncclEpHandleDestroy.argtypes = [vp]
        L.ncclEpDispatch.argtypes = [vp, ctypes.POINTER(DispIn), ctypes.POINTER(DispOut), ctypes.POINTER(LayoutInfo), ctypes.POINTER(DispCfg), vp]
        L.ncclEpCombine.argtypes = [vp, ctypes.POINTER(CombIO), ctypes.POINTER(CombIO), ctypes.POINTER(CombCfg), vp]
        L.ncclEpComplete.argtypes = [vp, vp, vp]
        dims = [ctypes.c_int, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t]
        L.b200EpDispatch.argtypes = [vp] + ([vp] + dims) * 4 + [vp] * 5 + [ctypes.c_int, vp]
        L.b200EpCombine.argtypes = [vp] + ([vp] + dims) * 2 + [ctypes.c_int, vp]
        L.ncclEpMaskQuery.argtypes = [vp, ctypes.POINTER(ctypes.c_int), vp]
        L.ncclEpMaskUpdate.argtypes = [vp, ctypes.POINTER(ctypes.c_int), vp]
        L.ncclEpMaskClean.argtypes = [vp, vp]
        cfg = _hdr(GroupCfg())
        cfg.version = 1
        cfg.num_experts = num_experts
        cfg.max_dispatch_tokens_per_rank = max_tokens
        cfg.max_token_bytes = hidden * 2
        cfg.max_num_sms = max_sms
        cfg.timeout_ns = timeout_ms * 1000000
        cfg.enable_mask = 1 if enable_mask else 0
        g = ctypes.c_void_p()
        _lib.check(L.ncclEpCreateGroup(ctypes.byref(g), comm.handle, ctypes.byref(cfg)), "ncclEpCreateGroup", L)
        self.group = g
        self._lead = {"expert_major": (self.El, self.cap), "rank_major": (self.n, max_tokens), "flat": (self.cap,)}[layout]
        fast = _lib.fastcall()
        entries = [_lib.address(L, name) for name in ("b200EpDispatch", "b200EpCombine")]
        self._fast = (fast.invoke, *entries) if fast and all(entries) else None
        self._moe_protos(fast)
        self.handle = None
        self._keep = None
        self.recv_total = None

    def destroy(self):
        if self.handle:
            self.lib.ncclEpHandleDestroy(self.handle)
            self.handle = None
        if self.group:
            self.lib.ncclEpGroupDestroy(self.group)
            self.group = None

    def _stream(self):
        return current_stream()

    def complete(self):
        """Runs the receiving half of the last ``send_only`` dispatch / combine."""
        _lib.check(self.lib.ncclEpComplete(self.handle, None, self._stream()), "ncclEpComplete", self.lib)

    def mask(self):
        """Which ranks this rank leaves out (1 = left out)."""
        m = (ctypes.c_int * self.n)()
        _lib.check(self.lib.ncclEpMaskQuery(self.group, m, self._stream()), "ncclEpMaskQuery", self.lib)
        return list(m)

    def set_mask(self, mask):
        m = (ctypes.c_int * self.n)(*mask)
        _lib.check(self.lib.ncclEpMaskUpdate(self.group, m, self._stream()), "ncclEpMaskUpdate", self.lib)

    def clear_mask(self):
        _lib.check(self.lib.ncclEpMaskClean(self.group, self._stream()), "ncclEpMaskClean", self.lib)

    @staticmethod
    def _dims(t):
        """Dimensions and their sizes as the flat entry points take them."""
        d = t.shape
        return (3, d[0], d[1], d[2]) if len(d) == 3 else (2, d[0], d[1], 0) if len(d) == 2 else (len(d), 0, 0, 0)

    def dispatch(self, x, topk_idx, topk_weights, fp8=True, toks=None, scales=None, counts=None, send_only=False):
        """``send_only``: only queue the sends; ``complete()`` then waits for the peers' tokens and packs them
        (work queued in between overlaps the transfer)."""
        torch, L = self.torch, self.lib
        stream = self._stream()
        if self.handle is None:
            idx_t = _tensor(topk_idx, INT64)
            h = ctypes.c_void_p()
            _lib.check(L.ncclEpCreateHandle(ctypes.byref(h), self.group, self.layout_code, ctypes.byref(idx_t), None, None, stream), "ncclEpCreateHandle", L)
            self.handle = h
        lead = self._lead
        if toks is None:
            toks = torch.empty(*lead, self.H, dtype=torch.uint8 if fp8 else torch.bfloat16, device=x.device)
        if scales is None and fp8:
            scales = torch.empty(*lead, self.H // 128, dtype=torch.float32, device=x.device)
        if counts is None:
            counts = torch.zeros(self.El, dtype=torch.int32, device=x.device)
        recv = (None, None, None)
        if self.layout != "expert_major":
            K = topk_idx.shape[1]
            self.recv_topk_idx = torch.empty(*lead, K, dtype=torch.int64, device=x.device)
            self.recv_topk_weights = torch.empty(*lead, K, dtype=torch.float32, device=x.device)
            if self.layout == "flat" or self.recv_total is None:   # nothing writes the rank-major one: it stays zero
                self.recv_total = torch.zeros(1, dtype=torch.int32, device=x.device)
            recv = (self.recv_topk_idx.data_ptr(), self.recv_topk_weights.data_ptr(), self.recv_total.data_ptr() if self.layout == "flat" else None)
        sp = scales.data_ptr() if fp8 else None
        if self._fast:   # a shape stands for the four words of `_dims`
            rc = self._fast[0](self._fast[1], self.handle, x.data_ptr(), x.shape, topk_idx.data_ptr(), topk_idx.shape, topk_weights.data_ptr(), topk_weights.shape,
                               toks.data_ptr(), toks.shape, sp, counts.data_ptr(), *recv, int(send_only), stream)
        else:
            rc = L.b200EpDispatch(self.handle, x.data_ptr(), *self._dims(x), topk_idx.data_ptr(), *self._dims(topk_idx), topk_weights.data_ptr(),
                                  *self._dims(topk_weights), toks.data_ptr(), *self._dims(toks), sp, counts.data_ptr(), *recv, int(send_only), stream)
        _lib.check(rc, "ncclEpDispatch", L)
        self._keep = (x, topk_idx, topk_weights, toks, scales, counts)
        self.T = x.shape[0]
        return toks, scales, counts

    def combine(self, y, out=None, send_only=False):
        torch, L = self.torch, self.lib
        out = out if out is not None else torch.empty(self.T, self.H, dtype=torch.bfloat16, device=y.device)
        if self._fast:
            rc = self._fast[0](self._fast[2], self.handle, y.data_ptr(), y.shape, out.data_ptr(), out.shape, int(send_only), self._stream())
        else:
            rc = L.b200EpCombine(self.handle, y.data_ptr(), *self._dims(y), out.data_ptr(), *self._dims(out), int(send_only), self._stream())
        _lib.check(rc, "ncclEpCombine", L)
        self._keep_c = (y, out)
        return out

    # ------------------------------------------------------------------ routing, the experts' products, and the gradients across the exchange
    def _moe_protos(self, fast):
        L, P, I = self.lib, ctypes.c_void_p, ctypes.c_int
        types = {"ncclEpRoute": [P, P, I, P, P, P, I, I, I, P, P], "ncclEpRouteBackward": [P, P, P, I, P, P, I, I, I, P, P],
                 "ncclEpExpertLinear": [P] * 8 + [I] * 5 + [P], "ncclEpExpertLinearBackward": [P] * 10 + [I] * 5 + [P],
                 "ncclEpDispatchRows": [P, P, P], "ncclEpCombineBackward": [P] * 7 + [I] * 4 + [P], "ncclEpDispatchBackward": [P] * 4 + [I] * 4 + [P]}
        self._moe = {}
        for name, args in types.items():
            fn = getattr(L, name, None)
            if fn is None:
                continue   # a library without them
            fn.argtypes = args
            entry = _lib.address(L, name) if fast else None
            self._moe[name] = functools.partial(fast.invoke, entry) if entry else fn
        if self._moe:
            L.ncclEpExpertLinearBackwardWork.argtypes = [P, I, I, I, I, I]
            L.ncclEpExpertLinearBackwardWork.restype = ctypes.c_size_t
        dev = ctypes.c_int()
        _lib.check(L.ncclCommCuDevice(self.comm.handle, ctypes.byref(dev)), "ncclCommCuDevice", L)
        torch = self.torch
        self._device, self._place = dev.value, torch.device("cuda", dev.value)
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or current_stream
        self._route_cfgs = {}
        self._logit_codes = {torch.float32: FP32, torch.float16: FP16, torch.bfloat16: BF16}

    def _moe_call(self, name, *args):
        rc = self._moe[name](*args, self._raw_stream(self._device))
        if rc:
            _lib.check(rc, name, self.lib)

    def _need(self, name, t, dtype, shape):
        """Checks a tensor: type, shape, contiguous, on the group's GPU."""
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

    def _route_cfg(self, *rule):
        """The configuration, kept for the next call. Whoever hands its address on holds it until then: another thread may clear the store."""
        cfg = self._route_cfgs.get(rule)
        if cfg is None:
            score, groups, keep, group_score, renormalize, scale = rule
            if score not in self.SCORES:
                raise ValueError("score must be one of %s, not %r" % (", ".join(map(repr, self.SCORES)), score))
            if group_score not in self.GROUP_SCORES:
                raise ValueError("group_score must be one of %s, not %r" % (", ".join(map(repr, self.GROUP_SCORES)), group_score))
            if max(abs(groups), abs(keep)) >> 31:
                raise ValueError("%r groups, %r kept" % (groups, keep))   # (the library refuses what 32 bits can say)
            cfg = _hdr(RouteCfg())
            cfg.score, cfg.groups, cfg.keep_groups, cfg.group_score = self.SCORES[score], groups, keep, self.GROUP_SCORES[group_score]
            cfg.renormalize, cfg.scale = int(bool(renormalize)), scale
            if len(self._route_cfgs) >= 64:
                self._route_cfgs.clear()
            self._route_cfgs[rule] = cfg
        return cfg

    def _logits(self, logits):
        code, shape = self._logit_codes.get(logits.dtype), logits.shape
        if code is None or len(shape) != 2 or shape[1] != self.E or shape[0] >= 1 << 31:
            raise ValueError("logits must be an fp32, fp16 or bf16 tensor [tokens, %d], not %s %s" % (self.E, str(logits.dtype).replace("torch.", ""), list(shape)))
        self._need("logits", logits, logits.dtype, shape)
        return code

    def route(self, logits, topk, score="softmax", bias=None, groups=1, keep_groups=None, group_score="max", renormalize=True, scale=1.0, idx=None, weights=None):
        """What ``dispatch`` takes: (int64 [tokens, topk] expert ids, fp32 [tokens, topk] weights) from router logits [tokens, num_experts].

        Scores are the softmax or sigmoid of the logits (fp32, fp16 or bf16). Experts are ranked by score + ``bias`` (fp32 [num_experts]; it
        chooses and does not weigh) among the ``keep_groups`` best of ``groups`` equal runs of experts; a group counts as its best expert
        (``group_score="max"``) or the sum of its two best ("top2"). Best first; equal ones by index. Weights are ``scale`` * score, with
        ``renormalize`` divided by the sum of the taken experts' scores. Experts whose logit is -inf or NaN are never taken: entries that
        find none are -1 with weight 0, which ``dispatch`` leaves out (rows of -inf stand for padding)."""
        code = self._logits(logits)
        topk = int(topk)
        T, i64, f32 = logits.shape[0], self.torch.int64, self.torch.float32
        if bias is not None:
            self._need("bias", bias, f32, (self.E,))
        cfg = self._route_cfg(score, groups, groups if keep_groups is None else keep_groups, group_score, renormalize, scale)
        idx, weights = self._result("idx", idx, i64, (T, topk)), self._result("weights", weights, f32, (T, topk))
        self._moe_call("ncclEpRoute", self.group, logits.data_ptr(), code, None if bias is None else bias.data_ptr(), idx.data_ptr(), weights.data_ptr(), T, self.E, topk, ctypes.addressof(cfg))
        return idx, weights

    def route_backward(self, dweights, logits, idx, score="softmax", renormalize=True, scale=1.0, out=None):
        """Gradient of the logits (their type) from that of the weights; ``idx`` and the rule as ``route`` had them. The choice has no gradient.
        ``out`` may be the logits."""
        code = self._logits(logits)
        T, topk = idx.shape
        self._need("dweights", dweights, self.torch.float32, (T, topk))
        self._need("idx", idx, self.torch.int64, (logits.shape[0], topk))
        cfg = self._route_cfg(score, 1, 1, "max", renormalize, scale)
        out = self._result("out", out, logits.dtype, logits.shape)
        self._moe_call("ncclEpRouteBackward", self.group, dweights.data_ptr(), logits.data_ptr(), code, idx.data_ptr(), out.data_ptr(), T, self.E, topk, ctypes.addressof(cfg))
        return out

    def _linear(self, x, w, counts, activation):
        """(experts, rows, n, k, columns of the result, code of the activation) of a product, its operands checked."""
        torch = self.torch
        if activation not in self.ACTIVATIONS:
            raise ValueError("activation must be one of %s, not %r" % (", ".join(map(repr, self.ACTIVATIONS)), activation))
        if x.dim() != 3 or w.dim() != 3:
            raise ValueError("x must be [experts, rows, k] and w [experts, n, k], not %s and %s" % (list(x.shape), list(w.shape)))
        E, rows, k = x.shape
        n = w.shape[1]
        gated = activation in ("swiglu", "geglu")
        if n % (16 if gated else 8) or k % 8 or not 0 < E <= 256 or max(rows, n, k) > 1 << 24 or not n or not k:
            raise ValueError("%d experts (at most 256) of %d rows, n = %d must be a multiple of %d and k = %d of 8, none above 2^24" % (E, rows, n, 16 if gated else 8, k))
        self._need("x", x, torch.bfloat16, (E, rows, k))
        self._need("w", w, torch.bfloat16, (E, n, k))
        if counts is not None:
            self._need("counts", counts, torch.int32, (E,))
        return E, rows, n, k, n // 2 if gated else n, self.ACTIVATIONS[activation]

    def _pre(self, pre, shape):
        """What the type of the kept pre-activations adds to the activation's code."""
        fp32 = pre.dtype is self.torch.float32
        self._need("pre", pre, self.torch.float32 if fp32 else self.torch.bfloat16, shape)
        return self.PRE_FP32 if fp32 else 0

    def expert_linear(self, x, w, counts, bias=None, activation=None, residual=None, out=None, pre=None):
        """act(x w^T + bias) + residual for every expert over its rows in use, as ``dispatch`` packs and counts them; bf16 with fp32 sums.

        x [experts, rows, k], w [experts, n, k], counts int32 [experts] (None: all rows), bias [experts, n], residual and the result [experts, rows, n].
        activation: None, "relu", "gelu" (by erf), "silu", or gated, "swiglu" and "geglu": w is then gate rows and up rows one after the other, and
        the result, silu(gate) * up or gelu(gate) * up, has n / 2 columns. n and k are multiples of 8 (gated: n of 16). ``pre``
        [experts, rows, n], bf16 or fp32, gets x w^T + bias for the backward pass: fp32 for gradients as exact as bf16 products make them, bf16
        for half the memory. Rows behind an expert's last are not written; ``residual`` may be ``out``."""
        torch = self.torch
        E, rows, n, k, cols, act = self._linear(x, w, counts, activation)
        bf16, ptr = torch.bfloat16, lambda t: None if t is None else t.data_ptr()   # noqa: E731
        if bias is not None:
            self._need("bias", bias, bf16, (E, n))
        if residual is not None:
            self._need("residual", residual, bf16, (E, rows, cols))
        if pre is not None:
            act |= self._pre(pre, (E, rows, n))
        out = self._result("out", out, bf16, (E, rows, cols))
        self._moe_call("ncclEpExpertLinear", self.group, x.data_ptr(), w.data_ptr(), ptr(counts), ptr(bias), ptr(residual), out.data_ptr(), ptr(pre), E, rows, n, k, act)
        return out

    def expert_linear_backward(self, dout, x, w, counts, pre=None, activation=None, need_dx=True, need_dw=True, need_dbias=False, dx=None, dw=None, dbias=None):
        """(dx, dw, dbias) of ``expert_linear``, None for those that are not needed; the residual's gradient is ``dout`` itself. ``pre`` as the
        forward call filled it (not needed without an activation). dx has the rows in use only; dw and dbias are zero for experts without rows."""
        torch = self.torch
        E, rows, n, k, cols, act = self._linear(x, w, counts, activation)
        bf16, ptr = torch.bfloat16, lambda t: None if t is None else t.data_ptr()   # noqa: E731
        self._need("dout", dout, bf16, (E, rows, cols))
        if act:
            if pre is None:
                raise ValueError("the gradient of an activation needs what it was applied to: give expert_linear and this call the same `pre`")
            act |= self._pre(pre, (E, rows, n))
        dx = self._result("dx", dx, bf16, (E, rows, k)) if need_dx else None
        dw = self._result("dw", dw, bf16, (E, n, k)) if need_dw else None
        dbias = self._result("dbias", dbias, bf16, (E, n)) if need_dbias else None
        size = self.lib.ncclEpExpertLinearBackwardWork(self.group, E, rows, n, act, int(need_dbias))
        work = torch.empty(size, dtype=torch.uint8, device=self._place) if size else None
        self._moe_call("ncclEpExpertLinearBackward", self.group, dout.data_ptr(), x.data_ptr(), w.data_ptr(), ptr(counts), ptr(pre) if act else None, ptr(dx), ptr(dw),
                       ptr(dbias), ptr(work), E, rows, n, k, act)
        return dx, dw, dbias

    def dispatch_rows(self, rows=None):
        """int32 [tokens, topk]: the row of the dispatched tensor (as [experts * capacity, hidden]) that holds each entry of the last ``dispatch``, -1
        for entries without an expert. Groups of one rank with the expert-major layout; the next dispatch moves the rows."""
        if self.handle is None or self._keep is None:
            raise ValueError("nothing has been dispatched yet")
        idx = self._keep[1]
        rows = self._result("rows", rows, self.torch.int32, tuple(idx.shape))
        self._moe_call("ncclEpDispatchRows", self.handle, rows.data_ptr())
        return rows

    def combine_backward(self, dout, y, weights, rows, dy=None, dweights=None):
        """(dy, dweights) of ``combine`` from the gradient [tokens, hidden] of its result: dy[row] = weight * dout[token] for the rows that
        ``rows`` (see ``dispatch_rows``) names, each by one entry; dweights[t, k] = <dout[t], y[row]>. dy is like y and may be y."""
        torch = self.torch
        if dout.dim() != 2 or y.dim() < 2 or weights.dim() != 2:
            raise ValueError("dout must be [tokens, hidden], y [..., hidden], weights [tokens, topk], not %s, %s, %s" % (list(dout.shape), list(y.shape), list(weights.shape)))
        (T, H), K, bf16 = dout.shape, weights.shape[1], torch.bfloat16
        if H == 0 or H % 8 or not 0 < K <= 16 or y.numel() // H >= 1 << 31 or T >= 1 << 31:
            raise ValueError("hidden = %d must be a multiple of 8, topk = %d at most 16, rows and tokens below 2^31" % (H, K))
        self._need("dout", dout, bf16, (T, H))
        self._need("y", y, bf16, (*y.shape[:-1], H))
        self._need("weights", weights, torch.float32, (T, K))
        self._need("rows", rows, torch.int32, (T, K))
        dy, dweights = torch.empty_like(y) if dy is None else self._result("dy", dy, bf16, y.shape), self._result("dweights", dweights, torch.float32, (T, K))
        self._moe_call("ncclEpCombineBackward", self.group, dout.data_ptr(), y.data_ptr(), weights.data_ptr(), rows.data_ptr(), dy.data_ptr(), dweights.data_ptr(), T, K, H,
                       y.numel() // H)
        return dy, dweights

    def dispatch_backward(self, dtoks, rows, out=None):
        """Gradient of the tokens, [tokens, hidden], from that of the dispatched rows: the sum over the token's rows."""
        torch = self.torch
        if dtoks.dim() < 2 or rows.dim() != 2:
            raise ValueError("dtoks must be [..., hidden] and rows [tokens, topk], not %s and %s" % (list(dtoks.shape), list(rows.shape)))
        (T, K), H = rows.shape, dtoks.shape[-1]
        if H == 0 or H % 8 or not 0 < K <= 16 or dtoks.numel() // H >= 1 << 31 or T >= 1 << 31:
            raise ValueError("hidden = %d must be a multiple of 8, topk = %d at most 16, rows and tokens below 2^31" % (H, K))
        self._need("dtoks", dtoks, torch.bfloat16, dtoks.shape)
        self._need("rows", rows, torch.int32, (T, K))
        out = self._result("out", out, torch.bfloat16, (T, H))
        self._moe_call("ncclEpDispatchBackward", self.group, dtoks.data_ptr(), rows.data_ptr(), out.data_ptr(), T, K, H, dtoks.numel() // H)
        return out
