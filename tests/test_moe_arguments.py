"""What the mixture-of-experts operators refuse before anything reaches a GPU, and what they hand to the library: tensors in host memory,
with the library's calls recorded."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture()
def ep():
    from nccl_b200.core import BF16, FP16, FP32
    from nccl_b200.ops.ep import ExpertParallel
    e = ExpertParallel.__new__(ExpertParallel)
    e.torch, e.E, e.El, e._device, e._place, e.group, e.handle = torch, 16, 16, -1, torch.device("cpu"), 111, None
    e._raw_stream, e._route_cfgs = (lambda device: 222), {}
    e._logit_codes = {torch.float32: FP32, torch.float16: FP16, torch.bfloat16: BF16}
    e.calls = []

    class Lib:
        @staticmethod
        def ncclEpExpertLinearBackwardWork(group, experts, rows, n, act, bias):
            return 64

    e.lib = Lib()

    def record(name):
        def call(*args):
            e.calls.append((name,) + args)
            return 0
        return call

    e._moe = {n: record(n) for n in ("ncclEpRoute", "ncclEpRouteBackward", "ncclEpExpertLinear", "ncclEpExpertLinearBackward", "ncclEpDispatchRows",
                                     "ncclEpCombineBackward", "ncclEpDispatchBackward")}
    return e


def test_route_hands_over_its_rule(ep):
    from nccl_b200.ops.ep import EP_MAGIC, RouteCfg
    logits, bias = torch.randn(5, 16), torch.zeros(16)
    idx, w = ep.route(logits, 3, score="sigmoid", bias=bias, groups=4, keep_groups=2, group_score="top2", renormalize=False, scale=2.5)
    name, group, at, code, b, i, ww, tokens, experts, topk, cfg, stream = ep.calls[0]
    assert (name, group, at, code, b, i, ww) == ("ncclEpRoute", 111, logits.data_ptr(), 7, bias.data_ptr(), idx.data_ptr(), w.data_ptr())
    assert (tokens, experts, topk, stream) == (5, 16, 3, 222) and idx.dtype == torch.int64 and w.dtype == torch.float32 and idx.shape == w.shape == (5, 3)
    c = ctypes.cast(cfg, ctypes.POINTER(RouteCfg)).contents
    assert (c.size, c.magic, c.score, c.groups, c.keep_groups, c.group_score, c.renormalize, c.scale) == (ctypes.sizeof(RouteCfg), EP_MAGIC, 1, 4, 2, 1, 0, 2.5)
    ep.route(logits.bfloat16(), 3, groups=4)   # all groups stay unless told otherwise
    c = ctypes.cast(ep.calls[1][-2], ctypes.POINTER(RouteCfg)).contents
    assert (ep.calls[1][3], ep.calls[1][4], c.score, c.groups, c.keep_groups, c.renormalize, c.scale) == (9, None, 0, 4, 4, 1, 1.0)
    ep.route_backward(w, logits, idx, score="sigmoid", renormalize=False, scale=2.5)
    c = ctypes.cast(ep.calls[2][-2], ctypes.POINTER(RouteCfg)).contents
    assert ep.calls[2][0] == "ncclEpRouteBackward" and (c.score, c.renormalize, c.scale) == (1, 0, 2.5)
    for _ in range(200):   # configurations do not pile up
        ep.route(logits, 2, scale=1.0 + len(ep.calls))
    assert len(ep._route_cfgs) <= 64


def test_route_refuses(ep):
    l = torch.randn(5, 16)
    idx, w = ep.route(l, 4)
    for bad in (l[:, :8], l.double(), l.t().contiguous().t(), l[0], l[None]):
        with pytest.raises(ValueError):
            ep.route(bad, 4)
        with pytest.raises(ValueError):
            ep.route_backward(w, bad, idx)
    for kw in (dict(score="tanh"), dict(group_score="mean"), dict(bias=torch.zeros(15)), dict(bias=torch.zeros(16).half()), dict(idx=idx.int()), dict(weights=w[:3])):
        with pytest.raises(ValueError):
            ep.route(l, 4, **kw)
    for dw, i, kw in ((w.double(), idx, {}), (w[:, :2], idx, {}), (w, idx[:4], {}), (w, idx.int(), {}), (w, idx, dict(out=l.half())), (w, idx, dict(score=None))):
        with pytest.raises(ValueError):
            ep.route_backward(dw, l, i, **kw)
    assert len(ep.calls) == 1


def test_a_rule_in_use_outlives_the_store(ep):
    """Another thread may clear the store of rules between a call's look into it and its launch."""
    import weakref
    result, kept = ep._result, []

    def clearing(*args):
        kept.extend(weakref.ref(c) for c in ep._route_cfgs.values())
        ep._route_cfgs.clear()
        return result(*args)

    ep._result = clearing
    alive = []
    for name in ("ncclEpRoute", "ncclEpRouteBackward"):
        ep._moe[name] = lambda *args: alive.append(kept[-1]() is not None) or 0
    logits = torch.randn(5, 16)
    idx, w = ep.route(logits, 3, scale=1.25)
    ep.route_backward(w, logits, idx, scale=1.5)
    assert alive == [True, True] and len(kept) == 2


@pytest.mark.parametrize("kw", [dict(groups=1 + (1 << 32)), dict(groups=4, keep_groups=2 + (1 << 32)), dict(groups=1 - (1 << 32))])
def test_numbers_of_groups_beyond_32_bits(ep, kw):
    with pytest.raises(ValueError):
        ep.route(torch.randn(5, 16), 2, **kw)


def test_expert_linear_hands_over_and_refuses(ep):
    bf = dict(dtype=torch.bfloat16)
    x, w, c = torch.randn(2, 16, 32).bfloat16(), torch.randn(2, 48, 32).bfloat16(), torch.tensor([16, 3], dtype=torch.int32)
    out = ep.expert_linear(x, w, c, activation="swiglu")
    assert out.shape == (2, 16, 24) and ep.calls[0][1:] == (111, x.data_ptr(), w.data_ptr(), c.data_ptr(), None, None, out.data_ptr(), None, 2, 16, 48, 32, 4, 222)
    pre, d = torch.empty(2, 16, 48, **bf), torch.empty(2, 16, 24, **bf)
    dx, dw, db = ep.expert_linear_backward(d, x, w, None, pre=pre, activation="geglu", need_dx=False)
    assert dx is None and db is None and dw.shape == w.shape and ep.calls[1][5:8] == (None, pre.data_ptr(), None) and ep.calls[1][8] == dw.data_ptr()
    done = len(ep.calls)
    d = torch.empty(2, 16, 48, **bf)
    for args, kw in (((x.float(), w, c), {}), ((x, w.float(), c), {}), ((x, w[:, :, :16], c), {}), ((x, w, c.long()), {}), ((x, w, c[:1]), {}), ((x[0], w, c), {}),
                     ((x, w[:1], c), {}), ((x.transpose(0, 1), w, c), {}), ((x, w, c), dict(activation="tanh")), ((x, w[:, :40].contiguous(), c), dict(activation="swiglu")),
                     ((x[:, :, :12].contiguous(), w[:, :, :12].contiguous(), c), {}), ((x, w, c), dict(bias=torch.zeros(2, 47, **bf))),
                     ((x, w, c), dict(residual=d.float())), ((x, w, c), dict(out=d[:, :8])), ((x, w, c), dict(pre=x)),
                     ((torch.empty(257, 1, 8, **bf), torch.empty(257, 8, 8, **bf), None), {}), ((torch.empty(0, 1, 8, **bf), torch.empty(0, 8, 8, **bf), None), {})):
        with pytest.raises(ValueError):
            ep.expert_linear(*args, **kw)
    for args, kw in (((d[:, :, :40].contiguous(), x, w, c), {}), ((d, x, w, c), dict(activation="gelu")), ((d, x, w, c), dict(activation="gelu", pre=x)),
                     ((d, x, w, c), dict(dx=d)), ((d, x, w, c), dict(need_dbias=True, dbias=d))):
        with pytest.raises(ValueError):
            ep.expert_linear_backward(*args, **kw)
    assert len(ep.calls) == done


def test_gradients_of_the_exchange_refuse(ep):
    x, y, w, rows = torch.randn(3, 128).bfloat16(), torch.randn(4, 16, 128).bfloat16(), torch.rand(3, 2), torch.zeros(3, 2, dtype=torch.int32)
    dy, dw = ep.combine_backward(x, y, w, rows)
    assert dy.shape == y.shape and dw.shape == w.shape and ep.calls[0][-5:] == (3, 2, 128, 64, 222)
    assert ep.dispatch_backward(y, rows).shape == (3, 128) and ep.calls[1][-5:] == (3, 2, 128, 64, 222)
    for args in ((x.float(), y, w, rows), (x, y.float(), w, rows), (x, y[..., :64], w, rows), (x, y, w.double(), rows), (x, y, w, rows.long()), (x, y, w, rows[:2]),
                 (x, y, w[:, :1], rows), (x[:, :100].contiguous(), y[..., :100].contiguous(), w, rows), (x, y.transpose(0, 1), w, rows), (x[0], y, w, rows),
                 (x, y, torch.rand(3, 17), torch.zeros(3, 17, dtype=torch.int32)), (x[:, :0], y[..., :0], w, rows)):
        with pytest.raises(ValueError):
            ep.combine_backward(*args)
    for args in ((y.float(), rows), (y, rows.long()), (y, rows[0]), (y.transpose(0, 1), rows), (y[0, 0], rows), (y[..., :0], rows)):
        with pytest.raises(ValueError):
            ep.dispatch_backward(*args)
    with pytest.raises(ValueError):
        ep.dispatch_rows()
    assert len(ep.calls) == 2


def test_entry_points_without_a_group(lib):
    """Null handles are refused, not followed."""
    lib = ctypes.CDLL(lib._name)   # prototypes of its own
    for name, n in (("ncclEpRoute", 11), ("ncclEpRouteBackward", 11), ("ncclEpExpertLinear", 14), ("ncclEpExpertLinearBackward", 16), ("ncclEpDispatchRows", 3),
                    ("ncclEpCombineBackward", 12), ("ncclEpDispatchBackward", 9)):
        fn = getattr(lib, name)
        fn.argtypes = [ctypes.c_void_p] * n
        fn.restype = ctypes.c_int
        assert fn(*[None] * n) == 4, name
    lib.ncclEpExpertLinearBackwardWork.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 5
    lib.ncclEpExpertLinearBackwardWork.restype = ctypes.c_size_t
    assert lib.ncclEpExpertLinearBackwardWork(None, 1, 1, 8, 1, 1) == 0
