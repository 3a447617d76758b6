"""What lies behind the lengths of a padded batch reaches no result, in the forms that long calls take: two tiles of queries to a CTA, keys or queries cut into parts. Values are compared bit
for bit with those beside zeros, and those with 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

from cp_reference import Reference, check  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def cp():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from nccl_b200 import Communicator, get_unique_id
    from nccl_b200.ops.cp import ContextParallel
    torch.cuda.set_device(0)
    comm = Communicator(1, 0, get_unique_id())
    c = ContextParallel(comm)
    yield c
    torch.cuda.synchronize()
    assert comm.async_error() == 0
    c.destroy()
    comm.destroy()


CASES = [
    # B, Q, K, H, G, D, causal, q_lengths, kv_lengths, what is in parts: forward, backward (keys and values of a batch, queries)
    (4, 300, 640, 40, 8, 72, True, (300, 299, 1, 130), (639, 513, 1, 0), False, False),              # pairs
    (2, 700, 900, 32, 8, 64, False, (513, 700), (897, 385), False, False),
    (3, 1024, 1024, 16, 16, 64, True, (1, 900, 1023), (1, 900, 1023), False, False),
    (2, 40, 3000, 4, 2, 72, True, (40, 33), (2999, 1793), True, True),                               # one tile of queries, keys in 12 parts
    (2, 100, 4000, 4, 2, 64, False, (99, 0), (3900, 4000), True, True),
    (3, 1, 5000, 8, 2, 128, True, None, (4999, 129, 2600), True, True),                              # few rows
    (3, 3, 4000, 8, 2, 72, True, (3, 2, 3), (3973, 1, 2049), True, True),
    (2, 2048, 2048, 1, 1, 64, True, (2047, 1300), (2047, 1300), True, True),                         # back: both in parts
    (2, 1500, 260, 8, 1, 64, False, (1499, 700), (259, 200), False, True),
    (2, 700, 900, 4, 1, 96, True, (677, 130), (897, 385), False, True),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_rows_behind_the_lengths_may_hold_anything(cp, dtype, case):
    B, Q, K, H, G, D, causal, ql, kl, forward_parts, backward_parts = case
    g = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)   # noqa: E731
    operands = r(B, Q, H, D), r(B, K, G, D), r(B, K, G, D), r(B, Q, H, D)
    ql, kl = (None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ql, kl))
    rule = dict(causal=causal, q_lengths=ql, kv_lengths=kl)

    def filled(what):
        ts = [t.clone() for t in operands]
        for t, n in zip(ts, (ql, kl, kl, ql)):
            for b in range(B if n is not None else 0):
                t[b, int(n[b]):] = what
        return ts
    cp._shapes.clear()
    got = []
    for junk in (0.0, math.nan, math.inf, torch.finfo(dtype).min):
        q, k, v, dout = filled(junk)
        out, lse = cp.attention(q, k, v, **rule)
        grads = cp.attention_backward(dout, q, k, v, out, lse, **rule)
        delta = cp.attention_delta(dout, out, ql)
        assert all(torch.equal(a, b) for a, b in zip(grads, cp.attention_backward(dout, q, k, v, None, lse, delta=delta, **rule)))
        got.append((out, lse) + grads)
    for junk in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], junk))
    # the case is of the form that it stands for: parts have a workspace
    sizes = [what[-1][2] for what in cp._shapes.values() if what[-1].__class__ is tuple]
    rows = B * Q * H * D * 4, B * K * G * D * 4
    assert (sizes[0] > 0) == forward_parts and (sizes[1] >= 2 * min(rows)) == backward_parts, sizes
    q, k, v, dout = filled(0.0)
    ref = Reference(q, k, v, causal, None, None, ql, kl, dout=dout, out=got[0][0])
    check("lse", got[0][1], ref.lse, ref.lse_tol)
    check("out", got[0][0], ref.out, ref.out_tol)
    for name, t in zip(("dv", "dk", "dq"), got[0][:1:-1]):
        check(name, t, getattr(ref, name), getattr(ref, name + "_tol"))
