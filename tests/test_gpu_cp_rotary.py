"""Rotary positions of ``ContextParallel`` against 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

from cp_reference import half_step, rotary  # noqa: E402

pytestmark = pytest.mark.gpu


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


def check(got, want, x, amplitude, half):
    """An angle of less than half a turn is rounded to fp32 (2^-24 of at most pi, so 2^-22.3), its sine and cosine and the two products and their sum by a few 2^-24 each: together
    less than 2^-20 of |a| + |b|; and the result by half a step."""
    m = torch.finfo(x.dtype)
    size = amplitude * 2 * x.detach().cpu().double().abs().amax(-1, keepdim=True)
    tol = want.abs() * half_step(x.dtype) * (1 + 2.0 ** -10) + size * 2.0 ** -20 + m.smallest_normal * m.eps
    tol[..., 2 * half:] = 0
    off = (got.detach().cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol.clamp_min(1e-300)).max())


CASES = [
    # B, T, heads, kv_heads, channels, turned, type, interleaved, positions, offset
    (1, 1, 32, 8, 128, 128, torch.bfloat16, False, "int64", 0),
    (2, 37, 4, 2, 128, 128, torch.bfloat16, False, None, 1000003),
    (3, 133, 12, 4, 80, 40, torch.float16, True, "int64", 0),
    (1, 9, 3, 1, 24, 14, torch.float32, False, "int32", 0),
    (1, 9, 3, 1, 24, 14, torch.float32, True, None, -5),
    (2, 50, 1, 1, 2, 2, torch.float16, True, None, 7),
    (1, 700, 7, 1, 64, 64, torch.float32, True, "int64", 0),
    (1, 5, 2, 2, 1024, 1024, torch.bfloat16, False, "int32", 0),
    (4, 1024, 8, 8, 64, 48, torch.bfloat16, False, None, 1 << 40),
    (1, 3, 70, 3, 1023, 6, torch.float16, False, None, 3),
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_rotary(cp, case, inverse):
    B, T, H, G, D, turned, dtype, interleaved, kind, offset = case
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k = (torch.randn(B, T, n, D, device="cuda", generator=g).to(dtype) for n in (H, G))
    positions = None if kind is None else torch.randint(0, 1 << 20, (B, T), device="cuda", generator=g).to(getattr(torch, kind))
    freqs = cp.rotary_frequencies(turned, base=500000.0, amplitude=1.25)
    from nccl_b200.ops.cp import rotary_turns
    turns = rotary_turns(turned, 500000.0)
    at = positions if positions is not None else (offset + torch.arange(T)).expand(B, T)
    got = cp.rotary(q, k, freqs, positions=positions, offset=offset, interleaved=interleaved, inverse=inverse)
    for x, y in zip((q, k), got):
        check(y, rotary(x, at, turns, 1.25, interleaved, inverse), x, 1.25, turned // 2)
    alone = cp.rotary(q, None, freqs, positions=positions, offset=offset, interleaved=interleaved, inverse=inverse)
    assert alone[1] is None and torch.equal(alone[0], got[0])
    place = cp.rotary(q, k, freqs, positions=positions, offset=offset, interleaved=interleaved, inverse=inverse, out=(q, k))
    assert place[0] is q and torch.equal(q, got[0]) and torch.equal(k, got[1])


def test_rotary_of_one_projection(cp):
    """Queries and keys between one another's rows, in place; what lies behind them stays."""
    B, T, H, G, D = 2, 65, 6, 2, 64
    x = torch.randn(B, T, H + 2 * G, D, device="cuda").bfloat16()
    q, k, v = x.split((H, G, G), dim=2)
    freqs = cp.rotary_frequencies(D)
    want = cp.rotary(q.contiguous(), k.contiguous(), freqs, offset=11)
    before = v.clone()
    cp.rotary(q, k, freqs, offset=11, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, before)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(cp.rotary(heads_first, None, freqs, offset=3)[0], cp.rotary(q, None, freqs, offset=3)[0])


def test_rotary_gradient(cp):
    """The inverse is the transposed map: <turn(x), y> = <x, turn back(y)>, to the rounding of fp32."""
    x, y = (torch.randn(1, 40, 2, 64, device="cuda") for _ in range(2))
    freqs = cp.rotary_frequencies(48, scaling="ntk", factor=4.0, amplitude=0.5)
    a = (cp.rotary(x, None, freqs, offset=90000, interleaved=True)[0].double() * y.double()).sum()
    b = (x.double() * cp.rotary(y, None, freqs, offset=90000, interleaved=True, inverse=True)[0].double()).sum()
    assert abs(float(a - b)) <= 2.0 ** -19 * float((x.double().abs() * y.double().abs()).sum() + x.numel())


def test_rotary_without_tokens(cp):
    freqs = cp.rotary_frequencies(16)
    q, k = cp.rotary(torch.empty(2, 0, 4, 16, device="cuda"), torch.empty(2, 0, 1, 16, device="cuda"), freqs)
    assert q.shape == (2, 0, 4, 16) and k.shape == (2, 0, 1, 16)
    assert math.isclose(freqs.amplitude, 1.0)
