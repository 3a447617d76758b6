"""Rotary positions of as many tokens as a call takes: 2^31 - 1."""
import pytest

torch = pytest.importorskip("torch")

from cp_reference import half_step, rotary  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T", [(1, 2 ** 31 - 1), (3, (2 ** 31 - 1) // 3), (2 ** 31 - 1, 1)])
def test_as_many_tokens_as_a_call_takes(B, T):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    from nccl_b200 import Communicator, get_unique_id
    from nccl_b200.ops.cp import ContextParallel
    torch.cuda.set_device(0)
    comm = Communicator(1, 0, get_unique_id())
    cp = ContextParallel(comm)
    freqs = cp.rotary_frequencies(2, base=10.0)
    pattern = torch.randn(1 << 20, 2, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).half()
    flat = torch.empty(B * T, 2, dtype=torch.float16, device="cuda")
    for i in range(0, B * T, 1 << 20):
        flat[i:i + (1 << 20)] = pattern[:min(1 << 20, B * T - i)]
    x = flat.view(B, T, 1, 2)
    turns = freqs.turns.tolist()
    got = cp.rotary(x, None, freqs, offset=5, out=(x, None))[0]
    assert got is x
    torch.cuda.synchronize()
    for i in (0, T - 500, T, 2 * T - 300, (B * T) // 2, B * T - 1000):   # around the sequences' ends, and where the counts end
        lo = min(max(0, i), B * T - 1000)
        hi = lo + 1000
        at = torch.arange(lo, hi)
        before = pattern.cpu()[at % (1 << 20)].view(1, -1, 1, 2)
        want = rotary(before, 5 + at[None] % T, turns)
        off = (flat[lo:hi].cpu().double() - want.view(-1, 2)).abs()
        # (bounds as for any call: 2^-20 of |a| + |b| for the angle and the sum, half a step for the result)
        tol = want.view(-1, 2).abs() * half_step(torch.float16) * (1 + 2.0 ** -10) + 2 * before.double().abs().amax(-1).view(-1, 1) * 2.0 ** -20 + 2.0 ** -24
        assert bool((off <= tol).all())
    del x, flat, got
    torch.cuda.empty_cache()
    assert comm.async_error() == 0
    cp.destroy()
    comm.destroy()
