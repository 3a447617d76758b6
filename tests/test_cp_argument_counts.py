"""Tuples of tensors that the context-parallel operators take: one of another length would put every pointer behind it in a wrong place."""
import pytest

torch = pytest.importorskip("torch")

from test_cp_arguments import cp, qkv  # noqa: E402, F401


def test_gradients_to_add_to_come_in_threes(cp):   # noqa: F811
    q, k, v = qkv()
    out, lse = cp.attention(q, k, v)
    sums = torch.zeros(q.shape), torch.zeros(k.shape), torch.zeros(k.shape)
    n = len(cp.calls)
    for add in ((), sums[:1], sums[:2], sums + (sums[0],), sums[0][:0]):
        with pytest.raises(ValueError):
            cp.attention_backward(out, q, k, v, out, lse, add=add)
    assert len(cp.calls) == n
    for add in (sums, list(sums), iter(sums)):
        cp.attention_backward(out, q, k, v, out, lse, add=add)
        assert len(cp.calls[-1]) == 20 and cp.calls[-1][12:15] == tuple(t.data_ptr() for t in sums)


def test_what_joins_is_a_pair(cp):   # noqa: F811
    q, k, v = qkv()
    join = torch.zeros(q.shape), torch.zeros(2, 4, 5)
    n = len(cp.calls)
    for bad in ((), join[:1], join + (join[1],)):
        with pytest.raises(ValueError):
            cp.attention(q, k, v, join=bad)
    assert len(cp.calls) == n
    cp.attention(q, k, v, join=list(join))
    assert cp.calls[-1][8:10] == tuple(t.data_ptr() for t in join)
